"""The products' tiles of 256 x 256 (hip_f8.h) where a workgroup goes on to a next tile: gathered
and gated rows of several experts, and the fewest channels that the form takes.  There (257 to
384) the next tile's rows are asked for in a tile's first block and used in its second, and the
one after that is its last.  Inputs and comparison: test_gpu_f8_forms.py."""
import pytest

import test_gpu_f8_forms as forms
from f8_ref import BF16, F16
from test_f8_plan import plan
from test_gpu_f8 import dev  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

CUS = 256  # workgroups of a stream
MANY = (513, 0, 257, 1025, 5, 769, 300)


@pytest.mark.parametrize("ty,gated,rows,n,k", (
    (F16, False, 5100, 4200, 257), (BF16, True, 4100, 2600, 384), (F16, True, 2600, 4200, 257)))
def test_dense(dev, ty, gated, rows, n, k):  # noqa: F811
    p = plan(ty, rows, n, k, gated)[1]
    assert p.row_tiles * p.n_tiles > CUS
    forms.test_dense(dev, "TILE_256", ty, gated, rows, n, k)


@pytest.mark.parametrize("gather", (False, True))
@pytest.mark.parametrize("ty,gated,counts,n,k", (
    (BF16, True, MANY, 3100, 257), (F16, True, MANY, 3100, 384), (BF16, False, MANY, 4200, 257),
    (F16, False, forms.RAGGED, 6200, 384), (BF16, True, forms.RAGGED, 3700, 1000),
    (F16, True, (1300, 2600, 1, 1300, 1300, 1300), 1500, 300)))
def test_grouped(dev, ty, gated, counts, n, k, gather):  # noqa: F811
    # the tiles that there are, of which the host knows only the most that there can be
    assert sum(-(-c // 256) for c in counts) * -(-n // (128 if gated else 256)) > CUS
    forms.test_grouped(dev, "TILE_256", ty, gated, counts, n, k, gather)
