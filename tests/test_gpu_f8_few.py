"""The products of hip_f8.h around the border between few rows and tiles: dense calls of several
tiles of 16 rows, and tiles where most of many experts have a few rows and some have many.
Inputs and comparison: test_gpu_f8_forms.py."""
import pytest

import test_gpu_f8_forms as forms
from f8_ref import BF16, F16, F32
from test_gpu_f8 import dev  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty,gated,rows,n,k", (
    (F32, False, 100, 600, 2000), (F32, True, 128, 200, 1100), (F16, False, 33, 1000, 300), (BF16, False, 128, 200, 1100),
    (F32, False, 17, 2500, 1100)))
def test_dense_few(dev, ty, gated, rows, n, k):  # noqa: F811
    forms.test_dense(dev, "FEW_LONG", ty, gated, rows, n, k)


@pytest.mark.parametrize("gather", (False, True))
@pytest.mark.parametrize("ty,gated,counts,n,k", (
    (F32, False, (7, 0, 12, 1, 3) * 30, 700, 257), (BF16, True, (7, 0, 12, 1, 3) * 30, 1000, 257),
    (F32, True, (3, 0, 0, 40, 1) * 20, 1000, 257), (F16, False, (10, 0, 33, 9) * 20, 700, 391),
    (BF16, False, (0,) * 60 + (1, 300, 0, 70) + (2,) * 30, 1000, 257)))
def test_grouped_tiles(dev, ty, gated, counts, n, k, gather):  # noqa: F811
    forms.test_grouped(dev, "TILE_64", ty, gated, counts, n, k, gather)
