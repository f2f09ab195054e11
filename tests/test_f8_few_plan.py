"""Where products of 8-bit floating point take the forms of few rows (f8_mul_plan): on the
CPU.  Grouped calls whose experts have few rows on average can be large, and their rows need
not be spread evenly; dense calls of more than 16 rows can be small."""
import pytest

from hipf8 import BF16, F32
from test_f8_plan import form


# times, microseconds: the form taken, and the one of few rows
@pytest.mark.parametrize("type,rows,experts,n,k,gated", (
    (BF16, 8192, 1024, 512, 512, True),   # 262 of 381; skewed 244 of 379
    (F32, 10240, 1024, 512, 512, True),   # 296 of 637; skewed 282 of 636
    (BF16, 1536, 64, 1024, 2048, True),   # 57 of 67; skewed 62 of 76
    (BF16, 512, 64, 2048, 1024, False),   # 34 of 50; skewed 33 of 51
    (F32, 896, 64, 2048, 1024, False),    # 41 of 52; skewed 40 of 54
    (F32, 160, 8, 14336, 4096, True)))    # 195 of 240; skewed 197 of 273
def test_large_grouped_calls_of_few_rows_an_expert(type, rows, experts, n, k, gated):
    assert form(type, rows, n, k, gated, experts=experts) == "TILE_64"


@pytest.mark.parametrize("type,rows,experts,n,k,gated", (
    (BF16, 32, 8, 14336, 4096, True), (F32, 256, 64, 1024, 2048, True), (BF16, 256, 64, 1024, 2048, True)))
def test_grouped_steps(type, rows, experts, n, k, gated):
    assert form(type, rows, n, k, gated, experts=experts) == "FEW_GATED"


@pytest.mark.parametrize("type", (BF16, F32))
@pytest.mark.parametrize("rows,n,k", (  # fp32: 10.6 of 15.5, 8.6 of 14.7, 27.7 of 40.6 us
    (24, 4096, 4096), (48, 1024, 4096), (24, 4096, 14336)))
def test_dense_calls_of_more_than_a_tile(type, rows, n, k):
    assert form(type, rows, n, k) == "FEW_LONG"


@pytest.mark.parametrize("rows,n,k,gated", ((24, 14336, 4096, True), (24, 50304, 2048, False), (129, 1024, 4096, False)))
def test_dense_calls_with_enough_work_for_tiles(rows, n, k, gated):
    assert form(BF16, rows, n, k, gated)[:3] != "FEW"
