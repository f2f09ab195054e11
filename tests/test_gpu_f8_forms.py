"""The products of hip_f8.h in every form that they take, at sizes where it is taken, with
tiles that are not full, channels that end inside a block, addends, gathered rows, rows
from outside and NaN.  Compared with numpy in 64 bits at the tiles' edges and some other
rows (tolerances: test_gpu_f8.py); NaN at all."""
import numpy as np
import pytest

import f8_ref as ref
import hipf8
from f8_ref import BF16, F16, F32, Dev, DevMat, DevRows, up_typed, wide
from test_f8_plan import form
from test_gpu_f8 import check_product, dev, product  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def rows_with_nan(dev, rng, n, k):
    """Rows two of which hold a NaN code or scale, and which these are."""
    x = rng.standard_normal((n, k)) * (1 + 7 * (rng.random(k) < 0.05))
    codes, scale = ref.quantize(x.astype(np.float32))
    bad = np.unique([min(5, n - 1), n - 1])
    codes[bad[0], k // 2] = 0x7f
    scale[-1, bad[-1]] = np.nan
    return DevRows(dev, codes, scale, pad=1, scale_pad=3), bad


def mat_with_nan(dev, rng, n, k, count=1):
    codes = ref.random_codes(rng, (count, n, k))
    codes[0, n - 1, k - 1] = 0xff
    return DevMat(dev, rng, n, k, count, pad=1, scale_pad=1, codes=codes)


def some(rng, n):
    i = np.arange(n)
    edge = np.isin(i % 256, (0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 129, 255)) & (rng.random(n) < 0.5)
    return np.flatnonzero(edge | (rng.random(n) < 40 / n) | (i >= n - 3))


DENSE = (  # form, type, gated, rows, n, k
    ("FEW_LONG", BF16, False, 7, 500, 1100), ("FEW_LONG", F32, True, 16, 300, 2000), ("FEW_WIDE", F16, False, 3, 20000, 400),
    ("FEW_WIDE", F32, False, 1, 17001, 1030), ("FEW_GATED", BF16, True, 16, 17000, 390), ("MID_32", F16, False, 40, 4000, 650),
    ("MID_64", BF16, False, 2725, 285, 2293), ("MID_64", F32, True, 64, 4100, 2000), ("MID_128", BF16, False, 1300, 1500, 391),
    ("MID_128", F32, False, 1300, 1500, 391), ("MID_SQUARE", F32, False, 1000, 3000, 650), ("MID_SQUARE", F32, True, 450, 3000, 650),
    ("TILE_64", F16, False, 1300, 6000, 520), ("TILE_64", BF16, True, 1300, 6000, 400), ("TILE_64", F32, True, 1500, 4352, 400),
    ("TILE_64", F32, False, 3000, 3000, 640),
    ("TILE_128", BF16, False, 2100, 2200, 520), ("TILE_128", F16, True, 1000, 3000, 520), ("TILE_128F", F32, False, 4100, 4352, 400),
    ("TILE_128F", F32, True, 4100, 4352, 400), ("TILE_256", F16, False, 4100, 6200, 520), ("TILE_256", BF16, True, 4500, 3000, 391),
    ("TILE_256", F16, True, 2100, 6200, 391))


@pytest.mark.parametrize("name,ty,gated,rows,n,k", DENSE)
def test_dense(dev, name, ty, gated, rows, n, k):  # noqa: F811
    assert form(ty, rows, n, k, gated) == name
    rng = np.random.default_rng(rows + n)
    X, bad = rows_with_nan(dev, rng, rows, k)
    W = mat_with_nan(dev, rng, n, k)
    U = DevMat(dev, rng, n, k) if gated else None
    stride = wide(n, ty, 1)
    add = None if gated else ref.from_type(ref.to_type(rng.standard_normal((rows, n)), ty), ty)
    d_o = up_typed(dev, np.zeros((rows, 0), np.float32), ty, stride, fill=-3.0)
    a_s = 0 if gated else wide(n, ty)
    hipf8.mul(X.rows, W.mat, U and U.mat, ty, d_o, stride, None if gated else up_typed(dev, add, ty, a_s), a_s)
    got = dev.get(d_o, (rows, stride), ref.np_dtype(ty))
    assert np.all(ref.from_type(got[:, n:], ty) == -3.0)
    nan = np.zeros((rows, n), bool)
    nan[bad], nan[:, n - 1] = True, True
    assert np.array_equal(np.isnan(ref.from_type(got[:, :n], ty)), nan)
    at = np.setdiff1d(some(rng, rows), bad)
    want, size = product(X.x[at], W.w[0][:n - 1], U and U.w[0][:n - 1], None if gated else add[at, :n - 1])
    check_product(ref.from_type(got[at, :n - 1], ty), want, size, ty)


RAGGED = (700, 3, 0, 1300, 257, 900)
GROUPED = (  # form, type, gated, experts' rows, n, k
    ("FEW_LONG", BF16, False, (3, 0, 17, 1, 5, 40) + (0,) * 94, 100, 300), ("FEW_GATED", F16, True, (9, 0, 30, 1) + (7,) * 90, 200, 520),
    ("FEW_32", F32, False, (20, 0, 45, 31, 1, 33), 300, 391), ("FEW_32", F16, True, (23,) * 70, 96, 200),
    ("MID_32", BF16, True, (300, 2, 500), 384, 272), ("TILE_64", BF16, True, (300, 3, 0, 500, 67, 200), 1500, 520),
    ("TILE_64", F32, True, RAGGED, 3000, 520), ("TILE_128", F16, False, (2000, 1, 1500, 0, 40), 2000, 400),
    ("TILE_128F", F32, True, (2000, 1, 1500, 0, 40), 2000, 400), ("TILE_64", BF16, False, (60, 0, 90) * 40, 700, 300),
    ("TILE_256", BF16, True, RAGGED, 1500, 1000), ("TILE_256", F16, False, RAGGED, 6200, 520))


@pytest.mark.parametrize("gather", (False, True))
@pytest.mark.parametrize("name,ty,gated,counts,n,k", GROUPED)
def test_grouped(dev, name, ty, gated, counts, n, k, gather):  # noqa: F811
    NE, total = len(counts), sum(counts)
    rows = total + 3  # and three of no expert
    assert form(ty, rows, n, k, gated, experts=NE) == name
    rng = np.random.default_rng(total + n)
    tokens = max(8, total // 3) if gather else rows
    X, bad = rows_with_nan(dev, rng, tokens, k)
    W = mat_with_nan(dev, rng, n, k, NE)
    U = DevMat(dev, rng, n, k, NE) if gated else None
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    frm = rng.integers(0, tokens, rows).astype(np.int32)
    frm[[1, total // 2, total - 1]] = tokens, -1, 1 << 30
    src = frm if gather else np.arange(rows)
    stride = wide(n, ty, 1)
    d_o = up_typed(dev, np.zeros((rows, 0), np.float32), ty, stride, fill=-3.0)
    hipf8.group_mul(X.rows, dev.up(frm) if gather else None, dev.up(start), rows, W.mat, U and U.mat, ty, d_o, stride)
    got = dev.get(d_o, (rows, stride), ref.np_dtype(ty))
    assert np.all(ref.from_type(got[:, n:], ty) == -3.0) and np.all(ref.from_type(got[total:], ty) == -3.0)
    none = (src < 0) | (src >= tokens)
    nan = np.zeros((total, n), bool)
    nan[none[:total] | np.isin(src[:total], bad)] = True
    nan[:counts[0], n - 1] = True  # the first expert's matrix has one
    assert np.array_equal(np.isnan(ref.from_type(got[:total, :n], ty)), nan)
    for e in range(NE):
        if not counts[e] or (NE > 20 and rng.random() > 0.2):
            continue
        at = start[e] + some(rng, counts[e])
        at = at[~nan[at, 0]]
        want, size = product(X.x[src[at]], W.w[e][:n - 1], U and U.w[e][:n - 1])
        if at.size:
            check_product(ref.from_type(got[at, :n - 1], ty), want, size, ty)
