"""How exact the 8-bit floating-point products (hip_f8.h) are: what the header states,
where other tests' inputs do not reach it.

Sums.  A block's 128 products are exact in fp32, their sum is off by 127 roundings of
2^-24 of the block's size, size = sum |x w|: below 2^-17 of it.  The product of two scales
is one rounding, joining the accumulator one more of at most size 2^-24 for each of the
(k + 127) / 128 blocks (partial sums of blocks that are added up at the end take no more).
With one more for what is of second order, E = 2^-17 + (k / 128 + 3) 2^-24.  16-bit outputs
have 2^-10 on top, from the matrix cores' cutting of each of eight products at 2^-13 of the
largest one's power of two.
"""
import numpy as np
import pytest

import f8_ref as ref
import hipf8
from f8_ref import BF16, BLOCK, F16, F32, Dev, wide
from test_f8_plan import form
from test_gpu_f8 import dev  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def E(ty, k):
    return 2.0 ** -17 + (k / BLOCK + 3) * 2.0 ** -24 + (0 if ty == F32 else 2.0 ** -10)


def rows_on(dev, codes, scale):  # noqa: F811
    n, k = codes.shape
    room = np.full((n, -(-k // 16) * 16), 0x7f, np.uint8)
    room[:, :k] = codes
    return hipf8.Rows(dev.up(room), room.shape[1], dev.up(scale.astype(np.float32)), n, n, k)


def mat_on(dev, codes, scale, count=1):  # noqa: F811
    """Matrices that are all the same."""
    n, k = codes.shape
    room = np.full((n, -(-k // 16) * 16), 0x7f, np.uint8)
    room[:, :k] = codes
    return hipf8.Mat(dev.up(room), room.shape[1], dev.up(scale.astype(np.float32)), ref.blocks(k), n, k, count, 0, 0)


@pytest.mark.parametrize("ty", (F32, F16, BF16))
@pytest.mark.parametrize("rows,n,experts,name", ((3, 40, 0, "FEW_LONG"), (150, 64, 0, "MID_64"), (40, 64, 2, "FEW_32")))
def test_a_million_channels_of_one_sign(dev, ty, rows, n, experts, name):  # noqa: F811
    """Blocks that are all the same: an accumulator's roundings go the same way over a whole
    power of two, which is the most that they can be."""
    k = 1 << 20
    assert form(ty, rows, n, k, experts=experts) == name
    rng = np.random.default_rng(rows + experts)
    xc, wc = (ref.codes_of(np.abs(rng.standard_normal((m, BLOCK))) * 112 + 16) for m in (rows, n))
    sx = (1 + rng.random(rows)).astype(np.float32) * np.float32(2.0 ** -16)
    sw = (1 + rng.random(ref.blocks(n))).astype(np.float32) * np.float32(2.0 ** -19)
    X = rows_on(dev, np.tile(xc, k // BLOCK), np.tile(sx, (k // BLOCK, 1)))
    W = mat_on(dev, np.tile(wc, k // BLOCK), np.repeat(sw[:, None], k // BLOCK, 1), max(1, experts))
    stride = wide(n, ty)
    d_o = dev.up(np.zeros((rows, stride), ref.np_dtype(ty)))
    if experts:
        start = np.linspace(0, rows, experts + 1).astype(np.int32)
        hipf8.group_mul(X, None, dev.up(start), rows, W, None, ty, d_o, stride)
    else:
        hipf8.mul(X, W, None, ty, d_o, stride)
    got = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)[:, :n]
    scale = sx.astype(np.float64)[:, None] * np.repeat(sw.astype(np.float64), BLOCK)[:n]
    want = ref.VALUES[xc] @ ref.VALUES[wc].T * scale * (k // BLOCK)
    off = np.abs(got - want) / want
    print(f"off by 2^{np.log2(off.max()):.2f}")
    assert np.all(off <= E(ty, k) + ref.HALF_STEP[ty] * (1 + E(ty, k)))


@pytest.mark.parametrize("ty", (F32, BF16))
@pytest.mark.parametrize("rows,n,k", ((3, 40, 300), (40, 200, 300), (700, 1500, 300)))
def test_products_of_scales_below_the_normal_numbers(dev, ty, rows, n, k):  # noqa: F811
    """They are rounded to multiples of 2^-149: off by half of one times the codes' size more,
    and so is an output."""
    rng = np.random.default_rng(rows)
    xc, wc = (ref.random_codes(rng, (m, k)) for m in (rows, n))
    sx = ((1 + rng.random((ref.blocks(k), rows))) * 2.0 ** -90).astype(np.float32)
    sw = ((1 + rng.random((ref.blocks(n), ref.blocks(k)))) * 2.0 ** -50).astype(np.float32)
    stride = wide(n, ty)
    d_o = dev.up(np.zeros((rows, stride), ref.np_dtype(ty)))
    hipf8.mul(rows_on(dev, xc, sx), mat_on(dev, wc, sw), None, ty, d_o, stride)
    got = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)[:, :n]
    x, w = ref.rows_of(xc, sx), ref.mat_of(wc, sw)
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    codes = np.abs(ref.VALUES[xc]) @ np.abs(ref.VALUES[wc]).T
    tol = size * E(ty, k) + codes * 2.0 ** -150 + 2.0 ** -149
    assert np.all(np.abs(got - want) <= tol * (1 + ref.HALF_STEP[ty]) + np.abs(want) * ref.HALF_STEP[ty])
    assert np.abs(want).max() > 2.0 ** -122  # most of them are normal numbers


@pytest.mark.parametrize("ty", (F32, F16, BF16))
@pytest.mark.parametrize("rows", (9, 400))
def test_gates_of_any_size(dev, ty, rows):  # noqa: F811
    """silu(a) of exact a from -130 to 130, times a b large enough that no gate's own size
    hides what it is off by.  The exponential of a rounded a / ln 2 is |a| 2^-23 off in relation
    and its own, the sum's and the quotient's roundings 2^-20; a silu(a) below 2^-119 may be 0."""
    rng = np.random.default_rng(rows)
    a = np.concatenate([[-130, -104, -89, -88.5, -87.6, -87.2, -86, 0.01, 88], rng.uniform(0, 130, rows - 9)])
    a = a.astype(np.float32)
    one = np.full((rows, 1), 0x38, np.uint8)
    sign = np.where(np.arange(20) % 2, 0x38, 0xb8).astype(np.uint8)[:, None]
    big = np.float32(2.0 ** (90 if ty != F16 else 3))
    # row r's scale is |a[r]|, the outputs' matrix rows are -1 and 1: both signs of it
    X = rows_on(dev, one, np.abs(a)[None])
    W, U = mat_on(dev, sign, np.ones((1, 1))), mat_on(dev, np.full((20, 1), 0x38, np.uint8), np.full((1, 1), big))
    d_o = dev.up(np.zeros((rows, 24), ref.np_dtype(ty)))
    hipf8.mul(X, W, U, ty, d_o, 24)
    got = ref.from_type(dev.get(d_o, (rows, 24), ref.np_dtype(ty)), ty)[:, :20]
    a = np.abs(a).astype(np.float64)[:, None] * ref.VALUES[sign[:, 0]]
    b = np.abs(a) * np.float64(big)
    want = ref.gate(a, b)
    tol = np.abs(want) * (ref.HALF_STEP[ty] + 2.0 ** -20 + np.abs(a) * 2.0 ** -23) + b * 2.0 ** -119
    tol += 2.0 ** -25 if ty == F16 else 2.0 ** -140
    fine = np.abs(got - want) <= tol
    if ty == F16:  # 65520 and more are rounded to infinity
        fine |= (got == np.inf) & (want + tol >= 65520)
    assert np.all(fine)


def cut_error(rng, xc, xs, wc, ws, pairs=400):
    """What 16-bit outputs' sums are off by at most, root of the mean square over outputs: where a
    product has bits below 2^-13 of the power of two of the largest of its eight, a unit of those.
    Cut towards 0, products of either sign are off by either sign, so that squares add up; a
    unit is three times what the squares of cut-off bits are on average."""
    r, c = rng.integers(0, xc.shape[0], pairs), rng.integers(0, wc.shape[0], pairs)
    k = xc.shape[1]
    p = np.zeros((pairs, -(-k // 8) * 8))
    p[:, :k] = ref.VALUES[xc[r]] * ref.VALUES[wc[c]]
    g = p.reshape(pairs, -1, 8)
    unit = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(g).max(2, keepdims=True), 2.0 ** -60))) - 13)
    off = np.where(np.trunc(g / unit) * unit != g, unit, 0).reshape(pairs, -1)[:, :k]
    scale = np.repeat(xs[:, r].T.astype(np.float64) * ws[c // BLOCK], BLOCK, 1)[:, :k]
    return np.sqrt(((off * scale) ** 2).sum(1).mean())


@pytest.mark.parametrize("outliers", (0.0, 0.05))
@pytest.mark.parametrize("name,ty,rows,n,k", (
    ("FEW_LONG", BF16, 16, 500, 1100), ("FEW_WIDE", F16, 3, 20000, 400), ("MID_32", F16, 40, 4000, 650),
    ("MID_64", BF16, 2725, 285, 2293), ("MID_128", BF16, 1300, 1500, 391), ("TILE_64", F16, 1300, 6000, 520),
    ("TILE_128", BF16, 2100, 2200, 520), ("TILE_256", F16, 4100, 6200, 520), ("TILE_256", BF16, 4100, 6200, 520)))
def test_sums_of_16_bit_outputs(dev, name, ty, rows, n, k, outliers):  # noqa: F811
    """An addend of minus the rounded result leaves what the sum is off by: far less than a 16-bit
    output's own rounding.  Over whole outputs it is within what the matrix cores' cutting gives
    (and the remainder's rounding)."""
    assert form(ty, rows, n, k) == name
    rng = np.random.default_rng(rows + n + k)
    x = rng.standard_normal((rows, k)) * (1 + 7 * (rng.random(k) < outliers))
    xc, xs = ref.quantize(x.astype(np.float32))
    wc = ref.random_codes(rng, (n, k))
    ws = (rng.uniform(0.7, 1.3, (ref.blocks(n), ref.blocks(k))) * 2e-4).astype(np.float32)
    want = ref.rows_of(xc, xs) @ ref.mat_of(wc, ws).T
    stride = wide(n, ty)
    add = np.zeros((rows, stride), ref.np_dtype(ty))
    add[:, :n] = ref.to_type(-want, ty)
    rest = want + ref.from_type(add, ty)[:, :n]
    d_o = dev.up(add)
    hipf8.mul(rows_on(dev, xc, xs), mat_on(dev, wc, ws), None, ty, d_o, stride, d_o, stride)
    got = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)[:, :n]

    def rms(v):
        return np.sqrt(np.square(v).mean())
    cut = cut_error(rng, xc, xs, wc, ws)
    print(f"off by {rms(got - rest) / rms(want):.2e} of the outputs, cutting at most {cut / rms(want):.2e}")
    assert rms(got - rest) <= cut + ref.HALF_STEP[ty] * rms(rest) + (2.0 ** -25 if ty == F16 else 0)
    assert cut <= 1e-4 * rms(want)


@pytest.mark.parametrize("ty", (F32, F16, BF16))
def test_what_follows_a_row_in_its_16_bytes_does_not_matter(dev, ty):  # noqa: F811
    """Rows of x, y and add end inside 16 bytes, the rest of which is NaN; one row of add for all."""
    rng = np.random.default_rng(3)
    n = 101
    stride = wide(n, ty)

    def up(rows):
        v = np.full((rows, stride), np.nan, np.float32)
        v[:, :n] = rng.standard_normal((rows, n))
        return dev.up(ref.to_type(v, ty)), ref.from_type(ref.to_type(v, ty), ty)[:, :n]

    (d_x, x), (d_add, add) = up(7), up(1)
    d_c, d_s = dev.up(np.zeros((7, 112), np.uint8)), dev.up(np.zeros((1, 7), np.float32))
    X = hipf8.Rows(d_c, 112, d_s, 7, 7, n)
    hipf8.quantize(ty, d_x, stride, X)
    codes, scale = ref.quantize(x)
    assert np.array_equal(dev.get(d_c, (7, 112), np.uint8)[:, :n], codes)
    assert np.array_equal(dev.get(d_s, (1, 7), np.float32), scale)
    pos, w = rng.integers(0, 7, (5, 2)).astype(np.int32), rng.random((5, 2)).astype(np.float32)
    d_o = dev.up(np.zeros((7, stride), ref.np_dtype(ty)))
    for d_a, a in ((d_add, add), (None, 0 * add)):
        hipf8.combine(ty, d_x, stride, 7, dev.up(pos), dev.up(w), 5, 2, n, d_a, 0, d_o, stride)
        got = ref.from_type(dev.get(d_o, (7, stride), ref.np_dtype(ty)), ty)[:5, :n]
        terms = w[..., None].astype(np.float64) * x[pos]
        want, size = a + terms.sum(1), np.abs(a) + np.abs(terms).sum(1)
        assert np.all(np.abs(got - want) <= np.abs(want) * ref.HALF_STEP[ty] + size * 3 * 2.0 ** -23 + 2.0 ** -25)
    wc = ref.random_codes(rng, (n, n))
    W = mat_on(dev, wc, np.full((1, 1), 2e-4, np.float32))
    hipf8.mul(X, W, None, ty, d_o, stride, d_add, 0)
    got = ref.from_type(dev.get(d_o, (7, stride), ref.np_dtype(ty)), ty)[:, :n]
    xd, wd = ref.rows_of(codes, scale), ref.mat_of(wc, np.full((1, 1), 2e-4, np.float32))
    want, size = xd @ wd.T + add, np.abs(xd) @ np.abs(wd).T + np.abs(add)
    assert np.all(np.abs(got - want) <= np.abs(want) * ref.HALF_STEP[ty] + size * E(ty, n) + 2.0 ** -25)
