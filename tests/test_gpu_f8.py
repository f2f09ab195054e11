"""The 8-bit floating-point products (hip_f8.h) on the GPU, against numpy in 64
bits (f8_ref.py).

Tolerances.  Codes, scales, and the sort's numbers are equal.  A product's output is
off by its own rounding (half a step of its type) and by E * size, size = sum |x w|.
fp32 outputs: the 128 products of a block are exact in fp32 (8 bits each) and their sum, in
whatever order, is off by 127 roundings of 2^-24 of at most the block's size each:
just below 2^-17.  Scaling and adding up a block takes three roundings more (the
product of the scales, its product with the sum joined to the accumulator, which
is one), and an accumulator's is at most size * 2^-24 each for k / 128 blocks: up to
100 blocks keep all of it below size * 2^-17 * (1 + 103 / 128).  E = 2^-16 bounds both.
16-bit outputs: the matrix cores cut each of eight products that they add up at 2^-13 of
the largest one's power of two, so that a group is off by 8 * 2^-13 of its largest, and
all of them by 2^-10 of the size; E = 2^-10 + 2^-16.
Over whole outputs the roundings are independent, so that 127 of them are as one
of sqrt(127): relative L2 error within sqrt(127) * 2^-24 * sqrt(2) < 1e-6 for fp32.
A gated output is g(a) b with g' at most 1.1 and |g(a)| <= |a|: off by
  1.1 E size_a |b| + |a| E size_b, and 2^-20 of itself for the exponential and the
division.
A combined output of n addends is off by n 2^-23 of their sizes' sum.
"""
import ctypes as C

import numpy as np
import pytest

import f8_ref as ref
import hipf8
import hipmoe
from f8_ref import BF16, BLOCK, F16, F32, Dev, DevMat, DevRows, random_rows, up_typed, wide

pytestmark = pytest.mark.gpu

TYPES = (F32, F16, BF16)
E = (2.0 ** -16, 2.0 ** -10 + 2.0 ** -16, 2.0 ** -10 + 2.0 ** -16)


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.free()


# --------------------------------------------------------------------------
# quantizing
# --------------------------------------------------------------------------

def quantize_on(dev, x, ty, pad=0, out_pad=0, scale_pad=0):
    """(codes, scales, whole codes) of values x [n][k] of the type."""
    n, k = x.shape
    stride = wide(k, ty, pad)
    d_x = up_typed(dev, x, ty, stride, fill=np.nan)
    o_stride = -(-k // 16) * 16 + 16 * out_pad
    d_c = dev.up(np.full((n, o_stride), 0x55, np.uint8))
    d_s = dev.up(np.full((ref.blocks(k), n + scale_pad), -5, np.float32))
    hipf8.quantize(ty, d_x, stride, hipf8.Rows(d_c, o_stride, d_s, n + scale_pad, n, k))
    codes = dev.get(d_c, (n, o_stride), np.uint8)
    scale = dev.get(d_s, (ref.blocks(k), n + scale_pad), np.float32)
    assert np.all(scale[:, n:] == -5)
    end = -(-k // 16) * 16
    assert np.all(codes[:, k:end] == 0) and np.all(codes[:, end:] == 0x55)
    return codes[:, :k], scale[:, :n]


def check_quantized(x, ty, got):
    codes, scale = ref.quantize(ref.from_type(ref.to_type(x, ty), ty))
    assert np.array_equal(got[1], scale, equal_nan=True)
    # a zero's sign is not told apart where the scale's rounding decides it
    assert np.array_equal(ref.VALUES[got[0]], ref.VALUES[codes])


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n,k,pads", (
    (1, 1, (0, 0, 0)), (1, 128, (0, 0, 0)), (3, 129, (1, 2, 5)), (17, 640, (0, 1, 0)), (4, 2047, (3, 0, 1)),
    (5, 100, (0, 0, 0)), (16, 4096, (0, 0, 0)), (2500, 1040, (0, 0, 3)), (1, 20000, (0, 0, 0))))
def test_quantize(dev, ty, n, k, pads):
    rng = np.random.default_rng(n * 31 + k)
    x = (rng.standard_normal((n, k)) * 2.0 ** rng.integers(-12, 12, (n, 1))).astype(np.float32)
    check_quantized(x, ty, quantize_on(dev, x, ty, *pads))


@pytest.mark.parametrize("ty", TYPES)
def test_quantize_next_to_borders(dev, ty):
    """Values halfway between two codes times the scale, and their neighbours; scales that are
    powers of two (every border is reached) and others."""
    rng = np.random.default_rng(5)
    v = np.sort(ref.VALUES[:127])
    mid = np.concatenate([(v[1:] + v[:-1]) / 2, v])
    rows = []
    for top in (448.0, 3.5, 7.0 * 2.0 ** -20, 448 * 1.2345, 1.0, 3.0, 0.1, 2.0 ** -14):
        s = np.float32(top) / np.float32(448)
        m = (mid[rng.integers(0, mid.size, 4 * BLOCK)] * s).astype(np.float32)
        m = np.minimum(m, np.float32(top))
        up, down = np.nextafter(m, np.float32(np.inf)), np.nextafter(m, np.float32(0))
        for x in (m, np.minimum(up, np.float32(top)), down):
            x = x * rng.choice((-1, 1), x.size).astype(np.float32)
            x[::BLOCK] = top
            rows.append(x)
    x = np.stack(rows)
    check_quantized(x, ty, quantize_on(dev, x, ty))


@pytest.mark.parametrize("ty", TYPES)
def test_quantize_blocks_of_zeros_extremes_and_nan(dev, ty):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((12, 3 * BLOCK)).astype(np.float32)
    x[0] = 0
    x[1, :BLOCK] = 0
    x[2] = np.float32(6e4 if ty == F16 else 3.3e38)
    x[3] = 1e-45 if ty == F32 else 6e-8 if ty == F16 else 1e-38
    x[4, 5] = np.nan
    x[5, BLOCK + 7] = np.inf
    x[6, 2 * BLOCK + 127] = -np.inf
    x[7] = x[7] * np.float32(2.0 ** -110)
    x[8, 0] = 1e30 if ty != F16 else 6e4
    x[9] = -0.0
    x[10, ::2] = np.nan
    x[11] = x[11] * np.float32(2.0 ** -90)
    check_quantized(x, ty, quantize_on(dev, x, ty))


# --------------------------------------------------------------------------
# products
# --------------------------------------------------------------------------

def product(x, w, u=None, add=None):
    """(result, what it may be off by without its rounding) for E = 1"""
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if u is None:
        return (y, size) if add is None else (y + add, size + np.abs(y) + np.abs(add))
    z, other = x @ u.T, np.abs(x) @ np.abs(u).T
    out = ref.gate(y, z)
    return out, 1.1 * size * np.abs(z) + np.abs(y) * other + np.abs(out) / 16


def check_product(got, want, size, ty):
    tol = np.abs(want) * (ref.HALF_STEP[ty] + 2.0 ** -24) + size * E[ty]
    if ty == F16:
        tol += 2.0 ** -25  # results below its smallest normal
    err = np.abs(got - want)
    assert np.all(err <= tol), (err / np.maximum(tol, 1e-300)).max()
    if ty == F32 and want.size >= 4096:
        assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


SHAPES = (  # rows, n, k
    (1, 1, 1), (1, 128, 128), (1, 300, 2048), (3, 17, 100), (5, 130, 257), (16, 256, 1024), (17, 64, 127),
    (33, 129, 640), (64, 512, 384), (65, 200, 4097), (130, 70, 272), (257, 384, 512), (300, 1000, 144),
    (513, 640, 1152), (31, 2080, 16), (2, 5000, 3200), (9, 48, 11000))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("gated", (False, True))
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_mul(dev, ty, gated, rows, n, k):
    rng = np.random.default_rng(rows * 7 + n + k)
    X = random_rows(dev, rng, rows, k, pad=rows % 3, scale_pad=k % 3)
    W = DevMat(dev, rng, n, k, pad=n % 2, scale_pad=rows % 2)
    U = DevMat(dev, rng, n, k, pad=1) if gated else None
    stride = wide(n, ty, 1)
    d_o = up_typed(dev, np.zeros((rows, 0), np.float32), ty, stride, fill=-3.0)
    hipf8.mul(X.rows, W.mat, U and U.mat, ty, d_o, stride)
    got = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)
    assert np.all(got[:, n:] == -3.0)
    want, size = product(X.x, W.w[0], U and U.w[0])
    check_product(got[:, :n], want, size, ty)
    hipf8.mul(X.rows, W.mat, U and U.mat, ty, d_o, stride)  # the same call, the same bits
    again = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)
    assert np.array_equal(again, got)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,n,k", ((1, 130, 384), (20, 257, 128), (150, 520, 640)))
def test_mul_add(dev, ty, rows, n, k):
    rng = np.random.default_rng(n)
    X, W = random_rows(dev, rng, rows, k), DevMat(dev, rng, n, k)
    stride = wide(n, ty)
    add = ref.from_type(ref.to_type(rng.standard_normal((rows, n)), ty), ty)
    d_o = dev.up(np.zeros((rows, stride), ref.np_dtype(ty)))
    for a, a_stride in ((add, wide(n, ty, 2)), (add[:1], 0)):
        d_a = up_typed(dev, a, ty, a_stride or stride)
        hipf8.mul(X.rows, W.mat, None, ty, d_o, stride, d_a, a_stride)
        got = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)
        check_product(got[:, :n], *product(X.x, W.w[0], add=a), ty)
    # in place
    d_a = up_typed(dev, add, ty, stride)
    hipf8.mul(X.rows, W.mat, None, ty, d_a, stride, d_a, stride)
    got = ref.from_type(dev.get(d_a, (rows, stride), ref.np_dtype(ty)), ty)
    check_product(got[:, :n], *product(X.x, W.w[0], add=add), ty)


def group_case(rng, experts, counts, gap=0):
    start = np.concatenate([[gap], gap + np.cumsum(counts)]).astype(np.int32)
    assert len(start) == experts + 1
    return start


GROUPS = (  # rows of the experts, n, k
    ([1], 64, 128), ([0, 0, 3, 0], 100, 256), ([5, 0, 1, 70], 257, 130), ([16, 16, 17, 15], 128, 384),
    ([64, 1, 0, 128, 65, 200], 200, 512), ([0] * 70 + [3] + [0] * 60 + [20] + [0] * 3, 96, 128),
    ([1, 2] * 100, 48, 256), ([300, 2, 500], 384, 272), ([0, 0, 0], 64, 64), ([2] * 8, 2048, 1040))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("gated", (False, True))
@pytest.mark.parametrize("gather", (False, True))
@pytest.mark.parametrize("counts,n,k", GROUPS)
def test_group_mul(dev, ty, gated, gather, counts, n, k):
    rng = np.random.default_rng(sum(counts) + n + k)
    NE = len(counts)
    gap = 3 if gather else 0  # rows before the first expert's and behind the last's
    start = group_case(rng, NE, counts, gap)
    rows = int(start[-1]) + 2
    tokens = max(1, rows // 2) if gather else rows
    X = random_rows(dev, rng, tokens, k, pad=1, scale_pad=2)
    W = DevMat(dev, rng, n, k, NE, pad=1)
    U = DevMat(dev, rng, n, k, NE, scale_pad=1) if gated else None
    frm = rng.integers(0, tokens, rows).astype(np.int32)
    frm[:gap], frm[rows - 2:] = -7, 1 << 30  # of no expert: not read
    stride = wide(n, ty, 1)
    d_o = up_typed(dev, np.zeros((rows, 0), np.float32), ty, stride, fill=-3.0)
    hipf8.group_mul(X.rows, dev.up(frm) if gather else None, dev.up(start), rows, W.mat, U and U.mat, ty, d_o,
                    stride)
    got = ref.from_type(dev.get(d_o, (rows, stride), ref.np_dtype(ty)), ty)
    assert np.all(got[:, n:] == -3.0) and np.all(got[:gap] == -3.0) and np.all(got[start[-1]:] == -3.0)
    for e in range(NE):
        a, b = start[e], start[e + 1]
        if b > a:
            x = X.x[frm[a:b]] if gather else X.x[a:b]
            check_product(got[a:b, :n], *product(x, W.w[e], U and U.w[e]), ty)


def test_group_rows_from_outside_are_nan(dev):
    rng = np.random.default_rng(9)
    X, W = random_rows(dev, rng, 10, 256), DevMat(dev, rng, 70, 256, 3)
    start = np.array([0, 4, 4, 30], np.int32)
    frm = rng.integers(0, 10, 30).astype(np.int32)
    frm[[2, 9, 29]] = 10, -1, 1 << 30
    d_o = dev.up(np.zeros((30, 72), np.float32))
    hipf8.group_mul(X.rows, dev.up(frm), dev.up(start), 30, W.mat, None, F32, d_o, 72)
    got = dev.get(d_o, (30, 72), np.float32)[:, :70]
    assert np.array_equal(np.isnan(got).all(1), (frm < 0) | (frm > 9)) and np.isnan(got).sum() == 3 * 70
    for r in range(30):
        if 0 <= frm[r] < 10:
            want, size = product(X.x[frm[r]:frm[r] + 1], W.w[0 if r < 4 else 2])
            check_product(got[r:r + 1], want, size, F32)


def test_group_starts_past_the_rows(dev):
    """What a start says past the rows of the call is cut to them, and rows that fall back are none."""
    rng = np.random.default_rng(10)
    X, W = random_rows(dev, rng, 20, 128), DevMat(dev, rng, 16, 128, 4)
    start = np.array([-5, 6, 3, 1 << 30, 1 << 30], np.int32)
    d_o = dev.up(np.full((24, 16), -3, np.float32))
    hipf8.group_mul(X.rows, None, dev.up(start), 20, W.mat, None, F32, d_o, 16)
    got = dev.get(d_o, (24, 16), np.float32)
    assert np.all(got[20:] == -3)
    check_product(got[:3], *product(X.x[:3], W.w[0]), F32)
    check_product(got[6:20], *product(X.x[6:], W.w[2]), F32)


@pytest.mark.parametrize("rows", (1, 20, 100))
def test_nan_codes_and_scales_stay_in_their_rows(dev, rows):
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, 300)).astype(np.float32)
    codes, scale = ref.quantize(x)
    codes[0, 299] = 0xff
    if rows > 1:
        scale[1, rows - 1] = np.nan
    X = DevRows(dev, codes, scale)
    w = ref.random_codes(rng, (1, 140, 300))
    w[0, 139, 0] = 0x7f
    W = DevMat(dev, rng, 140, 300, codes=w)
    d_o = dev.up(np.zeros((rows, 140), np.float32))
    hipf8.mul(X.rows, W.mat, None, F32, d_o, 140)
    got = dev.get(d_o, (rows, 140), np.float32)
    with np.errstate(invalid="ignore"):
        want, size = product(X.x, W.w[0])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    check_product(got[fine], want[fine], size[fine], F32)


# --------------------------------------------------------------------------
# the sort and the sum
# --------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,topk,experts", (
    (1, 1, 1), (1, 8, 64), (16, 2, 8), (5, 3, 130), (1000, 7, 12), (333, 8, 256), (4000, 6, 1024), (8192, 8, 64),
    (70000, 1, 3), (65537, 1, 5), (30001, 9, 700)))
@pytest.mark.parametrize("away", (0.0, 0.4, 1.0))
def test_sort(dev, tokens, topk, experts, away):
    rng = np.random.default_rng(tokens + topk)
    ids = rng.integers(0, experts, (tokens, topk)).astype(np.uint32)
    far = np.array([experts, experts + 1, 1 << 31, 0xffffffff], np.uint32)
    ids = np.where(rng.random(ids.shape) < away, far[rng.integers(0, 4, ids.shape)], ids)
    d_s, d_f = dev.up(np.full(experts + 1, -9, np.int32)), dev.up(np.full(tokens * topk, -9, np.int32))
    d_p = dev.up(np.full((tokens, topk), -9, np.int32))
    hipf8.sort(dev.up(ids), tokens, topk, experts, d_s, d_f, d_p)
    start, frm, pos = ref.sort(ids, experts)
    assert np.array_equal(dev.get(d_s, experts + 1, np.int32), start)
    got = dev.get(d_f, tokens * topk, np.int32)
    assert np.array_equal(got[:frm.size], frm) and np.all(got[frm.size:] == -9)
    assert np.array_equal(dev.get(d_p, (tokens, topk), np.int32), pos)


def test_sort_without_tokens(dev):
    d_s = dev.up(np.full(6, -9, np.int32))
    hipf8.sort(None, 0, 2, 5, d_s, None, None)
    assert np.all(dev.get(d_s, 6, np.int32) == 0)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("tokens,topk,n,add", (
    (1, 1, 1, None), (16, 2, 4096, "rows"), (3, 8, 2049, "row"), (40, 5, 100, "in place"), (1000, 3, 24, None),
    (7, 9, 700, "rows"), (130, 1, 2600, "in place")))
def test_combine(dev, ty, tokens, topk, n, add):
    rng = np.random.default_rng(tokens * topk + n)
    y_rows = max(1, tokens * topk // 2)
    y = ref.from_type(ref.to_type(rng.standard_normal((y_rows, n)), ty), ty)
    pos = rng.integers(0, y_rows, (tokens, topk)).astype(np.int32)
    pos[rng.random(pos.shape) < 0.3] = -1
    pos[0, 0], pos[-1, -1] = y_rows, -(1 << 31)
    w = rng.random((tokens, topk)).astype(np.float32)
    here = (pos >= 0) & (pos < y_rows)
    w[~here] = np.nan  # not read
    ys, os = wide(n, ty, 2), wide(n, ty, 1)
    a = ref.from_type(ref.to_type(rng.standard_normal((tokens, n)), ty), ty)
    if add == "row":
        a = a[:1]
    d_o = up_typed(dev, a if add == "in place" else a[:0], ty, os, fill=-3.0) if add == "in place" else \
        up_typed(dev, np.zeros((tokens, 0), np.float32), ty, os, fill=-3.0)
    d_a, a_s = {None: (None, 0), "in place": (d_o, os), "row": (up_typed(dev, a, ty, wide(n, ty)), 0),
                "rows": (up_typed(dev, a, ty, ys), ys)}[add]
    hipf8.combine(ty, up_typed(dev, y, ty, ys, fill=np.nan), ys, y_rows, dev.up(pos), dev.up(w), tokens, topk, n,
                  d_a, a_s, d_o, os)
    got = ref.from_type(dev.get(d_o, (tokens, os), ref.np_dtype(ty)), ty)
    assert np.all(got[:, n:] == -3.0)
    terms = np.where(here[..., None], np.where(here, w, 0)[..., None].astype(np.float64) * y[np.where(here, pos, 0)], 0)
    base = np.zeros((tokens, n)) if add is None else np.broadcast_to(a, (tokens, n))
    want = terms.sum(1) + base
    size = np.abs(terms).sum(1) + np.abs(base)
    tol = np.abs(want) * ref.HALF_STEP[ty] + size * (topk + 1) * 2.0 ** -23 + (2.0 ** -25 if ty == F16 else 0)
    assert np.all(np.abs(got[:, :n] - want) <= tol)


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("tokens,topk,experts,width,inner", ((1, 2, 8, 256, 384), (19, 3, 6, 384, 200), (200, 2, 12, 256, 256)))
def test_an_experts_layer(dev, ty, tokens, topk, experts, width, inner):
    """Sort, quantize, gate and up, quantize, down, combine with the residual: each step against
    its formula on what the steps before it gave."""
    rng = np.random.default_rng(tokens + width)
    ids = np.stack([rng.permutation(experts + 2)[:topk] for _ in range(tokens)]).astype(np.uint32)
    w = rng.dirichlet(np.ones(topk), tokens).astype(np.float32)
    x = rng.standard_normal((tokens, width)).astype(np.float32)
    x = ref.from_type(ref.to_type(x, ty), ty)
    P = tokens * topk
    gate, up = DevMat(dev, rng, inner, width, experts), DevMat(dev, rng, inner, width, experts)
    down = DevMat(dev, rng, width, inner, experts)
    ws, ins = wide(width, ty), wide(inner, ty)
    d_x, d_y = up_typed(dev, x, ty, ws), dev.up(np.zeros((P, ws), ref.np_dtype(ty)))
    d_h, d_out = dev.up(np.zeros((P, ins), ref.np_dtype(ty))), dev.up(np.zeros((tokens, ws), ref.np_dtype(ty)))
    d_s, d_f, d_p = (dev.up(np.zeros(m, np.int32)) for m in (experts + 1, P, P))
    xq = hipf8.Rows(dev.up(np.zeros((tokens, wide(width, F32, 8)), np.uint8)), width,
                    dev.up(np.zeros((ref.blocks(width), tokens), np.float32)), tokens, tokens, width)
    hs = -(-inner // 16) * 16
    hq = hipf8.Rows(dev.up(np.zeros((P, hs), np.uint8)), hs, dev.up(np.zeros((ref.blocks(inner), P), np.float32)),
                    P, P, inner)
    hipf8.sort(dev.up(ids), tokens, topk, experts, d_s, d_f, d_p)
    hipf8.quantize(ty, d_x, ws, xq)
    hipf8.group_mul(xq, d_f, d_s, P, gate.mat, up.mat, ty, d_h, ins)
    hipf8.quantize(ty, d_h, ins, hq)
    hipf8.group_mul(hq, None, d_s, P, down.mat, None, ty, d_y, ws)
    hipf8.combine(ty, d_y, ws, P, d_p, dev.up(w), tokens, topk, width, d_x, ws, d_out, ws)
    start, frm, pos = ref.sort(ids, experts)
    rows = start[-1]
    h = ref.from_type(dev.get(d_h, (P, ins), ref.np_dtype(ty)), ty)[:, :inner]
    y = ref.from_type(dev.get(d_y, (P, ws), ref.np_dtype(ty)), ty)
    got = ref.from_type(dev.get(d_out, (tokens, ws), ref.np_dtype(ty)), ty)
    xd, hd = ref.rows_of(*ref.quantize(x)), ref.rows_of(*ref.quantize(h))
    for e in range(experts):
        r = slice(start[e], start[e + 1])
        if r.stop > r.start:
            check_product(h[r], *product(xd[frm[r]], gate.w[e], up.w[e]), ty)
            check_product(y[r], *product(hd[r], down.w[e]), ty)
    assert np.all(y[rows:] == 0)
    terms = np.where((pos >= 0)[..., None], w[..., None].astype(np.float64) * y[np.maximum(pos, 0)], 0)
    want, size = x + terms.sum(1), np.abs(x) + np.abs(terms).sum(1)
    tol = np.abs(want) * ref.HALF_STEP[ty] + size * (topk + 1) * 2.0 ** -23 + (2.0 ** -25 if ty == F16 else 0)
    assert np.all(np.abs(got - want) <= tol)
