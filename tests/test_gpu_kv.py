"""Rotary positions, the paged 4-bit cache and its attention (hip_kv.h) on the
GPU, against numpy in 64 bits (kv_ref.py).

Tolerances.  A rotated value is one rounding off (through fp32 for the 16-bit
types, which can turn a tie: half a step and 2^-24).  Codes and scales are
equal.  An attention output is off by its own rounding and by
  mass * (2 * size * E + F), mass = sum p |v|, size = max_j |scale| sum |q k_j|:
the logits' error times 2 (numerator and sum).  E = 2^-17: a query in two f16
parts is within 2^-22 of itself, and a group's fp32 sum of 32 products with
codes up to 15, against a largest value of 8 in the group, within 2^-24 * 32 *
15 / 8 = 2^-18.1 of its largest term, and as much again for the offset.  F = 2^-19 for exponentials,
probabilities of 22 bits and the sums over cached rows, or 2^-11 where the
probabilities are rounded to f16 (bf16 outputs).  A probability times its row's
value scale is held in f16 parts scaled by a power of two that takes the
largest such product into [2^4, 2^11) (its bound into [2^5, 2^11), an exponent
above); below f16's smallest normal the last part is off by half of 2^-24, which a
code of up to 8 multiplies: n cached rows add n * 2^-25 * 8 / 2^4 = n * 2^-26
times the largest value scale dmax, whatever their probabilities.
Over whole outputs of fp32 the roundings are independent: relative L2 error
within 4e-6, and within 2^-23 of the largest logit's size more: fp32 holds a
logit (its sum, its scaling, its distance to the maximum) to half a step, 2^-24
of it, each time, and a probability moves by as much.
"""
import ctypes as C

import numpy as np
import pytest

import hipkv
import hipmoe
import kv_ref as ref
from kv_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu

TYPES = (F32, F16, BF16)


class Dev:
    """Device memory of one test, freed at its end."""

    def __init__(self):
        self.h, self.p = hipmoe.hip(), []

    def up(self, a):
        self.p.append(self.h.upload(a))
        return self.p[-1]

    def get(self, p, shape, dtype):
        self.h.sync()
        return self.h.download(p, shape, dtype)

    def free(self):
        self.h.sync()
        for p in self.p:
            self.h.free(p)


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.free()


def up_typed(dev, x, ty, stride, fill=7.0):
    """Rows x [T][n] of the type, stride values apart, the gaps filled."""
    T = x.shape[0]
    a = np.full((max(T, 1), stride), fill, np.float32)
    a[:T, :x.shape[1]] = x
    return dev.up(ref.to_type(a, ty))


# --------------------------------------------------------------------------
# rotation
# --------------------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("layout", (hipkv.PAIRS, hipkv.HALVES))
@pytest.mark.parametrize("rows,heads,D,rot,pad", (
    (1, 1, 2, 2, 0), (1, 32, 128, 128, 0), (3, 5, 128, 64, 8), (17, 2, 96, 96, 0),
    (65, 3, 80, 32, 3), (130, 1, 256, 250, 1), (2, 7, 64, 6, 64), (300, 4, 128, 128, 0)))
def test_rope(dev, ty, layout, rows, heads, D, rot, pad):
    rng = np.random.default_rng(rows * 1000 + D)
    x = rng.standard_normal((rows, heads, D)).astype(np.float32)
    pos = rng.integers(-50, 1 << 21, rows).astype(np.int32)
    f, mag = hipkv.rope_freqs(rot, 5e5, hipkv.YARN, 4.0, 8192.0)
    stride = heads * D + pad
    d_x = up_typed(dev, x.reshape(rows, -1), ty, stride)
    d_o = up_typed(dev, np.zeros((rows, heads * D), np.float32), ty, stride + 5, fill=-3.0)
    R = hipkv.Rope(rot, layout, dev.up(f), mag)
    d_pos = dev.up(pos)
    hipkv.rope(R, ty, d_x, stride, d_o, stride + 5, rows, heads, D, d_pos)
    got = ref.from_type(dev.get(d_o, (rows, stride + 5), ref.np_dtype(ty)), ty)
    assert np.all(got[:, heads * D:] == -3.0)
    want = ref.rotate(ref.from_type(ref.to_type(x, ty), ty), pos, f, mag, layout)
    err = np.abs(got[:, :heads * D].reshape(want.shape) - want)
    # positions to 2^21: the angle's own last bit moves a value by 2^-31 of the pair
    tol = np.abs(want) * (ref.HALF_STEP[ty] + 2.0 ** -24) + 2.0 ** -29
    if ty == F16:
        tol += 2.0 ** -25  # results below its smallest normal
    assert np.all(err <= tol), (err / tol).max()
    # in place: the same bits
    hipkv.rope(R, ty, d_x, stride, d_x, stride, rows, heads, D, d_pos)
    again = ref.from_type(dev.get(d_x, (rows, stride), ref.np_dtype(ty)), ty)
    assert np.array_equal(again[:, :heads * D], got[:, :heads * D])
    assert np.all(again[:, heads * D:] == 7.0)


# --------------------------------------------------------------------------
# storing and reading
# --------------------------------------------------------------------------

class Case:
    """Sequences of rows[s] new rows and len[s] rows in all, on shuffled pages
    of a pool of random codes."""

    def __init__(self, dev, rng, rows, lens, page, KH, D, extra_pages=2, slack=0, fill=None):
        self.dev, self.rows, self.lens, self.page, self.KH, self.D = dev, rows, lens, page, KH, D
        need = [-(-max(0, n) // page) for n in lens]
        self.pages = sum(need) + extra_pages
        ids = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(rows), max(need + [1]) + slack), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.pool = ref.Pool(self.pages, page, KH, D)
        if fill is None:
            self.pool.random(rng)
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.T = int(self.start[-1])
        self.d_pool = dev.up(self.pool.bytes)
        self.d_err = dev.up(np.zeros(1, np.uint32))
        self.d_len = dev.up(np.asarray(lens, np.int32))
        self.d_start, self.d_table = dev.up(self.start), dev.up(self.table)
        self.cache = hipkv.Cache(self.d_pool, self.pages, page, KH, D, self.d_err)
        self.batch = hipkv.Batch(len(rows), self.T, max(rows + [0]), max(lens + [1]), self.d_start,
                                 self.d_len, self.d_table, self.table.shape[1])

    def positions(self):
        return np.concatenate([np.arange(m - n, m) for n, m in zip(self.rows, self.lens)]
                              ).astype(np.int32)

    def sequences(self):
        return np.repeat(np.arange(len(self.rows)), self.rows)

    def pool_bytes(self):
        return self.dev.get(self.d_pool, self.pool.bytes.shape, np.uint8)

    def errors(self):
        return int(self.dev.get(self.d_err, (1,), np.uint32)[0])


SHAPES = (
    # rows, lengths, page, KH, D, heads
    ([1], [1], 32, 1, 64, 1),
    ([1, 1, 1], [33, 32, 31], 32, 2, 128, 8),
    ([3, 0, 2, 1], [7, 5, 66, 64], 64, 3, 64, 3),
    ([37, 64, 5], [40, 64, 133], 32, 1, 256, 4),
    ([70, 1, 33], [70, 100, 97], 128, 2, 128, 6),
    ([4, 6], [2, 6], 32, 5, 128, 5),       # two rows at positions below 0
    ([31, 2], [32, 34], 1024, 2, 64, 14),
)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}")
@pytest.mark.parametrize("layout,rot", ((hipkv.PAIRS, 1.0), (hipkv.HALVES, 1.0), (hipkv.HALVES, 0.5),
                                        (hipkv.PAIRS, 0.25), (None, 0)))
def test_append_stores_the_codes_and_keeps_the_rest(dev, ty, shape, layout, rot):
    rows, lens, page, KH, D, H = shape
    rng = np.random.default_rng(sum(rows) + D + ty)
    c = Case(dev, rng, rows, lens, page, KH, D)
    n = int(D * rot)
    # q, k and v as one product's rows, with a gap after them
    x = rng.standard_normal((c.T, H + 2 * KH, D)).astype(np.float32)
    x[:, H:H + KH, ::7] *= 9
    stride = (H + 2 * KH) * D + 16
    d_x = up_typed(dev, x.reshape(c.T, -1), ty, stride)
    x = ref.from_type(ref.to_type(x, ty), ty)
    b, pos, seq = ref.BYTES[ty], c.positions(), c.sequences()
    q, k, v = x[:, :H], x[:, H:H + KH], x[:, H + KH:]
    if layout is None:
        hipkv.append(c.cache, c.batch, ty, d_x + H * D * b, d_x + (H + KH) * D * b, stride)
    else:
        f, mag = hipkv.rope_freqs(n, 1e4)
        R = hipkv.Rope(n, layout, dev.up(f), mag)
        d_q = up_typed(dev, np.zeros((c.T, H * D), np.float32), ty, H * D, fill=0)
        hipkv.append(c.cache, c.batch, ty, d_x + H * D * b, d_x + (H + KH) * D * b, stride, rope=R,
                     q=d_x, q_stride=stride, heads=H, q_out=d_q, q_out_stride=H * D)
        k = ref.rotate(k, pos, f, mag, layout)
        want = ref.rotate(q, pos, f, mag, layout) * (pos >= 0)[:, None, None]
        got = ref.from_type(dev.get(d_q, (c.T, H, D), ref.np_dtype(ty)), ty)
        tol = np.abs(want) * (ref.HALF_STEP[ty] + 2.0 ** -24) + 2.0 ** -25
        assert np.all(np.abs(got - want) <= tol)
    for i in range(c.T):
        if pos[i] >= 0:
            c.pool.store(c.table[seq[i]], pos[i], k[i].astype(np.float32), v[i].astype(np.float32))
    got = c.pool_bytes()
    assert np.array_equal(got, c.pool.bytes), np.argwhere(got != c.pool.bytes)[:5]
    assert c.errors() == 0

    # the values the rows stand for; rows that are not there stay
    d_k, d_v = (up_typed(dev, np.full((c.T, KH * D), 5.0, np.float32), ty, KH * D + 8) for _ in "kv")
    hipkv.read(c.cache, c.batch, ty, d_k, d_v, KH * D + 8)
    for d, which in ((d_k, 0), (d_v, 1)):
        got = dev.get(d, (c.T, KH * D + 8), ref.np_dtype(ty))
        want = np.full((c.T, KH * D + 8), 5.0)
        want[:, KH * D:] = 7.0
        for i in range(c.T):
            if pos[i] >= 0:
                want[i, :KH * D] = c.pool.load(c.table[seq[i]], pos[i])[which].ravel()
        assert np.array_equal(got, ref.to_type(want, ty))


def test_append_in_place_and_with_positions_of_its_own(dev):
    rng = np.random.default_rng(5)
    rows, lens, KH, D, H = [40, 1], [60, 77], 2, 128, 4
    c = Case(dev, rng, rows, lens, 64, KH, D)
    x = rng.standard_normal((c.T, H + 2 * KH, D)).astype(np.float32)
    stride = (H + 2 * KH) * D
    d_x = dev.up(x)
    pos = rng.integers(0, 100000, c.T).astype(np.int32)
    f, mag = hipkv.rope_freqs(D, 1e6, hipkv.NTK, 2.0)
    hipkv.append(c.cache, c.batch, F32, d_x + H * D * 4, d_x + (H + KH) * D * 4, stride,
                 rope=hipkv.Rope(D, hipkv.HALVES, dev.up(f), mag), pos=dev.up(pos), q=d_x,
                 q_stride=stride, heads=H, q_out=d_x, q_out_stride=stride)
    q = ref.rotate(x[:, :H], pos, f, mag, hipkv.HALVES)
    k = ref.rotate(x[:, H:H + KH], pos, f, mag, hipkv.HALVES).astype(np.float32)
    got = dev.get(d_x, x.shape, np.float32)
    assert np.all(np.abs(got[:, :H] - q) <= np.abs(q) * 2.0 ** -23 + 2.0 ** -29)
    assert np.array_equal(got[:, H:], x[:, H:])
    at, seq = c.positions(), c.sequences()
    for i in range(c.T):
        c.pool.store(c.table[seq[i]], at[i], k[i], x[i, H + KH:])
    assert np.array_equal(c.pool_bytes(), c.pool.bytes)


def test_append_of_extreme_values(dev):
    """Zeros, ties of the largest magnitude, exact ties between codes, values
    past f16 scales, below them, infinities and NaN."""
    KH, D, T = 1, 128, 34
    rng = np.random.default_rng(6)
    c = Case(dev, rng, [T], [T], 64, KH, D)
    k = rng.standard_normal((T, KH, D)).astype(np.float32)
    k[0] = 0
    k[1, 0, :2] = (4, -4)
    k[1, 0, 2:] = 0.25                       # d = 0.5 or -0.5: exactly between two codes
    k[2] *= 1e7
    k[3] *= 1e-9
    k[4] *= 1e-42                            # subnormal: no f16 scale is left
    k[5, 0, 3] = np.inf
    k[6, 0, 40] = -np.inf
    k[7, 0, 100] = np.nan
    k[8, 0, :] = -0.0
    k[9] = 3.0
    k[10] = -3.0
    k[11, 0, ::2] = 3e38
    v = k[::-1].copy()
    d_k, d_v = dev.up(k), dev.up(v)
    hipkv.append(c.cache, c.batch, F32, d_k, d_v, KH * D)
    for i in range(T):
        c.pool.store(c.table[0], i, k[i], v[i])
    got, want = c.pool_bytes(), c.pool.bytes
    # NaN groups: any NaN scale, any codes
    for i in range(T):
        pg, t, r = int(c.table[0, i // 64]), i % 64 // 32, i % 32
        for at, x in ((32 * D + 2 * (r * 4 + 3), k[i, 0, 96:]), (34 * D + 2 * r, v[i, 0])):
            if np.isnan(x).any():
                assert np.isnan(got[pg, 0, t, at:at + 2].view(np.float16)[0])
    P = ref.Pool(c.pages, 64, KH, D)
    P.bytes = got
    for i in range(T):
        for a, b in zip(P.load(c.table[0], i), c.pool.load(c.table[0], i)):
            assert np.array_equal(a, b, equal_nan=True), i


def test_offsets_past_32_bits(dev):
    """Rows on pages beyond 4 GiB of the pool."""
    KH, D, page = 16, 128, 1024
    size = hipkv.page_bytes(page, KH, D)
    pages = (1 << 32) // size + 3
    h = dev.h
    pool = h.malloc(pages * size)
    dev.p.append(pool)
    rng = np.random.default_rng(7)
    rows, lens = [33, 2], [1030, 31]
    k, v = rng.standard_normal((2, 35, KH, D)).astype(np.float32)
    table = np.array([[pages - 2, pages - 1], [pages - 3, 0]], np.int32)
    ref_pool = ref.Pool(3, page, KH, D, fill=0)
    h.copy_in(pool + (pages - 3) * size, ref_pool.bytes)
    cache = hipkv.Cache(pool, pages, page, KH, D)
    batch = hipkv.Batch(2, 35, 33, 1030, dev.up(np.array([0, 33, 35], np.int32)),
                        dev.up(np.array(lens, np.int32)), dev.up(table), 2)
    hipkv.append(cache, batch, F32, dev.up(k), dev.up(v), KH * D)
    for i, (s, p) in enumerate([(0, p) for p in range(997, 1030)] + [(1, 29), (1, 30)]):
        ref_pool.store(table[s] - (pages - 3), p, k[i], v[i])
    got = dev.get(pool + (pages - 3) * size, ref_pool.bytes.shape, np.uint8)
    assert np.array_equal(got, ref_pool.bytes)
    # the attention reads them: one row that sees the last 34 rows
    q = rng.standard_normal((35, KH, D)).astype(np.float32)
    d_q, d_o = dev.up(q), dev.up(np.zeros_like(q))
    ws = hipkv.attn_ws(cache, batch, KH)
    d_ws = h.malloc(ws)
    dev.p.append(d_ws)
    hipkv.attn(cache, batch, F32, d_q, KH * D, KH, d_o, KH * D, 0.09, 33, d_ws, ws)
    kk, vv = (np.stack(x) for x in zip(*[ref_pool.load(table[0] - (pages - 3), p)
                                         for p in range(1030)]))
    want, mass, _ = ref.attend(q[32].astype(np.float64), kk, vv, 1029, 0.09, 33)
    got = dev.get(d_o, q.shape, np.float32)[32]
    assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def check_attention(dev, c, H, ty, window, rng, scale=None, qscale=1.0, pad=0, check=None):
    KH, D = c.KH, c.D
    scale = D ** -0.5 if scale is None else scale
    q = (qscale * rng.standard_normal((c.T, H, D))).astype(np.float32)
    d_q = up_typed(dev, q.reshape(c.T, -1), ty, H * D + pad)
    d_o = up_typed(dev, np.full((c.T + 1, H * D), 3.0, np.float32), ty, H * D + 2 * pad, fill=3.0)
    q = ref.from_type(ref.to_type(q, ty), ty)
    ws = hipkv.attn_ws(c.cache, c.batch, H)
    d_ws = dev.h.malloc(ws)
    dev.p.append(d_ws)
    hipkv.attn(c.cache, c.batch, ty, d_q, H * D + pad, H, d_o, H * D + 2 * pad, scale, window,
               d_ws if ws else None, ws)
    got = ref.from_type(dev.get(d_o, (c.T + 1, H * D + 2 * pad), ref.np_dtype(ty)), ty)
    assert np.all(got[:, H * D:] == 3.0) and np.all(got[c.T] == 3.0)
    got = got[:c.T, :H * D].reshape(c.T, H, D)
    want, mass, size = np.zeros_like(got), np.zeros_like(got), np.zeros((c.T, H))
    pos, seq = c.positions(), c.sequences()
    rows = {}
    for s, m in enumerate(c.lens):
        if m > 0:
            rows[s] = [np.stack(x) for x in zip(*[c.pool.load(c.table[s], p) for p in range(m)])]
    for i in (range(c.T) if check is None else check):
        if seq[i] in rows:
            want[i], mass[i], size[i] = ref.attend(q[i], *rows[seq[i]], pos[i], scale, window)
    if check is not None:
        pick = np.asarray(check)
        got, want, mass, size = got[pick], want[pick], mass[pick], size[pick]
    # what infinite scales make of a row is not finite
    bad = ~np.isfinite(want)
    assert np.all(~np.isfinite(got[bad]))
    got, want, mass = (np.where(bad, 0, a) for a in (got, want, mass))
    F = 2.0 ** -11 if ty == BF16 else 2.0 ** -19
    d = np.abs(c.pool.bytes[..., 34 * D:].view(np.float16).astype(np.float64))
    dmax = d[np.isfinite(d)].max()
    tol = np.abs(want) * ref.HALF_STEP[ty] + mass * (2 * size[..., None] * 2.0 ** -17 + F)
    tol += max(c.lens) * 2.0 ** -26 * dmax
    if ty == F16:
        tol += 2.0 ** -25
    err = np.abs(got - want)
    assert np.all(err <= tol), (err / np.maximum(tol, 1e-300)).max()
    if ty == F32:
        assert np.linalg.norm(got - want) <= (4e-6 + 2.0 ** -23 * size.max()) * np.linalg.norm(want)
    return got


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}")
@pytest.mark.parametrize("window", (0, 1, 33))
def test_attention(dev, ty, shape, window):
    rows, lens, page, KH, D, H = shape
    rng = np.random.default_rng(sum(lens) + D + ty)
    c = Case(dev, rng, rows, lens, page, KH, D, slack=1)
    check_attention(dev, c, H, ty, window, rng, pad=8)
    assert c.errors() == 0


@pytest.mark.parametrize("ty,D,KH,H,rows,lens,window", (
    (F32, 128, 2, 8, [1] * 5, [700, 1, 513, 2048, 129], 0),   # split along the cache
    (F32, 128, 1, 7, [3, 2], [1500, 900], 200),
    (F16, 64, 2, 4, [1, 1], [3000, 40], 0),
    (BF16, 256, 1, 8, [2], [1111], 500),
    (F32, 64, 1, 1, [130], [400], 0),                         # row tiles of one head
    (BF16, 128, 1, 3, [150, 7], [150, 600], 0),
    (F32, 256, 1, 2, [70], [290], 65),
    (F16, 128, 2, 32, [33, 21], [33, 300], 0),
))
def test_attention_long(dev, ty, D, KH, H, rows, lens, window):
    rng = np.random.default_rng(sum(lens))
    c = Case(dev, rng, rows, lens, 64, KH, D)
    check_attention(dev, c, H, ty, window, rng, qscale=2.0)


@pytest.mark.parametrize("ty,D,KH,H,rows,lens,page,window", (
    (F32, 64, 16, 16, [270] * 4, [270, 300, 333, 1000], 32, 0),
    (F16, 128, 4, 16, [130] * 9, [130, 131, 160, 700, 130, 65, 10, 400, 223], 64, 0),
    (BF16, 128, 16, 32, [131] * 4, [131, 290, 500, 140], 32, 100),
    (F32, 256, 8, 16, [140] * 8, [140, 141, 200, 300, 139, 150, 160, 170], 64, 0),
    (F32, 128, 8, 32, [530] * 4, [530, 531, 900, 300], 256, 0),
    (BF16, 128, 16, 64, [515, 20, 0, 511], [700, 20, 0, 1300], 128, 300),
    (F16, 64, 16, 48, [700, 701], [700, 1111], 64, 0),
    (BF16, 64, 16, 16, [1025] * 4, [1025, 1030, 1100, 1500], 64, 50),
))
def test_attention_of_many_rows(dev, ty, D, KH, H, rows, lens, page, window):
    """Calls with enough query rows to fill the chip, against a sample of them:
    the first and last rows of sequences and of tiles, and others."""
    rng = np.random.default_rng(sum(lens))
    c = Case(dev, rng, rows, lens, page, KH, D)
    start = c.start[:-1]
    at = np.concatenate([start, start + 1, start + 15, start + 16, start + 64, c.start[1:] - 1,
                         rng.integers(0, c.T, 6)])
    check = sorted({int(i) for i in at if 0 <= i < c.T})
    check_attention(dev, c, H, ty, window, rng, qscale=2.0, pad=8, check=check)


@pytest.mark.parametrize("window", (0, 45))
@pytest.mark.parametrize("ty,D,KH,G,rows,lens", tuple(
    # one to eight query rows of a kv head, in columns of two and of four or alone
    (ty, D, 2, G, rows, lens)
    for ty, D in ((F32, 128), (F16, 256), (BF16, 64), (BF16, 128), (F32, 256), (F16, 64))
    for G, rows, lens in ((1, [1] * 3, [1, 33, 300]), (2, [2, 1], [70, 31]), (3, [1], [95]), (4, [1] * 2, [640, 32]),
                          (5, [1], [200]), (1, [4, 3, 1], [4, 100, 67]), (2, [3, 2], [129, 2]), (8, [1], [257]),
                          (7, [1], [64]), (1, [9, 5, 0], [40, 77, 0]))) + (
    # longer than a workgroup's whole cache, in pieces
    (F32, 128, 1, 4, [1], [1100]), (BF16, 128, 2, 1, [3], [2500]), (F16, 64, 1, 8, [1], [1300]),
    (F32, 256, 1, 3, [1], [700]), (BF16, 256, 1, 6, [1], [700])))
def test_attention_of_few_rows(dev, ty, D, KH, G, rows, lens, window):
    rng = np.random.default_rng(sum(lens) + G)
    c = Case(dev, rng, rows, lens, 32, KH, D)
    check_attention(dev, c, KH * G, ty, window, rng, qscale=2.0, pad=8)
    assert c.errors() == 0


@pytest.mark.parametrize("ty", (F16, BF16))
@pytest.mark.parametrize("many", (False, True))
@pytest.mark.parametrize("size,qscale", ((1e-5, 1.0), (1e-3, 30.0), (40.0, 1e-3), (1.0, 1.0)))
def test_attention_sizes_in_16_bits(dev, ty, many, size, qscale):
    """Scales down to f16's subnormals, for few rows and in tiles of 32."""
    rng = np.random.default_rng(14)
    rows, lens, KH, H = ([270] * 4, [270, 300, 333, 400], 16, 32) if many else ([2, 1], [200, 90], 2, 4)
    c = Case(dev, rng, rows, lens, 32, KH, 128)
    half = c.pool.bytes[..., 34 * 128 - 256:].view(np.float16)
    half[..., :128] = half[..., :128] / np.float16(0.25) * np.float16(size)
    check_attention(dev, c_upload(c), H, ty, 0, rng, qscale=qscale,
                    check=sorted({0, 1, 100, 269, 270, 700, c.T - 1} & set(range(c.T))) if many else None)


@pytest.mark.parametrize("qscale,scale", ((1e-20, 1.0), (1e-38, 1.0), (30.0, None), (1e6, 1e-7), (1.0, 0.0),
                                          (1.0, -0.1)))
def test_attention_sizes_of_queries(dev, qscale, scale):
    rng = np.random.default_rng(11)
    c = Case(dev, rng, [2, 1], [200, 90], 32, 2, 128)
    check_attention(dev, c, 4, F32, 0, rng, qscale=qscale, scale=scale)


@pytest.mark.parametrize("size", (1e-6, 1e-3, 300.0, 40000.0, 60000.0))
@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_attention_sizes_of_values(dev, size):
    """Value scales from f16's subnormals to its largest (and past it: 1.5 *
    60000), and rows whose scales differ by the whole range."""
    rng = np.random.default_rng(12)
    c = Case(dev, rng, [2, 1], [200, 90], 32, 2, 128)
    half = c.pool.bytes[..., 34 * 128:].view(np.float16)
    half[...] = half / np.float16(0.25) * np.float16(size)
    check_attention(dev, c_upload(c), 4, F32, 0, rng)
    half[...] = np.where(rng.random(half.shape) < 0.02, np.float16(size), np.float16(1e-5))
    check_attention(dev, c_upload(c), 4, F32, 0, rng)


def c_upload(c):
    c.dev.h.sync()
    c.dev.h.copy_in(c.d_pool, c.pool.bytes)
    return c


def test_masked_rows_do_not_reach_the_output(dev):
    """NaN and infinite scales behind the length, before the window and in the
    later rows that a causal row must not see."""
    rng = np.random.default_rng(13)
    KH, D = 2, 128
    c = Case(dev, rng, [5, 3], [70, 45], 32, KH, D)
    bad = np.array([np.nan, np.inf, -np.inf, 65504], np.float16)

    def spoil(table, p):
        tile = c.pool.bytes[int(table[p // 32]), :, 0]
        half = tile[:, 32 * D:].view(np.float16)
        half[:, p % 32 * 4:p % 32 * 4 + 4] = rng.choice(bad, (KH, 4))
        half[:, D + p % 32] = rng.choice(bad, KH)

    for s, m in enumerate(c.lens):
        for p in range(m, -(-m // 32) * 32):
            spoil(c.table[s], p)
    check_attention(dev, c_upload(c), 4, F32, 0, rng)
    # rows 0 .. 36 and 0 .. 21 lie before every window
    for p in range(37):
        spoil(c.table[0], p)
    for p in range(14):
        spoil(c.table[1], p)
    check_attention(dev, c_upload(c), 4, F32, 29, rng)
    # the last row of each sequence is seen by its own query alone
    spoil(c.table[0], 69)
    spoil(c.table[1], 44)
    check_attention(dev, c_upload(c), 4, F32, 29, rng, check=[0, 1, 2, 3, 5, 6])


def test_nan_and_infinite_queries_stay_in_their_row(dev):
    rng = np.random.default_rng(14)
    c = Case(dev, rng, [6], [100], 32, 1, 128)
    H, D = 4, 128
    q = rng.standard_normal((6, H, D)).astype(np.float32)
    q[1, 2, 5], q[3, 0, 7], q[4, 1, 9] = np.nan, np.inf, -np.inf
    ws = hipkv.attn_ws(c.cache, c.batch, H)
    d_q, d_o, d_ws = dev.up(q), dev.up(np.zeros_like(q)), dev.h.malloc(ws)
    dev.p.append(d_ws)
    hipkv.attn(c.cache, c.batch, F32, d_q, H * D, H, d_o, H * D, 0.1, 0, d_ws, ws)
    got = dev.get(d_o, q.shape, np.float32)
    k, v = (np.stack(x) for x in zip(*[c.pool.load(c.table[0], p) for p in range(100)]))
    for i in range(6):
        want = ref.attend(np.nan_to_num(q[i].astype(np.float64)), k, v, 94 + i, 0.1, 0)[0]
        for h in range(H):
            if (i, h) in ((1, 2), (3, 0), (4, 1)):
                assert np.isnan(got[i, h]).all()
            else:
                assert np.linalg.norm(got[i, h] - want[h]) <= 1e-5 * np.linalg.norm(want[h])


def test_padded_batch_and_uniform_rows(dev):
    """Sequences without rows behind the last one, and row_start NULL."""
    rng = np.random.default_rng(15)
    c = Case(dev, rng, [2, 3, 0, 0], [50, 40, 0, 0], 32, 2, 64, slack=3)
    check_attention(dev, c, 4, F32, 0, rng)
    c = Case(dev, rng, [2, 2, 2], [50, 40, 2], 32, 2, 64)
    c.batch.row_start = None
    check_attention(dev, c, 4, F16, 0, rng)
    c = Case(dev, rng, [0, 0], [5, 5], 32, 2, 64)
    assert hipkv.attn_ws(c.cache, c.batch, 2) == 0
    hipkv.attn(c.cache, c.batch, F32, None, 0, 2, None, 0, 1.0)
    hipkv.append(c.cache, c.batch, F32, None, None, 0)
    hipkv.read(c.cache, c.batch, F32, None, None, 0)


def test_bad_pages_and_bounds_are_reported(dev):
    """Page ids outside the pool, and lengths and first rows outside the
    batch's bounds: nothing outside is touched, the rest is done, and the
    error word says so."""
    rng = np.random.default_rng(16)
    KH, D, H = 1, 64, 2
    for bad in (-1, 1 << 30, None):
        c = Case(dev, rng, [2, 2], [70, 40], 32, KH, D)
        table = c.table.copy()
        table[0, 2] = c.pages if bad is None else bad  # the page of both new rows
        d_table = dev.up(table)
        batch = hipkv.Batch(2, 4, 2, 70, c.d_start, c.d_len, d_table, table.shape[1])
        k, v = rng.standard_normal((2, 4, KH, D)).astype(np.float32)
        d_k, d_v = dev.up(k), dev.up(v)
        hipkv.append(c.cache, batch, F32, d_k, d_v, KH * D)
        for i, p in ((2, 38), (3, 39)):
            c.pool.store(c.table[1], p, k[i], v[i])
        assert np.array_equal(c.pool_bytes(), c.pool.bytes)
        assert c.errors() == hipkv.ERR_PAGE
        dev.h.copy_in(c.d_err, np.zeros(1, np.uint32))
        hipkv.read(c.cache, batch, F32, d_k, d_v, KH * D)
        got = dev.get(d_v, v.shape, np.float32)
        assert np.array_equal(got[:2], v[:2]) and c.errors() == hipkv.ERR_PAGE
        # the attention leaves the page out: rows 0 .. 63 of the first sequence
        dev.h.copy_in(c.d_err, np.zeros(1, np.uint32))
        q = rng.standard_normal((4, H, D)).astype(np.float32)
        ws = hipkv.attn_ws(c.cache, batch, H)
        d_q, d_o, d_ws = dev.up(q), dev.up(np.zeros_like(q)), dev.h.malloc(ws)
        dev.p.append(d_ws)
        hipkv.attn(c.cache, batch, F32, d_q, H * D, H, d_o, H * D, 0.125, 0, d_ws, ws)
        got = dev.get(d_o, q.shape, np.float32)
        kk, vv = (np.stack(x) for x in zip(*[c.pool.load(c.table[0], p) for p in range(64)]))
        for i in range(2):
            want = ref.attend(q[i].astype(np.float64), kk, vv, 63, 0.125, 0)[0]
            assert np.linalg.norm(got[i] - want) <= 1e-5 * np.linalg.norm(want)
        assert c.errors() == hipkv.ERR_PAGE

    # bounds: more rows than max_rows, a length past max_len, rows out of order
    c = Case(dev, rng, [3, 2], [33, 40], 32, KH, D)
    for what in ("rows", "len", "order"):
        dev.h.copy_in(c.d_err, np.zeros(1, np.uint32))
        batch = hipkv.Batch(2, 5, 3, 40, c.d_start, c.d_len, c.d_table, c.table.shape[1])
        if what == "rows":
            batch.max_rows = 2
        elif what == "len":
            batch.max_len = 34
        else:
            batch.row_start = dev.up(np.array([2, 9, -4], np.int32))
        q = np.zeros((5, H, D), np.float32)
        d_q, d_o = dev.up(q), dev.up(q)
        ws = hipkv.attn_ws(c.cache, batch, H)
        d_ws = dev.h.malloc(ws)
        dev.p.append(d_ws)
        hipkv.attn(c.cache, batch, F32, d_q, H * D, H, d_o, H * D, 0.1, 0, d_ws, ws)
        assert c.errors() == hipkv.ERR_BATCH, what
        hipkv.read(c.cache, batch, F32, d_q, d_o, H * D)
        assert c.errors() == hipkv.ERR_BATCH, what


def test_output_may_be_the_queries(dev):
    rng = np.random.default_rng(17)
    H, D = 4, 128
    for lens in ([40, 33], [900, 700]):
        c = Case(dev, rng, [3, 2], lens, 32, 2, D)
        q = rng.standard_normal((5, H, D)).astype(np.float32)
        ws = hipkv.attn_ws(c.cache, c.batch, H)
        d_q, d_o, d_ws = dev.up(q), dev.up(np.zeros_like(q)), dev.h.malloc(ws)
        dev.p.append(d_ws)
        hipkv.attn(c.cache, c.batch, F32, d_q, H * D, H, d_o, H * D, 0.1, 0, d_ws, ws)
        hipkv.attn(c.cache, c.batch, F32, d_q, H * D, H, d_q, H * D, 0.1, 0, d_ws, ws)
        assert np.array_equal(dev.get(d_q, q.shape, np.float32), dev.get(d_o, q.shape, np.float32))


@pytest.mark.parametrize("window", (0, 70))
@pytest.mark.parametrize("ty,D,KH,G,nseq", ((F32, 128, 8, 4, 64), (BF16, 128, 8, 1, 64), (F16, 64, 16, 8, 40),
                                            (F32, 64, 16, 1, 130), (BF16, 256, 8, 4, 64), (F32, 256, 4, 6, 128),
                                            (F32, 128, 8, 8, 64), (BF16, 128, 2, 7, 256)))
def test_many_caches_in_shares(dev, ty, D, KH, G, nseq, window):
    """A batch whose bound is far above its lengths: shares of a few tiles that begin
    and end inside sequences, of every length, without rows, or before their start."""
    rng = np.random.default_rng(nseq + D + G)
    lens = [int(n) for n in rng.integers(1, 200, nseq)]
    rows = [int(n) for n in rng.integers(1, max(1, 16 // G) + 1, nseq)]
    rows[3], lens[3], rows[nseq - 1], lens[nseq - 1] = 0, 50, 0, 0
    lens[0], lens[7], lens[20] = 900, 0, 32
    rows[0], rows[7] = 1, 1
    c = Case(dev, rng, rows, lens, 32, KH, D, slack=16384 // 32)
    c.batch.max_len = 16384
    at = [int(i) for i in c.start[:-1]]
    check = sorted({i for i in at if i < c.T} & set(at[:10] + at[-6:] + [at[int(k)] for k in rng.integers(0, nseq, 20)]))
    check_attention(dev, c, KH * G, ty, window, rng, qscale=2.0, pad=8, check=check)
    assert c.errors() == 0
    # a bad page and a bad length in one sequence each
    table, length = c.table.copy(), np.asarray(lens, np.int32)
    table[0, 1], length[5] = c.pages, 20000
    b = hipkv.Batch(nseq, c.T, max(rows), 16384, c.d_start, dev.up(length), dev.up(table), table.shape[1])
    q = rng.standard_normal((c.T, KH * G, D)).astype(np.float32)
    d_q, d_o = dev.up(ref.to_type(q, ty)), dev.up(np.zeros(q.shape, ref.np_dtype(ty)))
    ws = hipkv.attn_ws(c.cache, b, KH * G)
    d_ws = dev.h.malloc(ws)
    dev.p.append(d_ws)
    hipkv.attn(c.cache, b, ty, d_q, KH * G * D, KH * G, d_o, KH * G * D, 0.1, 0, d_ws, ws)
    assert c.errors() == hipkv.ERR_PAGE | hipkv.ERR_BATCH


@pytest.mark.parametrize("ty,H,KH,D,rows,lens", (
    (F32, 3, 1, 128, [1], [90]), (BF16, 8, 1, 64, [1, 1], [70, 64]),          # slots
    (F16, 4, 4, 256, [9], [300]), (F32, 16, 16, 128, [300] * 2, [300, 1100]),  # tiles of 16
    (BF16, 32, 16, 128, [270] * 4, [270, 1100, 300, 290]),                    # of 32
    (F32, 32, 32, 64, [200] * 3, [1030, 200, 450])))
def test_every_form_in_place_and_without_a_page(dev, ty, H, KH, D, rows, lens):
    """Outputs over the queries are those beside them, and a page outside the pool is
    left out of the sum and reported, whatever takes the call."""
    rng = np.random.default_rng(sum(lens) + D)
    c = Case(dev, rng, rows, lens, 32, KH, D)
    q = rng.standard_normal((c.T, H, D)).astype(np.float32)
    shape, np_ty = q.shape, ref.np_dtype(ty)
    ws = hipkv.attn_ws(c.cache, c.batch, H)
    d_ws = dev.h.malloc(max(ws, 16))
    dev.p.append(d_ws)

    def run(table, in_place):
        d_q = dev.up(ref.to_type(q, ty))
        d_o = d_q if in_place else dev.up(np.zeros(shape, np_ty))
        b = hipkv.Batch(len(rows), c.T, max(rows), max(lens), c.d_start, c.d_len, dev.up(table),
                        table.shape[1])
        hipkv.attn(c.cache, b, ty, d_q, H * D, H, d_o, H * D, D ** -0.5, 0, d_ws, ws)
        return dev.get(d_o, shape, np_ty)

    want = run(c.table, False)
    assert np.array_equal(run(c.table, True), want) and c.errors() == 0
    for bad in (-1, c.pages, 1 << 30):
        table = c.table.copy()
        table[0, 1] = bad  # rows 32 .. 63 of the first sequence
        got = ref.from_type(run(table, False), ty)
        assert c.errors() == hipkv.ERR_PAGE
        dev.h.copy_in(c.d_err, np.zeros(1, np.uint32))
        n = rows[0]
        assert np.array_equal(got[n:], ref.from_type(want, ty)[n:])
        kk, vv = (np.stack(x) for x in zip(*[c.pool.load(c.table[0], p) for p in range(lens[0])]))
        x = ref.from_type(ref.to_type(q, ty), ty)
        for i in sorted({0, n // 2, n - 1}):
            p = lens[0] - n + i
            keep = [j for j in range(p + 1) if not 32 <= j < 64]
            w = ref.attend(x[i], kk[keep], vv[keep], len(keep) - 1, D ** -0.5, 0)[0]
            assert np.linalg.norm(got[i] - w) <= max(1e-5, 2 * ref.HALF_STEP[ty]) * np.linalg.norm(w), i


@pytest.mark.parametrize("ty,D", ((F32, 128), (BF16, 128), (F16, 64), (BF16, 64)))
@pytest.mark.parametrize("rows", (64, 65, 95, 97))
def test_rows_beside_the_tiles_of_32(dev, ty, D, rows):
    """Rows that end beside a tile's end, lengths beside the cache's tiles, one row
    and none in the same call."""
    rng = np.random.default_rng(rows + D)
    all_rows = [rows, 1, rows, 0, rows, 2, rows, rows]
    c = Case(dev, rng, all_rows, [1024, 1, rows, 0, rows + 31, 33, rows + 32, rows + 1], 32, 32, D)
    at = c.start[[0, 2, 4, 6, 7]]
    check = sorted({int(i) for k in (0, 31, 32, 63, rows - 1) for i in at + k} | {rows, int(c.start[5])})
    check_attention(dev, c, 32, ty, 0, rng, qscale=2.0, check=check)


# --------------------------------------------------------------------------
# the operators together, as a decode loop runs them
# --------------------------------------------------------------------------

def test_a_decode_loop_from_one_captured_graph(dev):
    """Prompts of different lengths, then steps replayed from one graph (append
    with both rotations, attention) with the lengths advanced in between:
    each step equals the same calls made eagerly, bit for bit, and numpy over the
    rows that the cache holds."""
    rng = np.random.default_rng(18)
    h, KH, H, D, page = dev.h, 2, 8, 128, 32
    prompts, steps = [50, 31, 1], 6
    S, scale = len(prompts), 0.1
    c = Case(dev, rng, prompts, [n + steps for n in prompts], page, KH, D)
    stride = (H + 2 * KH) * D
    f, mag = hipkv.rope_freqs(D, 1e6)
    R = hipkv.Rope(D, hipkv.PAIRS, dev.up(f), mag)
    st = h.stream()

    def enqueue(cache, batch, d_x, d_q, d_o, d_ws, ws, stream):
        hipkv.append(cache, batch, F32, d_x + H * D * 4, d_x + (H + KH) * D * 4, stride, rope=R, q=d_x,
                     q_stride=stride, heads=H, q_out=d_q, q_out_stride=H * D, stream=stream)
        hipkv.attn(cache, batch, F32, d_q, H * D, H, d_o, H * D, scale, 0, d_ws, ws, stream=stream)

    def buffers(rows, batch):
        d_x = dev.up(np.zeros((rows, stride), np.float32))
        d_q, d_o = (dev.up(np.zeros((rows, H * D), np.float32)) for _ in "qo")
        ws = hipkv.attn_ws(c.cache, batch, H)
        d_ws = h.malloc(ws)
        dev.p.append(d_ws)
        return d_x, d_q, d_o, d_ws, ws

    most = max(prompts) + steps
    lens = np.asarray(prompts, np.int32)
    d_len = dev.up(lens)
    first = hipkv.Batch(S, c.T, max(prompts), most, c.d_start, d_len, c.d_table, c.table.shape[1])
    b = buffers(c.T, first)
    x0 = rng.standard_normal((c.T, H + 2 * KH, D)).astype(np.float32)
    h.copy_in(b[0], x0)
    enqueue(c.cache, first, *b, st)
    h.stream_sync(st)
    twin = hipkv.Cache(dev.up(c.pool_bytes()), c.pages, page, KH, D)

    step = hipkv.Batch(S, S, 1, most, None, d_len, c.d_table, c.table.shape[1])
    g, e = buffers(S, step), buffers(S, step)
    h.begin_capture(st)
    enqueue(c.cache, step, *g, st)
    graph = h.end_capture(st)
    for i in range(steps):
        lens = lens + 1
        x = rng.standard_normal((S, H + 2 * KH, D)).astype(np.float32)
        h.copy_in(d_len, lens)
        h.copy_in(g[0], x)
        h.copy_in(e[0], x)
        h.graph_launch(graph, st)
        h.stream_sync(st)
        enqueue(twin, step, *e, None)
        got, eager = dev.get(g[2], (S, H, D), np.float32), dev.get(e[2], (S, H, D), np.float32)
        assert np.array_equal(got, eager), i
        P = ref.Pool(c.pages, page, KH, D)
        P.bytes = c.pool_bytes()
        q = ref.rotate(x[:, :H], lens - 1, f, mag, hipkv.PAIRS)
        for s in range(S):
            k, v = (np.stack(y) for y in zip(*[P.load(c.table[s], p) for p in range(lens[s])]))
            want = ref.attend(q[s], k, v, lens[s] - 1, scale, 0)[0]
            assert np.linalg.norm(got[s] - want) <= 4e-6 * np.linalg.norm(want)
            # the newest row is the one just stored: within half a step of the row
            kk = ref.rotate(x[s:s + 1, H:H + KH], lens[s:s + 1] - 1, f, mag, hipkv.PAIRS)[0]
            top = np.abs(kk).reshape(KH, -1, 32).max(-1).repeat(32, -1)
            assert np.all(np.abs(k[-1] - kk) <= top / 8 * 1.01)
    h.h.hipGraphExecDestroy(graph)
    h.h.hipStreamDestroy(st)


def test_two_calls_at_once(dev):
    """Two streams read one cache, each call with its own workspace."""
    rng = np.random.default_rng(19)
    h, H, D = dev.h, 8, 128
    c = Case(dev, rng, [1, 1], [3000, 2900], 64, 2, D)
    ws = hipkv.attn_ws(c.cache, c.batch, H)
    q = rng.standard_normal((2, 2, H, D)).astype(np.float32)
    calls = []
    for i in range(2):
        d_ws = h.malloc(ws)
        dev.p.append(d_ws)
        calls.append((dev.up(q[i]), dev.up(np.zeros_like(q[i])), dev.up(np.zeros_like(q[i])), d_ws,
                      h.stream()))
    for d_q, d_o, _, d_ws, st in calls * 3:
        hipkv.attn(c.cache, c.batch, F32, d_q, H * D, H, d_o, H * D, 0.1, 0, d_ws, ws, stream=st)
    h.sync()
    for d_q, d_o, d_one, d_ws, st in calls:
        hipkv.attn(c.cache, c.batch, F32, d_q, H * D, H, d_one, H * D, 0.1, 0, d_ws, ws)
        assert np.array_equal(dev.get(d_o, q[0].shape, np.float32),
                              dev.get(d_one, q[0].shape, np.float32))
        h.h.hipStreamDestroy(st)
