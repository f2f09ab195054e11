"""The calls of hip_kv.h at the ends of their ranges: value scales that differ by
the whole range of f16, long caches of one sign, workgroups of several rows and
heads, lengths of nothing and near the largest, workspaces' ends.

Tolerances.  As in test_gpu_kv.py where values are compared one by one.  Whole
outputs are compared by their relative L2 error, to which a 16-bit type's own
rounding adds at most HALF_STEP (and 0.4 of it, 1 / sqrt(3) at a value's lower end and
half of that at its upper, where values are spread evenly): a kernel that is within
HALF_STEP altogether has erred by less than its rounding.  For fp32, see FP32.
"""
import numpy as np
import pytest

import hipkv
import kv_ref as ref
from kv_ref import BF16, F16, F32
from test_gpu_kv import TYPES, Case, c_upload, dev, up_typed  # noqa: F401  (dev: a fixture)

pytestmark = pytest.mark.gpu

# fp32, logits in powers of two within 16 of the reference 2^9 below the largest: a
# logit's last sum is rounded by up to 2^-21, rms 2^-21 / sqrt(3), times ln 2: 1.9e-7 of a
# probability; a probability in two f16 parts by up to 2^-22, rms 1.4e-7; a query's values
# by as much, of a logit of 1 or 2; exponentials, the sums of 16 or 32 tiles a wave and
# the quotient about 1e-7 together: 3.2e-7, all of them independent from row to row.  Three
# times that; codes as subnormals would be 3e-6.
FP32 = 1e-6
WHOLE = {F32: FP32, F16: ref.HALF_STEP[F16], BF16: ref.HALF_STEP[BF16]}


def rows_of(c, s, n):
    """(k, v) [n][KH][D] float64, the first n cached rows of sequence s."""
    P, D, KH = c.pool, c.D, c.KH
    t = np.arange(-(-n // 32))
    tiles = P.bytes[c.table[s][t * 32 // c.page], :, t % (c.page // 32)]  # [tiles][KH][bytes]
    words = np.ascontiguousarray(tiles).view(np.uint32)
    half = np.ascontiguousarray(tiles[..., 32 * D:]).view(np.float16).astype(np.float64)
    k, v = np.empty((2, len(t), 32, KH, D))
    for r in range(32):
        w, b = P._key_words(r)
        k[:, r] = (P._get(words.transpose(2, 0, 1), w, b[:, None, None]) - 8).transpose(1, 2, 0)
        k[:, r] *= np.repeat(half[..., r * (D // 32):(r + 1) * (D // 32)], 32, -1)
        w, b = P._value_words(r)
        v[:, r] = (P._get(words.transpose(2, 0, 1), w, b[:, None, None]) - 8).transpose(1, 2, 0)
        v[:, r] *= half[..., D + r, None]
    return k.reshape(-1, KH, D)[:n], v.reshape(-1, KH, D)[:n]


def attention(dev, c, H, ty, q, scale, window=0, batch=None, in_place=False):
    """hip_kv_attn_dev of q [T][H][D] (its type's values), with a pattern behind the
    workspace that has to stay."""
    b = batch or c.batch
    d_q = dev.up(ref.to_type(q, ty))
    d_o = d_q if in_place else dev.up(np.zeros(q.shape, ref.np_dtype(ty)))
    ws = hipkv.attn_ws(c.cache, b, H)
    d_ws = dev.up(np.full(ws + 4096, 0xa5, np.uint8))
    hipkv.attn(c.cache, b, ty, d_q, H * c.D, H, d_o, H * c.D, scale, window, d_ws, ws)
    got = ref.from_type(dev.get(d_o, q.shape, ref.np_dtype(ty)), ty)
    assert np.all(dev.get(d_ws, (ws + 4096,), np.uint8)[ws:] == 0xa5)
    return got


def typed(x, ty):
    return ref.from_type(ref.to_type(x, ty), ty)


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


# how a call is taken: (rows, lengths, KH, H)
FORMS = {"slots of 4": ([1], [200], 2, 6), "slots of 2": ([2, 1], [150, 77], 2, 6),
         "16 rows": ([9], [170], 1, 3), "pieces": ([1], [2200], 1, 4),
         "32 rows": ([270] * 4, [270, 300, 400, 290], 16, 32),
         "shares": ([1] * 64, [100] * 64, 8, 16)}


def form_case(dev, rng, form, D):
    rows, lens, KH, H = FORMS[form]
    c = Case(dev, rng, rows, lens, 32, KH, D, slack=512 if form == "shares" else 0)
    if form == "shares":
        c.batch.max_len = 16384
    return c, H


def check_rows(c, most=6):
    """Some rows of the call, the first and the last of sequences among them."""
    at = sorted({int(i) for s in range(len(c.rows)) for i in (c.start[s], c.start[s + 1] - 1) if c.rows[s]})
    return at if len(at) <= most else at[:most // 2] + at[-(most // 2):]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_whole_outputs(dev, ty, form):
    rng = np.random.default_rng(31)
    c, H = form_case(dev, rng, form, 128)
    q = typed(rng.standard_normal((c.T, H, 128)), ty)
    got = attention(dev, c, H, ty, q, 128 ** -0.5)
    pos, seq = c.positions(), c.sequences()
    for i in check_rows(c):
        k, v = rows_of(c, seq[i], pos[i] + 1)
        want = ref.attend(q[i], k, v, pos[i], 128 ** -0.5, 0)[0]
        assert off(got[i], want) <= WHOLE[ty], i


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", ("large", "larger than subnormal", "zeros", "zero sink"))
def test_value_scales_of_any_range(dev, ty, form, what):
    """Rows that carry nothing of the sum but have a large value scale (2^24 times the
    others', or 2^17 times f16's smallest, at a logit of -60), that have no value at all among rows of the smallest
    scales, or that take the probability (e^40 times the others') without a value.
    Logits are up to 2^7 from the reference: in fp32 they are rounded by 2^-18, rms
    2^-18 / sqrt(3) * ln 2 = 1.5e-6 of a probability, within 4 FP32 with the rest."""
    rng = np.random.default_rng(32)
    D = 128
    c, H = form_case(dev, rng, form, D)
    scale = D ** -0.5
    u = rng.standard_normal(D)
    u /= np.linalg.norm(u)
    # every query leans on u by 20; every key is without it, but for the odd rows
    q = rng.standard_normal((c.T, H, D))
    q += (20 - q @ u)[..., None] * u
    q = typed(q, ty)
    half = c.pool.bytes[..., 34 * D:].view(np.float16)  # value scales, by the row of a tile
    small, odd = {"large": (2.0 ** -10, 2.0 ** 14), "larger than subnormal": (2.0 ** -24, 2.0 ** -7),
                  "zeros": (2.0 ** -22, 0), "zero sink": (0.25, 0)}[what]
    half[...] = np.where(rng.random(half.shape) < 0.5, small, -small)
    if what == "zeros":
        half[..., np.arange(32) % 3 > 0] = 0
    else:
        half[..., 5] = odd
        codes, d = ref.quantize((u * (-60 if odd else 40) / 20 / scale).reshape(-1, 32))
        for s, n in enumerate(c.lens):
            for p in range(5, n, 32):
                tile = c.pool.bytes[c.table[s, p // 32], :, 0]
                for h in range(c.KH):
                    c.pool._put(tile[h].view(np.uint32), *c.pool._key_words(5), codes.ravel())
                    tile[h, 32 * D:].view(np.float16)[5 * D // 32:6 * D // 32] = d
    c_upload(c)
    got = attention(dev, c, H, ty, q, scale)
    assert np.all(np.isfinite(got))
    pos, seq = c.positions(), c.sequences()
    for i in check_rows(c):
        k, v = rows_of(c, seq[i], pos[i] + 1)
        want, _, size = ref.attend(q[i], k, v, pos[i], scale, 0)
        tol = 4 * WHOLE[ty]
        if ty == F16:  # results below its smallest normal
            tol += 2.0 ** -25 * np.sqrt(want.size) / np.linalg.norm(want)
        if what == "zero sink":
            # these rows are the whole sum, with one logit, which fp32 holds to 2^-24 of the
            # sum of its terms' sizes twice (its sum, its distance to the reference)
            tol += 2.0 ** -23 * size.max()
        e = off(got[i], want)
        assert e <= tol, (i, e, tol)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("D", (64, 128))
def test_long_caches_of_one_sign(dev, ty, D):
    """Tiles of 32 rows over 131072 cached rows whose value scales all have one sign and
    whose values cancel: a surplus of 8 a code, where it is carried along, does not, and
    outweighs the output 600 times."""
    rng = np.random.default_rng(33)
    n, rows, H = 131072, 512, 16
    c = Case(dev, rng, [rows], [n], 1024, 1, D)
    half = c.pool.bytes[..., 34 * D:].view(np.float16)
    half[...] = np.abs(half)
    nibbles = rng.integers(1, 16, (*c.pool.bytes.shape[:3], 32 * D), np.uint8)
    words = (nibbles[..., ::2] | nibbles[..., 1::2] << 4).view(np.uint32)
    c.pool.bytes[..., 16 * D:32 * D] = (words << 2 | words >> 30).view(np.uint8)
    c_upload(c)
    q = typed(rng.standard_normal((rows, H, D)), ty)
    got = attention(dev, c, H, ty, q, D ** -0.5)
    k, v = rows_of(c, 0, n)
    for i in (0, 300, 511):
        p = n - rows + i
        want = ref.attend(q[i], k[:p + 1], v[:p + 1], p, D ** -0.5, 0)[0]
        e = off(got[i], want)
        # (fp32: a wave adds n / 128 tiles, rounding each sum by up to 2^-24)
        assert e <= 2 * WHOLE[ty] + np.sqrt(n / 128) * 2.0 ** -24, i


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("D", (64, 128, 256))
@pytest.mark.parametrize("rows,KH,H", (([1], 1, 4), ([1, 2], 2, 2), ([40], 1, 2)))
def test_a_bound_of_no_rows_at_all(dev, ty, D, rows, KH, H):
    """max_len 0: every row is before its sequence's start, and its output 0."""
    rng = np.random.default_rng(35)
    c = Case(dev, rng, rows, [0] * len(rows), 32, KH, D)
    c.batch.max_len = 0
    q = typed(rng.standard_normal((c.T, H, D)), ty)
    assert np.all(attention(dev, c, H, ty, q, 0.1, in_place=True) == 0)
    assert c.errors() == 0


@pytest.mark.parametrize("ty", (F32, BF16))
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size,scale", ((1e-37, 1e-20), (0.0, 3e37), (1.0, 1e6)))
def test_scales_of_any_size(dev, ty, form, size, scale):
    """Logits that do not differ from 0: every row is the mean of the rows it sees, and
    of none that it does not see.  Logits that differ by thousands: it is one row."""
    rng = np.random.default_rng(34)
    D = 128
    c, H = form_case(dev, rng, form, D)
    half = c.pool.bytes[..., 32 * D:34 * D].view(np.float16)
    half[...] = half * np.float16(0.01)  # key scales: logits below 2^21
    c_upload(c)
    q = typed(rng.standard_normal((c.T, H, D)) * size, ty)
    got = attention(dev, c, H, ty, q, scale)
    pos, seq = c.positions(), c.sequences()
    for i in check_rows(c):
        k, v = rows_of(c, seq[i], pos[i] + 1)
        want = ref.attend(q[i], k, v, pos[i], scale, 0)[0]
        assert off(got[i], want) <= WHOLE[ty], i


@pytest.mark.parametrize("ty,D,max_rows", ((F32, 128, 2), (F16, 64, 70000), (BF16, 256, 70000)))
def test_positions_near_the_largest(dev, ty, D, max_rows):
    """Rows at positions up to 2^31 - 2^16 - 2, with a bound of rows that reaches past
    2^31, beside a short sequence: stored, read back and attended to in a window."""
    rng = np.random.default_rng(36)
    KH, H, page, window = 2, 4, 1024, 40
    longest = (1 << 31) - (1 << 16) - 1
    rows, lens = [2, 1], [longest, 7]
    c = Case(dev, rng, [2, 1], [2, 7], page, KH, D)  # pages 0, 1 of each in turn
    stride = -(-longest // page)
    d_table = dev.h.malloc(2 * stride * 4)
    dev.p.append(d_table)
    # the last page of the long sequence, the first of the short one
    dev.h.copy_in(d_table + (stride - 1) * 4, c.table[0, :1])
    dev.h.copy_in(d_table + stride * 4, c.table[1, :1])
    b = hipkv.Batch(2, max(3, max_rows), max_rows, longest, c.d_start, dev.up(np.asarray(lens, np.int32)),
                    d_table, stride)
    x = rng.standard_normal((3, H + 2 * KH, D)).astype(np.float32)
    d_x, n, e = dev.up(ref.to_type(x, ty)), (H + 2 * KH) * D, ref.BYTES[ty]
    x = typed(x, ty)
    pos = np.array([longest - 2, longest - 1, 6])
    f, mag = hipkv.rope_freqs(D, 1e4)
    hipkv.append(c.cache, b, ty, d_x + H * D * e, d_x + (H + KH) * D * e, n, q=d_x, q_stride=n, heads=H, q_out=d_x,
                 q_out_stride=n, rope=hipkv.Rope(D, hipkv.HALVES, dev.up(f), mag))
    # angles to 2^31 have their own last bit: 2^-22 of a pair; keys are those that were stored
    for i, s in ((0, 0), (1, 0), (2, 1)):
        c.pool.store(np.repeat(c.table[s], 2), pos[i] % page, np.zeros((KH, D)), x[i, H + KH:].astype(np.float32))
    got, want = c.pool_bytes(), c.pool.bytes
    keys = np.zeros(want.shape[-1], bool)
    keys[:16 * D] = keys[32 * D:34 * D] = True
    assert np.array_equal(got[..., ~keys], want[..., ~keys]) and c.errors() == 0
    untouched = np.ones(c.pages, bool)
    untouched[c.table[:, 0]] = False
    assert np.array_equal(got[untouched], want[untouched])
    c.pool.bytes = got
    stored = [c.pool.load(np.repeat(c.table[s], 2), pos[i] % page) for i, s in ((0, 0), (1, 0), (2, 1))]
    q = ref.rotate(x, pos, f, mag, hipkv.HALVES)
    for i in range(3):
        top = np.abs(q[i, H:H + KH]).reshape(KH, -1, 32).max(-1).repeat(32, -1)
        assert np.all(np.abs(stored[i][0] - q[i, H:H + KH]) <= top / 8 * 1.01)
    back = [dev.up(np.zeros((3, KH * D), ref.np_dtype(ty))) for _ in "kv"]
    hipkv.read(c.cache, b, ty, *back, KH * D)
    for d, which in zip(back, (0, 1)):
        want = np.stack([stored[i][which].ravel() for i in range(3)])
        assert np.array_equal(dev.get(d, (3, KH * D), ref.np_dtype(ty)), ref.to_type(want, ty))
    ws = hipkv.attn_ws(c.cache, b, H)
    d_ws, d_o = dev.h.malloc(max(ws, 16)), dev.up(np.zeros((3, H * D), ref.np_dtype(ty)))
    dev.p.append(d_ws)
    hipkv.attn(c.cache, b, ty, d_x, n, H, d_o, H * D, D ** -0.5, window, d_ws, ws)
    got = ref.from_type(dev.get(d_o, (3, H, D), ref.np_dtype(ty)), ty)
    q = ref.from_type(dev.get(d_x, (3, H + 2 * KH, D), ref.np_dtype(ty)), ty)[:, :H]
    for i, s in ((0, 0), (1, 0), (2, 1)):
        rows = range(max(0, pos[i] % page + 1 - window), pos[i] % page + 1)
        k, v = (np.stack(y) for y in zip(*[c.pool.load(np.repeat(c.table[s], 2), p) for p in rows]))
        want = ref.attend(q[i], k, v, len(rows) - 1, D ** -0.5, 0)[0]
        assert off(got[i], want) <= 2 * WHOLE[ty], i
    assert c.errors() == 0


# --------------------------------------------------------------------------
# workgroups of several rows and heads
# --------------------------------------------------------------------------

@pytest.mark.parametrize("layout", (hipkv.PAIRS, hipkv.HALVES))
@pytest.mark.parametrize("ty,rows,heads,D,rot,pad", (
    (F32, 1025, 3, 128, 128, 0), (BF16, 4099, 2, 128, 96, 8), (F16, 4099, 5, 64, 64, 0),
    (F32, 4099, 1, 90, 50, 3), (BF16, 1030, 3, 77, 70, 1),  # value by value
    (F32, 4099, 1, 1024, 1024, 0), (F16, 4101, 2, 1024, 912, 0), (F32, 4098, 1, 1023, 1022, 0)))
def test_rotations_of_many_rows(dev, ty, layout, rows, heads, D, rot, pad):
    """Up to eight rows a workgroup and a last one of fewer, whose angles take up to
    72 KB of LDS."""
    rng = np.random.default_rng(rows + D)
    x = rng.standard_normal((rows, heads, D)).astype(np.float32)
    pos = rng.integers(0, 1 << 17, rows).astype(np.int32)
    f, mag = hipkv.rope_freqs(rot, 1e6)
    stride = heads * D + pad
    d_x = up_typed(dev, x.reshape(rows, -1), ty, stride)
    d_o = up_typed(dev, np.zeros((rows + 1, heads * D), np.float32), ty, stride, fill=-3.0)
    R = hipkv.Rope(rot, layout, dev.up(f), mag)
    d_pos = dev.up(pos)
    hipkv.rope(R, ty, d_x, stride, d_o, stride, rows, heads, D, d_pos)
    got = ref.from_type(dev.get(d_o, (rows + 1, stride), ref.np_dtype(ty)), ty)
    assert np.all(got[:, heads * D:] == -3.0) and np.all(got[rows, :heads * D] == 0)
    want = ref.rotate(typed(x, ty), pos, f, mag, layout)
    err = np.abs(got[:rows, :heads * D].reshape(want.shape) - want)
    # angles to 2^17 have their last bit at 2^-36, times pairs of up to 8; f16's subnormals
    tol = np.abs(want) * (ref.HALF_STEP[ty] + 2.0 ** -24) + 2.0 ** -33 + (2.0 ** -25 if ty == F16 else 0)
    assert np.all(err <= tol), (err / tol).max()
    hipkv.rope(R, ty, d_x, stride, d_x, stride, rows, heads, D, d_pos)
    again = ref.from_type(dev.get(d_x, (rows, stride), ref.np_dtype(ty)), ty)
    assert np.array_equal(again[:, :heads * D], got[:rows, :heads * D]) and np.all(again[:, heads * D:] == 7.0)


def store_row(P, table, p, k, v):
    """Pool.store of one row, all heads at once."""
    D, KH = P.D, P.KH
    pg, t, r = int(table[p // P.page]), p % P.page // 32, p % 32
    tile = P.bytes[pg, :, t]
    words, half = tile.view(np.uint32), tile[:, 32 * D:].view(np.float16)

    def turned(codes, bit):
        z = codes.astype(np.uint64) << bit.astype(np.uint64)
        return ((z | z >> np.uint64(32)) & np.uint64(0xffffffff)).astype(np.uint32)

    q, d = ref.quantize(k.reshape(KH, -1, 32))
    w, b = P._key_words(r)
    words[:, w[::8]] = np.bitwise_or.reduce(turned(q.reshape(KH, D), b).reshape(KH, -1, 8), -1)
    half[:, r * (D // 32):(r + 1) * (D // 32)] = d
    q, d = ref.quantize(v)
    w, b = P._value_words(r)
    words[:, w] = words[:, w] & ~turned(np.full(D, 15), b) | turned(q, b)
    half[:, D + r] = d


@pytest.mark.parametrize("ty,D", ((F32, 64), (F16, 64), (BF16, 128), (F32, 128), (F16, 256), (F32, 256)))
@pytest.mark.parametrize("nseq,n,KH,H", ((22, 33, 5, 7),    # two heads a workgroup, the last one alone
                                         (64, 20, 5, 10),   # all five
                                         (300, 1, 5, 13),   # single rows, four heads and one
                                         (1, 2100, 7, 3)))  # fewer query heads than kv heads
def test_appends_of_many_rows_and_heads(dev, ty, D, nseq, n, KH, H):
    rng = np.random.default_rng(nseq + D + ty)
    rows = [int(i) for i in rng.integers(max(1, n // 2), n + 1, nseq)]
    rows[0] = n
    lens = [r + int(b) for r, b in zip(rows, rng.integers(0, 90, nseq))]
    if nseq > 1:
        lens[1] = rows[1] // 2  # some of its rows are not there
    c = Case(dev, rng, rows, lens, 64, KH, D)
    x = rng.standard_normal((c.T, H + 2 * KH, D)).astype(np.float32)
    x[:, H:H + KH, ::11] *= 7
    stride, e = (H + 2 * KH) * D, ref.BYTES[ty]
    d_x = dev.up(ref.to_type(x, ty))
    x = typed(x, ty)
    f, mag = hipkv.rope_freqs(D // 2, 1e4)
    hipkv.append(c.cache, c.batch, ty, d_x + H * D * e, d_x + (H + KH) * D * e, stride,
                 rope=hipkv.Rope(D // 2, hipkv.PAIRS, dev.up(f), mag), q=d_x, q_stride=stride, heads=H,
                 q_out=d_x, q_out_stride=stride)
    pos, seq = c.positions(), c.sequences()
    there = pos >= 0
    turned = ref.rotate(x[:, :H + KH], pos, f, mag, hipkv.PAIRS)
    got = ref.from_type(dev.get(d_x, x.shape, ref.np_dtype(ty)), ty)
    # rows that are not there keep their queries, as k and v do
    want = np.where(there[:, None, None], turned[:, :H], x[:, :H])
    tol = np.abs(want) * (ref.HALF_STEP[ty] + 2.0 ** -24) + 2.0 ** -25
    assert np.all(np.abs(got[:, :H] - want) <= tol)
    assert np.array_equal(got[:, H:], x[:, H:])
    for i in np.flatnonzero(there):
        store_row(c.pool, c.table[seq[i]], pos[i], turned[i, H:].astype(np.float32), x[i, H + KH:].astype(np.float32))
    got = c.pool_bytes()
    assert np.array_equal(got, c.pool.bytes), np.argwhere(got != c.pool.bytes)[:5]
    assert c.errors() == 0


# --------------------------------------------------------------------------
# shares of many caches
# --------------------------------------------------------------------------

@pytest.mark.parametrize("ty,D,KH,G,nseq,window", ((F32, 128, 8, 4, 64, 0), (BF16, 64, 16, 2, 70, 0), (F16, 256, 8, 3, 64, 70),
                                                   (BF16, 128, 4, 16, 129, 0)))
def test_shares_in_place_and_beside_bad_sequences(dev, ty, D, KH, G, nseq, window):
    """Outputs over the queries; a page outside the pool, which changes its own sequence
    alone; a length past the bound, which moves where every other sequence is cut."""
    rng = np.random.default_rng(37)
    H, scale = KH * G, D ** -0.5
    lens = [int(i) for i in rng.integers(1, 200, nseq)]
    lens[0], lens[5] = 333, 64
    c = Case(dev, rng, [1] * nseq, lens, 32, KH, D, slack=16384 // 32)
    c.batch.max_len = 16384
    q = typed(rng.standard_normal((nseq, H, D)), ty)
    want = attention(dev, c, H, ty, q, scale, window)
    assert np.array_equal(attention(dev, c, H, ty, q, scale, window, in_place=True), want) and c.errors() == 0

    def batch(table, length):
        return hipkv.Batch(nseq, nseq, 1, 16384, c.d_start, dev.up(np.asarray(length, np.int32)), dev.up(table),
                           table.shape[1])

    table = c.table.copy()
    table[0, 9] = c.pages  # rows 288 .. 319 of the first sequence
    got = attention(dev, c, H, ty, q, scale, window, batch=batch(table, lens))
    assert c.errors() == hipkv.ERR_PAGE
    assert np.array_equal(got[1:], want[1:])
    k, v = rows_of(c, 0, 333)
    keep = [j for j in range(max(0, 333 - window) if window else 0, 333) if not 288 <= j < 320]
    assert off(got[0], ref.attend(q[0], k[keep], v[keep], len(keep) - 1, scale, 0)[0]) <= 2 * WHOLE[ty]

    dev.h.copy_in(c.d_err, np.zeros(1, np.uint32))
    length = list(lens)
    length[5] = 20000
    got = attention(dev, c, H, ty, q, scale, window, batch=batch(c.table, length))
    assert c.errors() == hipkv.ERR_PAGE | hipkv.ERR_BATCH  # (nor has it pages to its bound)
    for i in (0, 1, 4, 6, 7, nseq - 2, nseq - 1):
        assert off(got[i], want[i]) <= 2 * WHOLE[ty], i


@pytest.mark.parametrize("H,n", ((2, 1), (16, 300)))
def test_a_pool_without_pages(dev, H, n):
    """Rows that see nothing report nothing; those that would are NaN and reported."""
    rng = np.random.default_rng(38)
    D, KH = 64, 2
    c = Case(dev, rng, [n] * 9, [0] * 9, 32, KH, D)
    c.cache.pages = 0
    q = typed(rng.standard_normal((c.T, H, D)), F32)
    c.batch.max_len = 2000
    c.batch.table, c.batch.table_stride = dev.up(np.zeros((9, 63), np.int32)), 63
    assert np.all(attention(dev, c, H, F32, q, 0.1) == 0) and c.errors() == 0
    c.batch.len = dev.up(np.full(9, 40, np.int32))
    got = attention(dev, c, H, F32, q, 0.1).reshape(9, n, -1)
    there = np.arange(n) >= n - 40
    assert np.all(np.isnan(got[:, there])) and np.all(got[:, ~there] == 0)
    assert c.errors() == hipkv.ERR_PAGE
