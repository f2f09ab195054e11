"""The 8-bit floating-point products (hip_f8.h) as a program runs them: captured into a
graph and replayed, on several streams at once, behind the router; and far apart in
memory.  Tolerances: test_gpu_f8.py."""
import numpy as np
import pytest

import f8_ref as ref
import hipf8
import hipmoe
from f8_ref import BF16, F16, F32, DevMat, DevRows, random_rows, up_typed, wide
from test_f8_plan import form
from test_gpu_f8 import check_product, dev, product  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


class Layer:
    """The experts of a layer, and the memory of one chain of calls for up to `tokens` tokens."""

    def __init__(self, dev, rng, ty, tokens, topk, experts, width, inner, mats=None):
        self.dev, self.ty, self.tokens, self.topk, self.experts = dev, ty, tokens, topk, experts
        self.width, self.inner = width, inner
        self.mats = mats or [DevMat(dev, rng, inner, width, experts), DevMat(dev, rng, inner, width, experts),
                             DevMat(dev, rng, width, inner, experts)]
        P = tokens * topk
        self.ws, self.hs, hq = wide(width, ty), wide(inner, ty), -(-inner // 16) * 16

        def room(shape, dtype):
            return dev.up(np.zeros(shape, dtype))

        self.x, self.out = room((tokens, self.ws), ref.np_dtype(ty)), room((tokens, self.ws), ref.np_dtype(ty))
        self.h, self.y = room((P, self.hs), ref.np_dtype(ty)), room((P, self.ws), ref.np_dtype(ty))
        self.ids, self.w = room((tokens, topk), np.uint32), room((tokens, topk), np.float32)
        self.start, self.frm, self.pos = room(experts + 1, np.int32), room(P, np.int32), room(P, np.int32)
        xq = -(-width // 16) * 16
        self.xq = hipf8.Rows(room((tokens, xq), np.uint8), xq, room((ref.blocks(width), tokens), np.float32), tokens,
                             tokens, width)
        self.hq = hipf8.Rows(room((P, hq), np.uint8), hq, room((ref.blocks(inner), P), np.float32), P, P, inner)

    def enqueue(self, stream=None):
        ty, P = self.ty, self.tokens * self.topk
        gate, up, down = (m.mat for m in self.mats)
        hipf8.sort(self.ids, self.tokens, self.topk, self.experts, self.start, self.frm, self.pos, stream)
        hipf8.quantize(ty, self.x, self.ws, self.xq, stream)
        hipf8.group_mul(self.xq, self.frm, self.start, P, gate, up, ty, self.h, self.hs, stream)
        hipf8.quantize(ty, self.h, self.hs, self.hq, stream)
        hipf8.group_mul(self.hq, None, self.start, P, down, None, ty, self.y, self.ws, stream)
        hipf8.combine(ty, self.y, self.ws, P, self.pos, self.w, self.tokens, self.topk, self.width, self.x, self.ws,
                      self.out, self.ws, stream)

    def put(self, rng):
        h = self.dev.h
        x = rng.standard_normal((self.tokens, self.ws)).astype(np.float32)
        ids = np.stack([rng.permutation(self.experts + 1)[:self.topk] for _ in range(self.tokens)])
        w = rng.dirichlet(np.ones(self.topk), self.tokens)
        h.copy_in(self.x, ref.to_type(x, self.ty))
        h.copy_in(self.ids, ids.astype(np.uint32))
        h.copy_in(self.w, w.astype(np.float32))
        return x, ids, w

    def get(self):
        return self.dev.get(self.out, (self.tokens, self.ws), ref.np_dtype(self.ty))


@pytest.mark.parametrize("ty,tokens,topk,experts,width,inner", (
    (F32, 3, 2, 8, 384, 256), (BF16, 70, 2, 5, 256, 400), (F16, 900, 4, 8, 512, 640)))
def test_a_captured_layer(dev, ty, tokens, topk, experts, width, inner):  # noqa: F811
    """One graph of all calls, replayed with other tokens, ids and weights: each time what the
    same calls give eagerly, bit for bit."""
    rng = np.random.default_rng(tokens)
    h, st = dev.h, dev.h.stream()
    a = Layer(dev, rng, ty, tokens, topk, experts, width, inner)
    b = Layer(dev, rng, ty, tokens, topk, experts, width, inner, a.mats)
    a.put(rng)
    h.begin_capture(st)
    a.enqueue(st)
    graph = h.end_capture(st)
    for i in range(4):
        a.put(np.random.default_rng(100 + i))
        b.put(np.random.default_rng(100 + i))
        h.graph_launch(graph, st)
        h.stream_sync(st)
        b.enqueue()
        got, want = a.get(), b.get()
        assert np.array_equal(got, want), i
        assert np.isfinite(ref.from_type(got, ty)).all()
    h.h.hipGraphExecDestroy(graph)
    h.h.hipStreamDestroy(st)


def test_layers_on_several_streams_at_once(dev):  # noqa: F811
    """Three streams run layers on the same matrices at the same time."""
    rng = np.random.default_rng(4)
    h = dev.h
    mats = Layer(dev, rng, BF16, 1, 2, 6, 512, 384).mats
    runs = []
    for i, tokens in enumerate((5, 300, 1500)):
        one, two = (Layer(dev, rng, BF16, tokens, 2, 6, 512, 384, mats) for _ in "12")
        one.put(np.random.default_rng(i))
        two.put(np.random.default_rng(i))
        runs.append((one, two, h.stream()))
    for one, _, st in runs * 4:
        one.enqueue(st)
    h.sync()
    for one, two, st in runs:
        two.enqueue()
        assert np.array_equal(one.get(), two.get())
        h.h.hipStreamDestroy(st)


def test_behind_the_router(dev):  # noqa: F811
    """Ids and weights as hip_moe_route_dev leaves them on the device go into the sort and the
    sum as they are."""
    rng = np.random.default_rng(8)
    E, EI, NE, topk, T = 256, 512, 16, 4, 37
    moe = hipmoe.MoeLayer.from_synth(hipmoe.synth_layer(7, 0, hipmoe.Q8_0, E, EI, NE, 0.02, None), topk, True)
    L = Layer(dev, rng, F32, T, topk, NE, E, EI)
    x, _, _ = L.put(rng)
    assert hipmoe.lib().hip_moe_route_dev(moe.h, L.x, T, None, None, None, L.ids, L.w, None) == 1
    L.enqueue()
    got = L.get()
    ids, w = dev.get(L.ids, (T, topk), np.uint32), dev.get(L.w, (T, topk), np.float32)
    assert len(np.unique(ids)) > 4
    xq = ref.rows_of(*ref.quantize(x))
    want = x.astype(np.float64)
    for t in range(T):
        for s in range(topk):
            e = ids[t, s]
            h = ref.gate(L.mats[0].w[e] @ xq[t], L.mats[1].w[e] @ xq[t])
            hq = ref.rows_of(*ref.quantize(h.astype(np.float32)[None]))[0]
            want[t] += w[t, s] * (L.mats[2].w[e] @ hq)
    # a value of h next to a border may be quantized the other way, off by a step of 2^-3 of it: that
    # is 2^-3 / sqrt(T topk EI) = 4.5e-4 of all of h if it is of ordinary size, and its 10^-6 of rounding
    # in a step of 2^-4 makes one or two of these 75776 such; 4 of 3 times the ordinary size pass
    assert np.linalg.norm(got - want) <= 3e-3 * np.linalg.norm(want - x)
    moe.free()


# --------------------------------------------------------------------------
# far apart
# --------------------------------------------------------------------------

def spread(dev, rows, stride):
    """Device memory with the rows `stride` bytes apart; what lies between is not set."""
    p = dev.h.malloc((len(rows) - 1) * stride + -(-rows[0].nbytes // 16) * 16)
    dev.p.append(p)
    for i, r in enumerate(rows):
        dev.h.copy_in(p + i * stride, r)
    return p


def gather(dev, p, rows, stride, n, dtype):
    dev.h.sync()
    return np.stack([dev.h.download(p + int(i) * stride, n, dtype) for i in rows])


def test_experts_5_gib_apart(dev):  # noqa: F811
    rng = np.random.default_rng(1)
    X, W = random_rows(dev, rng, 300, 400), DevMat(dev, rng, 200, 400, 2)
    step = 5 << 30
    codes = np.full((2, 200, 400), 0, np.uint8)
    codes[:, :, :400] = W.codes
    W.mat.codes, W.mat.step, W.mat.stride = spread(dev, list(codes.reshape(2, -1)), step), step, 400
    start = dev.up(np.array([0, 120, 300], np.int32))
    for ty in (BF16, F32):
        d_o = dev.up(np.zeros((300, 200), ref.np_dtype(ty)))
        hipf8.group_mul(X.rows, None, start, 300, W.mat, None, ty, d_o, 200)
        got = ref.from_type(dev.get(d_o, (300, 200), ref.np_dtype(ty)), ty)
        check_product(got[:120], *product(X.x[:120], W.w[0]), ty)
        check_product(got[120:], *product(X.x[120:], W.w[1]), ty)


@pytest.mark.parametrize("ty,total,n,k", ((BF16, 12, 300, 500), (F32, 400, 300, 500), (F16, 3400, 1500, 1000)))
def test_gathered_rows_over_5_gib(dev, ty, total, n, k):  # noqa: F811
    """Rows 16 MiB apart: their distances do not fit 32 bits, and the form that keeps them in as
    many is not taken."""
    rng = np.random.default_rng(total)
    tokens, stride, gated = 330, 1 << 24, ty == F16
    Y = random_rows(dev, rng, tokens, k)
    rows = [np.pad(r, (0, -k % 16)) for r in Y.codes]
    Y.rows.codes, Y.rows.stride = spread(dev, rows, stride), stride
    counts = [total // 2, 0, total - total // 2]
    if total == 3400:
        assert form(ty, total, n, k, gated, experts=3, gather=True, x_rows=tokens) == "TILE_256"
    W = DevMat(dev, rng, n, k, 3)
    U = DevMat(dev, rng, n, k, 3) if gated else None
    frm = rng.integers(0, tokens, total).astype(np.int32)
    d_o = dev.up(np.zeros((total, wide(n, ty)), ref.np_dtype(ty)))
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    hipf8.group_mul(Y.rows, dev.up(frm), dev.up(start), total, W.mat, U and U.mat, ty, d_o, wide(n, ty))
    got = ref.from_type(dev.get(d_o, (total, wide(n, ty)), ref.np_dtype(ty)), ty)[:, :n]
    for e in (0, 2):
        at = np.arange(start[e], start[e + 1])
        at = at[rng.random(at.size) < 60 / at.size]
        check_product(got[at], *product(Y.x[frm[at]], W.w[e], U and U.w[e]), ty)


@pytest.mark.parametrize("ty,rows,n,k", ((F32, 12, 100, 300), (BF16, 150, 200, 300), (F16, 4100, 6200, 520)))
def test_outputs_over_4_gib(dev, ty, rows, n, k):  # noqa: F811
    rng = np.random.default_rng(rows)
    stride = (5 << 30) // rows // 16 * 16 // (4 if ty == F32 else 2)
    stride -= stride % 8
    size = stride * (4 if ty == F32 else 2)
    X, W = random_rows(dev, rng, rows, k), DevMat(dev, rng, n, k)
    p = dev.h.malloc(rows * size)
    dev.p.append(p)
    hipf8.mul(X.rows, W.mat, None, ty, p, stride)
    at = np.unique(np.concatenate([[0, 1, rows - 1], rng.integers(0, rows, 20)]))
    got = ref.from_type(gather(dev, p, at, size, n, ref.np_dtype(ty)), ty)
    check_product(got, *product(X.x[at], W.w[0]), ty)


def test_rows_of_weights_16_mib_apart(dev):  # noqa: F811
    rng = np.random.default_rng(3)
    n, k, stride = 260, 300, 1 << 24
    W = DevMat(dev, rng, n, k)
    rows = [np.pad(r, (0, -k % 16)) for r in W.codes[0]]
    W.mat.codes, W.mat.stride = spread(dev, rows, stride), stride
    for ty, m in ((BF16, 3), (BF16, 40), (F32, 300), (F16, 5000)):
        X = random_rows(dev, rng, m, k)
        d_o = dev.up(np.zeros((m, 264), ref.np_dtype(ty)))
        hipf8.mul(X.rows, W.mat, None, ty, d_o, 264)
        got = ref.from_type(dev.get(d_o, (m, 264), ref.np_dtype(ty)), ty)[:, :n]
        at = np.unique(rng.integers(0, m, 50))
        check_product(got[at], *product(X.x[at], W.w[0]), ty)


def test_quantize_and_combine_over_4_gib(dev):  # noqa: F811
    rng = np.random.default_rng(5)
    n, k, stride = 5, 300, 1 << 28
    x = rng.standard_normal((n, k)).astype(np.float32)
    p = spread(dev, list(x), stride * 4)
    d_c, d_s = dev.up(np.zeros((n, 304), np.uint8)), dev.up(np.zeros((3, n), np.float32))
    hipf8.quantize(F32, p, stride, hipf8.Rows(d_c, 304, d_s, n, n, k))
    codes, scale = ref.quantize(x)
    assert np.array_equal(dev.get(d_c, (n, 304), np.uint8)[:, :k], codes)
    assert np.array_equal(dev.get(d_s, (3, n), np.float32), scale)
    pos = np.array([[4, 0], [1, -1], [3, 4]], np.int32)
    w = rng.random((3, 2)).astype(np.float32)
    out = dev.h.malloc(2 * stride * 4 + 1216)
    dev.p.append(out)
    hipf8.combine(F32, p, stride, n, dev.up(pos), dev.up(w), 3, 2, k, p, stride, out, stride)
    got = gather(dev, out, range(3), stride * 4, k, np.float32)
    here = pos >= 0
    want = x[:3].astype(np.float64) + (np.where(here, w, 0)[..., None] * x[np.where(here, pos, 0)].astype(np.float64)).sum(1)
    assert np.all(np.abs(got - want) <= 3 * 2.0 ** -23 * (np.abs(x[:3]) + 2 * np.abs(x).max()))


def test_rows_of_codes_16_mib_apart(dev):  # noqa: F811
    """Quantized rows whose codes are 5 GiB, and their product with fewer rows than a tile."""
    rng = np.random.default_rng(6)
    n, k, stride = 330, 200, 1 << 24
    x = rng.standard_normal((n, 200)).astype(np.float32)
    p = dev.h.malloc((n - 1) * stride + 208)
    dev.p.append(p)
    d_s = dev.up(np.zeros((2, n), np.float32))
    R = hipf8.Rows(p, stride, d_s, n, n, k)
    hipf8.quantize(F32, dev.up(x), k, R)
    codes, scale = ref.quantize(x)
    assert np.array_equal(gather(dev, p, range(n), stride, k, np.uint8), codes)
    W = DevMat(dev, rng, 70, k)
    d_o = dev.up(np.zeros((n, 72), np.float32))
    hipf8.mul(R, W.mat, None, F32, d_o, 72)
    got = dev.get(d_o, (n, 72), np.float32)[:, :70]
    check_product(got, *product(ref.rows_of(codes, scale), W.w[0]), F32)


def test_tiles_of_rows_16_mib_apart(dev):  # noqa: F811
    """Rows and rows of weights 16 MiB apart in the tiles of 256 x 256."""
    rng = np.random.default_rng(7)
    m, n, k, stride = 512, 30000, 1000, 1 << 24
    assert form(F16, m, n, k) == "TILE_256"
    X = random_rows(dev, rng, m, k)
    X.rows.codes, X.rows.stride = spread(dev, [np.pad(r, (0, -k % 16)) for r in X.codes], stride), stride
    codes = np.tile(ref.random_codes(rng, (1, 1000, k)), (1, 30, 1))
    W = DevMat(dev, rng, n, k, codes=codes)
    d_o = dev.up(np.zeros((m, n), np.float16))
    hipf8.mul(X.rows, W.mat, None, F16, d_o, n)
    got = dev.get(d_o, (m, n), np.float16)
    at, to = np.r_[0:3, 250:260, 509:512], np.r_[0:300, 20000:20100, 29900:30000]
    check_product(got[np.ix_(at, to)], *product(X.x[at], W.w[0][to]), F16)
