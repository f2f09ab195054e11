"""The 8-bit floating-point products of include/hip_f8.h in numpy and 64 bits: what
the GPU tests of hip_f8 compare with."""
import numpy as np

import hipf8
import hipmoe
from kv_ref import HALF_STEP, from_type, np_dtype, to_type  # noqa: F401  (the same three types)

F32, F16, BF16 = hipf8.F32, hipf8.F16, hipf8.BF16
BLOCK = hipf8.BLOCK

_m = np.arange(8)
_VALUES = np.concatenate([_m * 2.0 ** -9] + [(8 + _m) * 2.0 ** (e - 10) for e in range(1, 16)])
_VALUES[127] = np.nan
VALUES = np.concatenate([_VALUES, -_VALUES])  # of the codes 0 .. 255


def codes_of(q):
    """The codes of the e4m3 values nearest to q (any size up to 448 and a little), ties to even."""
    v = _VALUES[:127]
    mid = (v[1:] + v[:-1]) / 2
    a = np.abs(q)
    lo, hi = np.searchsorted(mid, a, "left"), np.searchsorted(mid, a, "right")
    c = np.where(lo % 2 == 0, lo, hi)
    return (c | np.where(np.signbit(q), 128, 0)).astype(np.uint8)


def blocks(k):
    return -(-k // BLOCK)


def quantize(x):
    """(codes [rows][k], scales float32 [blocks][rows]) of values x [rows][k]."""
    x = np.asarray(x, np.float64)
    n, k = x.shape
    codes, scale = np.zeros((n, k), np.uint8), np.zeros((blocks(k), n), np.float32)
    for b in range(blocks(k)):
        y = x[:, b * BLOCK:(b + 1) * BLOCK]
        bad = ~np.isfinite(y).all(1)
        z = np.where(bad[:, None], 0.0, y)
        # a quotient of two numbers of 24 bits that is not halfway between two is not so close to it
        # that its rounding to 53 bits changes the one to 24
        s = np.maximum((np.abs(z).max(1) / 448.0).astype(np.float32), np.float32(2.0 ** -96))
        c = codes_of(z / s.astype(np.float64)[:, None])
        codes[:, b * BLOCK:(b + 1) * BLOCK] = np.where(bad[:, None], 0, c)
        scale[b] = np.where(bad, np.float32(np.nan), s)
    return codes, scale


def rows_of(codes, scale):
    """What quantized rows stand for: codes [rows][k], scale [blocks][rows]."""
    k = codes.shape[1]
    return VALUES[codes] * np.repeat(scale.astype(np.float64).T, BLOCK, 1)[:, :k]


def mat_of(codes, scale):
    """What a matrix stands for: codes [n][k], scale [n / 128][k / 128]."""
    n, k = codes.shape
    s = np.repeat(np.repeat(scale.astype(np.float64), BLOCK, 0)[:n], BLOCK, 1)[:, :k]
    return VALUES[codes] * s


def gate(a, b):
    with np.errstate(over="ignore"):
        return a / (1 + np.exp(-a)) * b


def sort(ids, experts):
    """(start, from of the rows there are, pos)"""
    flat = np.asarray(ids, np.int64).ravel()
    order = np.argsort(np.where(flat < experts, flat, experts), kind="stable")
    total = int((flat < experts).sum())
    start = np.searchsorted(flat[order][:total], np.arange(experts + 1)).astype(np.int32)
    pos = np.full(flat.size, -1, np.int32)
    pos[order[:total]] = np.arange(total)
    return start, (order[:total] // ids.shape[1]).astype(np.int32), pos.reshape(ids.shape)


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


def up_typed(dev, x, ty, stride, fill=7.0):
    """Rows x [n][w] of the type, stride values apart, the gaps filled."""
    a = np.full((max(x.shape[0], 1), stride), fill, np.float32)
    a[:x.shape[0], :x.shape[1]] = x
    return dev.up(to_type(a, ty))


def wide(n, ty, pad=0):
    """Values that rows of n are apart: a multiple of 16 bytes, and pad times 16 bytes more."""
    by = 4 if ty == F32 else 8
    return (-(-n // by) + pad) * by


class DevRows:
    """Quantized rows on the device, their gaps full of NaN codes."""

    def __init__(self, dev, codes, scale, pad=0, scale_pad=0):
        n, k = codes.shape
        self.codes, self.scale = codes, scale
        stride = -(-k // 16) * 16 + 16 * pad
        room = np.full((max(n, 1), stride), 0x7f, np.uint8)
        room[:n, :k] = codes
        wide_scale = np.full((blocks(k), n + scale_pad + (n == 0)), np.nan, np.float32)
        wide_scale[:, :n] = scale
        self.stride, self.scale_stride = stride, wide_scale.shape[1]
        self.d_codes, self.d_scale = dev.up(room), dev.up(wide_scale)
        self.rows = hipf8.Rows(self.d_codes, stride, self.d_scale, self.scale_stride, n, k)
        self.x = rows_of(codes, scale)


class DevMat:
    """`count` matrices on the device, their gaps full of NaN codes."""

    def __init__(self, dev, rng, n, k, count=1, pad=0, scale_pad=0, codes=None):
        self.codes = random_codes(rng, (count, n, k)) if codes is None else codes
        self.scale = (rng.uniform(0.7, 1.3, (count, blocks(n), blocks(k))) * 2e-4).astype(np.float32)
        stride = -(-k // 16) * 16 + 16 * pad
        room = np.full((count, n, stride), 0xff, np.uint8)
        room[:, :, :k] = self.codes
        wide_scale = np.full((count, blocks(n), blocks(k) + scale_pad), np.nan, np.float32)
        wide_scale[:, :, :blocks(k)] = self.scale
        self.mat = hipf8.Mat(dev.up(room), stride, dev.up(wide_scale), blocks(k) + scale_pad, n, k, count,
                             n * stride, blocks(n) * (blocks(k) + scale_pad))
        self.w = [mat_of(c, s) for c, s in zip(self.codes, self.scale)]


def random_codes(rng, shape):
    """Codes as quantized normal values have them."""
    return codes_of(np.clip(rng.standard_normal(shape) * 112, -448, 448))


def random_rows(dev, rng, n, k, pad=0, scale_pad=0):
    x = rng.standard_normal((n, k)) * (1 + 7 * (rng.random(k) < 0.05))
    return DevRows(dev, *quantize(x.astype(np.float32)), pad, scale_pad)
