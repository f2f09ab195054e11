"""The 4-bit cache, rotations and attention of include/hip_kv.h in numpy and
64 bits: what the GPU tests of hip_kv compare with."""
import numpy as np

import hipkv

F32, F16, BF16 = hipkv.F32, hipkv.F16, hipkv.BF16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # relative, of one rounding
BYTES = {F32: 4, F16: 2, BF16: 2}


def to_type(x, ty):
    """x as the type's array (bf16: its upper 16 bits, rounded to nearest even)."""
    x = np.ascontiguousarray(x, np.float32)
    if ty == F32:
        return x
    if ty == F16:
        return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_type(a, ty):
    if ty == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def np_dtype(ty):
    return (np.float32, np.float16, np.uint16)[ty]


def rotate(x, pos, freq, mag, layout):
    """x [T][heads][D] float64, rows at pos [T]."""
    x = np.asarray(x, np.float64)
    n = len(freq)
    a = np.asarray(pos, np.float64)[:, None] * freq[None]
    c, s = (np.cos(a) * mag)[:, None], (np.sin(a) * mag)[:, None]
    y = x.copy()
    i1, i2 = ((slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if layout == hipkv.PAIRS
              else (slice(0, n), slice(n, 2 * n)))
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    return y


def quantize(x):
    """(codes 0 .. 15, float16 scales) of the groups x [...][n], float32."""
    x = np.asarray(x, np.float32)
    nan = np.isnan(x).any(-1)
    z = np.where(np.isnan(x), 0, x)
    lo, hi = z.min(-1), z.max(-1)
    m = np.where(hi > -lo, hi, lo)
    d = np.clip(m * np.float32(-0.125), -65504, 65504).astype(np.float16)
    w = d.astype(np.float64)[..., None]
    with np.errstate(invalid="ignore"):
        q = np.floor(z.astype(np.float64) / np.where(w == 0, 1, w) + 8.5)
    q = np.where(w == 0, 8, np.clip(q, 0, 15)).astype(np.uint8)
    return q, np.where(nan, np.float16(np.nan), d)


class Pool:
    """A cache's memory as the layout of include/hip_kv.h has it, on the host."""

    def __init__(self, pages, page, KH, D, fill=0xff):
        self.pages, self.page, self.KH, self.D = pages, page, KH, D
        self.bytes = np.full((pages, KH, page // 32, 34 * D + 64), fill, np.uint8)

    def _bit(self, j):
        return 2 + 4 * (j // 2) + 16 * (j % 2)

    def _key_words(self, r):
        D, P = self.D, min(4, self.D // 32)
        c = np.arange(D)
        g, part = c // 32, c % 32 // 8
        w = ((r // 16 * (D // 32 // P) + g // P) * 64 + 16 * part + r % 16) * P + g % P
        return w, self._bit(c % 8)

    def _value_words(self, r):
        c = np.arange(self.D)
        w = 4 * self.D + (c // 64 * 64 + r % 16 // 4 * 16 + c % 16) * 4 + c // 16 % 4
        return w, np.full(self.D, self._bit(r % 4 + 4 * (r // 16)))

    @staticmethod
    def _put(words, w, bit, code):
        for i, b, q in zip(w, bit, code):
            v = int(words[i]) | int(words[i]) << 32
            v = v & ~(15 << int(b)) | int(q) << int(b)
            u = v & 0xffffffff
            if b > 28:  # the upper bits of the code wrap into the word's lowest
                keep = (1 << (int(b) - 28)) - 1
                u = u & ~keep | (int(q) >> (32 - int(b)))
            words[i] = u

    @staticmethod
    def _get(words, w, bit):
        v = words[w].astype(np.uint64)
        return ((v | v << np.uint64(32)) >> bit.astype(np.uint64) & np.uint64(15)).astype(np.int64)

    def store(self, table, p, k, v):
        """Row p of the sequence with pages `table`: k, v [KH][D] float32."""
        pg, t, r, D = int(table[p // self.page]), p % self.page // 32, p % 32, self.D
        for h in range(self.KH):
            tile = self.bytes[pg, h, t]
            words, half = tile.view(np.uint32), tile[32 * D:].view(np.float16)
            q, d = quantize(k[h].reshape(-1, 32))
            self._put(words, *self._key_words(r), q.ravel())
            half[r * (D // 32):(r + 1) * (D // 32)] = d
            q, d = quantize(v[h][None])
            self._put(words, *self._value_words(r), q.ravel())
            half[D + r] = d[0]

    def load(self, table, p):
        """(k, v) [KH][D] float64 that row p stands for."""
        pg, t, r, D = int(table[p // self.page]), p % self.page // 32, p % 32, self.D
        k, v = np.empty((2, self.KH, D))
        for h in range(self.KH):
            tile = self.bytes[pg, h, t]
            words, half = tile.view(np.uint32), tile[32 * D:].view(np.float16).astype(np.float64)
            k[h] = (self._get(words, *self._key_words(r)) - 8) * np.repeat(
                half[r * (D // 32):(r + 1) * (D // 32)], 32)
            v[h] = (self._get(words, *self._value_words(r)) - 8) * half[D + r]
        return k, v

    def random(self, rng, scale=0.25):
        """Codes and finite scales of no particular rows."""
        D = self.D
        self.bytes[..., :32 * D] = rng.integers(0, 256, self.bytes[..., :32 * D].shape, np.uint8)
        d = (scale * (0.5 + rng.random(self.bytes.shape[:3] + (D + 32,)))
             * rng.choice((-1.0, 1.0), self.bytes.shape[:3] + (D + 32,)))
        self.bytes[..., 32 * D:] = d.astype(np.float16).view(np.uint8)


def attend(q, k, v, p, scale, window):
    """One query row [H][D] at position p over k, v [len][KH][D]: (out [H][D],
    sum of p |v| [H][D], largest logit bound [H])."""
    H, KH = q.shape[0], k.shape[1]
    lo, hi = (max(0, p + 1 - window) if window else 0), min(p + 1, len(k))
    out, mass, size = np.zeros_like(q), np.zeros_like(q), np.zeros(H)
    if hi <= lo:
        return out, mass, size
    for h in range(H):
        kk, vv = k[lo:hi, h // (H // KH)], v[lo:hi, h // (H // KH)]
        x = scale * (kk @ q[h])
        size[h] = abs(scale) * (np.abs(kk) @ np.abs(q[h])).max()
        with np.errstate(invalid="ignore"):
            w = np.exp(x - x.max())
        w /= w.sum()
        out[h], mass[h] = w @ vv, w @ np.abs(vv)
    return out, mass, size
