"""ctypes binding of the rotary positions, the paged 4-bit cache and its
attention (include/hip_kv.h).

Pointers are device addresses (a torch tensor's data_ptr(), Hip.malloc's
result); strides are counted in elements.  Like hipmoe.py it only marshals
arguments and raises what the library refuses.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

import hipmoe
from hipmoe import HipMoeError, last_error

F32, F16, BF16 = 0, 1, 2
PAIRS, HALVES = 0, 1
PLAIN, LINEAR, NTK, YARN = 0, 1, 2, 3
ERR_PAGE, ERR_BATCH = 1, 2

_vp, _sz, _i32 = C.c_void_p, C.c_size_t, C.c_int


class Rope(C.Structure):
    """hip_rope: rot rotated channels, PAIRS or HALVES, frequencies (device,
    float64 [rot / 2]) and the factor of cos and sin."""
    _fields_ = [("rot", _sz), ("layout", _i32), ("freq", _vp), ("mag", C.c_double)]


class Cache(C.Structure):
    """hip_kv_cache"""
    _fields_ = [("pool", _vp), ("pages", _sz), ("page", _sz), ("kv_heads", _sz),
                ("head_len", _sz), ("err", _vp)]


class Batch(C.Structure):
    """hip_kv_batch"""
    _fields_ = [("nseq", _sz), ("rows", _sz), ("max_rows", _sz), ("max_len", _sz),
                ("row_start", _vp), ("len", _vp), ("table", _vp), ("table_stride", _sz)]


_bound = None


def _bind():
    global _bound
    if _bound is None:
        L = hipmoe.lib()
        rope, cache, batch, f64 = (C.POINTER(t) for t in (Rope, Cache, Batch, C.c_double))
        L.hip_rope_freqs.restype = _i32
        L.hip_rope_freqs.argtypes = [_sz, C.c_double, _i32, C.c_double, C.c_double, C.c_double,
                                     C.c_double, _vp, f64]
        L.hip_rope_dev.restype = _i32
        L.hip_rope_dev.argtypes = [rope, _i32, _vp, _sz, _vp, _sz, _sz, _sz, _sz, _vp, _vp]
        L.hip_kv_page_bytes.restype = _sz
        L.hip_kv_page_bytes.argtypes = [_sz, _sz, _sz]
        L.hip_kv_append_dev.restype = _i32
        L.hip_kv_append_dev.argtypes = [cache, batch, rope, _i32, _vp, _vp, _sz, _vp, _vp, _sz, _sz,
                                        _vp, _sz, _vp]
        L.hip_kv_read_dev.restype = _i32
        L.hip_kv_read_dev.argtypes = [cache, batch, _i32, _vp, _vp, _sz, _vp]
        L.hip_kv_attn_ws.restype = _sz
        L.hip_kv_attn_ws.argtypes = [cache, batch, _sz]
        L.hip_kv_attn_dev.restype = _i32
        L.hip_kv_attn_dev.argtypes = [cache, batch, _i32, _vp, _sz, _sz, _vp, _sz, C.c_float, _sz, _vp,
                                      _sz, _vp]
        _bound = L
    return _bound


def _check(rc, what):
    if rc != 1:
        raise HipMoeError(f"{what}: {last_error()}")


def rope_freqs(rot, theta, scaling=PLAIN, factor=1.0, context=0.0, fast=0.0, slow=0.0):
    """(float64 [rot / 2], mag) of hip_rope_freqs."""
    f, mag = np.zeros(max(1, rot // 2)), C.c_double(0)
    _check(_bind().hip_rope_freqs(rot, theta, scaling, factor, context, fast, slow, f.ctypes.data,
                                  C.byref(mag)), "hip_rope_freqs")
    return f, mag.value


def rope(R, type, x, x_stride, out, out_stride, rows, heads, head_len, pos, stream=None):
    _check(_bind().hip_rope_dev(R, type, x, x_stride, out, out_stride, rows, heads, head_len, pos,
                                stream), "hip_rope_dev")


def page_bytes(page, kv_heads, head_len) -> int:
    return _bind().hip_kv_page_bytes(page, kv_heads, head_len)


def append(cache, batch, type, k, v, kv_stride, rope=None, pos=None, q=None, q_stride=0, heads=0,
           q_out=None, q_out_stride=0, stream=None):
    _check(_bind().hip_kv_append_dev(cache, batch, rope, type, k, v, kv_stride, pos, q, q_stride, heads,
                                     q_out, q_out_stride, stream), "hip_kv_append_dev")


def read(cache, batch, type, k, v, stride, stream=None):
    _check(_bind().hip_kv_read_dev(cache, batch, type, k, v, stride, stream), "hip_kv_read_dev")


def attn_ws(cache, batch, heads) -> int:
    return _bind().hip_kv_attn_ws(cache, batch, heads)


def attn(cache, batch, type, q, q_stride, heads, out, out_stride, scale, window=0, ws=None, ws_bytes=0,
         stream=None):
    _check(_bind().hip_kv_attn_dev(cache, batch, type, q, q_stride, heads, out, out_stride, scale, window,
                                   ws, ws_bytes, stream), "hip_kv_attn_dev")
