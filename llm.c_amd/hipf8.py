"""ctypes binding of the 8-bit floating-point products (include/hip_f8.h).

Pointers are device addresses (a torch tensor's data_ptr(), Hip.malloc's
result); strides are counted in elements.  Like hipmoe.py it only marshals
arguments and raises what the library refuses.
"""
from __future__ import annotations

import ctypes as C

import hipmoe
from hipmoe import HipMoeError, last_error

F32, F16, BF16 = 0, 1, 2
BLOCK = 128

_vp, _sz, _i32 = C.c_void_p, C.c_size_t, C.c_int


class Rows(C.Structure):
    """hip_f8_rows"""
    _fields_ = [("codes", _vp), ("stride", _sz), ("scale", _vp), ("scale_stride", _sz), ("rows", _sz),
                ("k", _sz)]


class Mat(C.Structure):
    """hip_f8_mat"""
    _fields_ = [("codes", _vp), ("stride", _sz), ("scale", _vp), ("scale_stride", _sz), ("n", _sz),
                ("k", _sz), ("count", _sz), ("step", _sz), ("scale_step", _sz)]


_bound = None


def _bind():
    global _bound
    if _bound is None:
        L = hipmoe.lib()
        rows, mat = C.POINTER(Rows), C.POINTER(Mat)
        L.hip_f8_quantize_dev.restype = _i32
        L.hip_f8_quantize_dev.argtypes = [_i32, _vp, _sz, rows, _vp]
        L.hip_f8_mul_dev.restype = _i32
        L.hip_f8_mul_dev.argtypes = [rows, mat, mat, _i32, _vp, _sz, _vp, _sz, _vp]
        L.hip_f8_sort_dev.restype = _i32
        L.hip_f8_sort_dev.argtypes = [_vp, _sz, _sz, _sz, _vp, _vp, _vp, _vp]
        L.hip_f8_group_mul_dev.restype = _i32
        L.hip_f8_group_mul_dev.argtypes = [rows, _vp, _vp, _sz, mat, mat, _i32, _vp, _sz, _vp]
        L.hip_f8_combine_dev.restype = _i32
        L.hip_f8_combine_dev.argtypes = [_i32, _vp, _sz, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _vp, _sz,
                                         _vp]
        _bound = L
    return _bound


def _check(rc, what):
    if rc != 1:
        raise HipMoeError(f"{what}: {last_error()}")


def quantize(type, x, x_stride, rows, stream=None):
    _check(_bind().hip_f8_quantize_dev(type, x, x_stride, rows, stream), "hip_f8_quantize_dev")


def mul(rows, mat, up, type, out, out_stride, add=None, add_stride=0, stream=None):
    _check(_bind().hip_f8_mul_dev(rows, mat, up, type, add, add_stride, out, out_stride, stream),
           "hip_f8_mul_dev")


def sort(ids, tokens, topk, experts, start, from_, pos, stream=None):
    _check(_bind().hip_f8_sort_dev(ids, tokens, topk, experts, start, from_, pos, stream),
           "hip_f8_sort_dev")


def group_mul(rows, from_, start, n_rows, mat, up, type, out, out_stride, stream=None):
    _check(_bind().hip_f8_group_mul_dev(rows, from_, start, n_rows, mat, up, type, out, out_stride,
                                        stream), "hip_f8_group_mul_dev")


def combine(type, y, y_stride, y_rows, pos, w, tokens, topk, n, add, add_stride, out, out_stride,
            stream=None):
    _check(_bind().hip_f8_combine_dev(type, y, y_stride, y_rows, pos, w, tokens, topk, n, add, add_stride,
                                      out, out_stride, stream), "hip_f8_combine_dev")
