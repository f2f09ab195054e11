"""How the attention over the 4-bit cache cuts a call up (kv_attn_plan of
llm.c_amd/csrc/kv_internal.h), and what its launches may ask of a kernel: on the CPU."""
import ctypes as C

import pytest

import hipmoe

_vp, _i = C.c_void_p, C.c_int
MANY = 8  # waves of the widest workgroups, which heads of 256 have no instance for


class Args(C.Structure):
    """kv_args"""
    _fields_ = [("pool", _vp), ("err", _vp), ("row_start", _vp), ("len", _vp), ("table", _vp),
                ("table_stride", C.c_long), ("pages", _i), ("page_shift", _i), ("kv_heads", _i),
                ("nseq", _i), ("rows", _i), ("max_rows", _i), ("max_len", _i)]


class Plan(C.Structure):
    """kv_plan"""
    _fields_ = [("row_tiles", _i), ("wide", _i), ("rows", _i), ("slots", _i), ("waves", _i),
                ("chunk", _i), ("splits", _i), ("shares", _i), ("ws", C.c_size_t)]


def plan(D, nseq, KH, G, rows, max_len, window=0):
    a = Args(page_shift=6, pages=1, kv_heads=KH, nseq=nseq, rows=nseq * rows, max_rows=rows,
             max_len=max_len)
    p = Plan()
    f = hipmoe.lib().kv_attn_plan
    f.restype, f.argtypes = None, [C.POINTER(Args), _i, _i, _i, C.POINTER(Plan)]
    f(C.byref(a), D, KH * G, window, C.byref(p))
    return p


@pytest.mark.parametrize("D", (64, 128, 256))
@pytest.mark.parametrize("nseq,KH,G,rows", ((1, 1, 1, 1), (3, 2, 3, 1), (64, 8, 4, 1), (2, 1, 16, 5), (9, 16, 2, 300)))
@pytest.mark.parametrize("max_len", (0, 1, 32, 33, 1024, 2304, 5000, 100000))
def test_heads_of_256_have_four_waves(D, nseq, KH, G, rows, max_len):
    for window in (0, 1, 500):
        if window >= max(max_len, 1):
            continue
        p = plan(D, nseq, KH, G, rows, max_len, window)
        if p.wide:
            assert D < 256
            continue
        assert p.waves in ((4, MANY) if D < 256 else (4,))
        assert p.splits >= 1 and p.chunk >= 0
