"""The forms that products of 8-bit floating point take (f8_mul_plan of
llm.c_amd/csrc/f8_internal.h): on the CPU."""
import ctypes as C

import pytest

import hipf8
import hipmoe

_vp, _l, _i, _sz = C.c_void_p, C.c_long, C.c_int, C.c_size_t
FORMS = ("FEW_LONG", "FEW_WIDE", "FEW_GATED", "FEW_32", "MID_32", "MID_64", "MID_128", "MID_SQUARE", "TILE_64",
         "TILE_128", "TILE_128F", "TILE_256")


class Args(C.Structure):
    """f8_mul_args"""
    _fields_ = [("x", _vp), ("xs", _vp), ("w", _vp * 2), ("ws", _vp * 2), ("frm", _vp), ("start", _vp), ("add", _vp),
                ("out", _vp), ("x_stride", _l), ("xs_stride", _l), ("w_stride", _l * 2), ("ws_stride", _l * 2),
                ("w_step", _l * 2), ("ws_step", _l * 2), ("add_stride", _l), ("out_stride", _l), ("x_rows", _i),
                ("rows", _i), ("n", _i), ("k", _i), ("count", _i)]


class Plan(C.Structure):
    """f8_plan"""
    _fields_ = [("type", _i), ("form", _i), ("row_tiles", _sz), ("n_tiles", _sz), ("threads", _i)]


def plan(type, rows, n, k, gated=False, experts=0, gather=False, x_rows=None):
    """(form's name, plan) of a product; experts 0: a dense one."""
    A = 1 << 20
    a = Args(rows=rows, n=n, k=k, count=max(1, experts), x_rows=rows if x_rows is None else x_rows,
             x_stride=-(-k // 16) * 16, start=A if experts else None, frm=A if gather else None)
    a.w[0], a.w[1] = A, A if gated else None
    p = Plan(type=type)
    f = hipmoe.lib().f8_mul_plan
    f.restype, f.argtypes = None, [C.POINTER(Args), C.POINTER(Plan)]
    f(C.byref(a), C.byref(p))
    return FORMS[p.form], p


def form(*args, **kw):
    return plan(*args, **kw)[0]


TILES = {"FEW_LONG": (16, 16), "FEW_WIDE": (16, 16), "FEW_GATED": (16, 32), "FEW_32": (32, 32), "MID_32": (32, 128),
         "MID_64": (64, 64), "MID_128": (64, 128), "MID_SQUARE": (128, 128), "TILE_64": (64, 128),
         "TILE_128": (128, 128), "TILE_128F": (128, 128), "TILE_256": (256, 256)}


@pytest.mark.parametrize("type", (hipf8.F32, hipf8.F16, hipf8.BF16))
@pytest.mark.parametrize("gated", (False, True))
def test_tiles_cover_every_product(type, gated):
    seen = set()
    for experts in (0, 1, 7, 64, 1000):
        for rows in (1, 8, 16, 17, 40, 100, 333, 1000, 5000, 70000):
            for n in (1, 16, 100, 1000, 4096, 14336, 200000):
                for k in (1, 128, 300, 1024, 4096, 20000):
                    name, p = plan(type, rows, n, k, gated, experts)
                    seen.add(name)
                    bt, bn = TILES[name]
                    if gated and name[:3] != "FEW":
                        bn //= 2
                    assert p.n_tiles == -(-n // bn)
                    # whatever the experts' rows: their tiles, each rounded up, are no more
                    most = -(-rows // bt) if not experts else rows // bt + min(rows, experts)
                    assert p.row_tiles == most
                    assert p.threads in (256, 512)
    never = {"FEW_GATED" if not gated else "FEW_WIDE"} | (
        {"TILE_128", "TILE_256"} if type == hipf8.F32 else {"MID_SQUARE", "TILE_128F"})
    assert seen == set(FORMS) - never


def test_streams_only_where_their_next_tile_can_be_asked_for():
    assert form(hipf8.BF16, 8192, 8192, 4096) == "TILE_256"
    assert form(hipf8.BF16, 8192, 8192, 256) != "TILE_256"
    big = dict(experts=8, gated=True, gather=True)
    assert form(hipf8.BF16, 8192, 14336, 4096, x_rows=4096, **big) == "TILE_256"
    assert form(hipf8.BF16, 8192, 14336, 4096, x_rows=(1 << 20) - 300, **big) == "TILE_256"
    assert form(hipf8.BF16, 8192, 14336, 4096, x_rows=1 << 20, **big) != "TILE_256"
