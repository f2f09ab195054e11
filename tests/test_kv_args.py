"""What the calls of hip_kv.h refuse, and the frequencies of hip_rope_freqs: on
the CPU.  Every refusal comes before anything is enqueued."""
import ctypes as C
import math
import os
import re

import numpy as np
import pytest

import hipkv
import hipmoe
from common import REPO

DEV = 1 << 20  # an aligned address that no call reads


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(REPO, "include", "hip_kv.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = {n for n in re.findall(r"\b(hip_[a-z_0-9]*)\s*\(", text)}
    assert len(names) == 7
    assert not [n for n in names if not hasattr(hipmoe.lib(), n)]


@pytest.mark.parametrize("rot", (2, 6, 64, 128))
def test_freqs(rot):
    i = np.arange(rot // 2)
    plain = 1e4 ** (-2.0 * i / rot)
    f, mag = hipkv.rope_freqs(rot, 1e4)
    assert mag == 1 and np.allclose(f, plain, rtol=1e-14)
    f, mag = hipkv.rope_freqs(rot, 1e4, hipkv.LINEAR, 8.0)
    assert mag == 1 and np.allclose(f, plain / 8, rtol=1e-14)
    f, mag = hipkv.rope_freqs(rot, 1e4, hipkv.NTK, 8.0)
    assert mag == 1 and f[0] == 1
    if rot > 2:  # the slowest pair is stretched by the whole factor
        assert np.isclose(f[-1], plain[-1] / 8, rtol=1e-12)
    f, mag = hipkv.rope_freqs(rot, 1e4, hipkv.YARN, 8.0, 4096.0)
    assert np.isclose(mag, 0.1 * math.log(8) + 1)
    turns = 4096 * plain / (2 * math.pi)
    # pairs past the ramp's ends, which are rounded outwards by a pair
    step = 1e4 ** (2.0 / rot)
    fast, slow = turns > 32 * step, turns < 1 / step
    assert np.allclose(f[fast], plain[fast], rtol=1e-14)
    assert np.allclose(f[slow], plain[slow] / 8, rtol=1e-14)
    assert np.all(f <= plain * (1 + 1e-14)) and np.all(f >= plain / 8 * (1 - 1e-14))


@pytest.mark.parametrize("args,msg", (
    ((3, 1e4), "rotated channels"), ((0, 1e4), "rotated channels"), ((2048, 1e4), "rotated channels"),
    ((64, 1.0), "theta"), ((64, math.nan), "theta"), ((64, math.inf), "theta"),
    ((64, 1e4, 4, 2.0), "scaling"), ((64, 1e4, -1, 2.0), "scaling"),
    ((64, 1e4, hipkv.LINEAR, 0.5), "factor"), ((64, 1e4, hipkv.NTK, math.inf), "factor"),
    ((64, 1e4, hipkv.YARN, 2.0, 0.0), "context"), ((64, 1e4, hipkv.YARN, 2.0, 99.0, 1.0, 2.0), "turns"),
    ((64, 1e4, hipkv.YARN, 2.0, 99.0, 4.0, -2.0), "turns"),
))
def test_freqs_refuses(args, msg):
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.rope_freqs(*args)
    L = hipkv._bind()
    m = C.c_double()
    assert L.hip_rope_freqs(64, 1e4, 0, 1.0, 0.0, 0.0, 0.0, None, C.byref(m)) == 0
    assert "NULL" in hipmoe.last_error()


@pytest.mark.parametrize("page,KH,D,size", (
    (32, 1, 64, 2240), (64, 8, 128, 2 * 8 * 4416), (1024, 4096, 256, 32 * 4096 * 8768),
    (16, 1, 64, 0), (48, 1, 64, 0), (2048, 1, 64, 0), (32, 0, 64, 0), (32, 4097, 64, 0),
    (32, 1, 96, 0), (32, 1, 512, 0), (0, 1, 64, 0)))
def test_page_bytes(page, KH, D, size):
    assert hipkv.page_bytes(page, KH, D) == size


def rope(**kw):
    a = dict(rot=64, layout=0, freq=DEV, mag=1.0)
    a.update(kw)
    return hipkv.Rope(*a.values())


@pytest.mark.parametrize("change,msg", (
    (dict(R=None), "NULL"), (dict(x=None), "NULL"), (dict(out=None), "NULL"), (dict(pos=None), "NULL"),
    (dict(ty=3), "type"), (dict(ty=-1), "type"), (dict(heads=0), "heads"), (dict(D=0), "heads"),
    (dict(D=1025, xs=5000, os=5000), "heads"), (dict(heads=65537), "heads"),
    (dict(R=rope(rot=63)), "rotated"), (dict(R=rope(rot=0)), "rotated"), (dict(R=rope(rot=130)), "rotated"),
    (dict(R=rope(layout=2)), "layout"), (dict(R=rope(freq=None)), "frequencies"),
    (dict(R=rope(freq=DEV + 4)), "frequencies"), (dict(rows=1 << 31), "rows"),
    (dict(xs=511), "apart"), (dict(os=511), "apart"), (dict(xs=1 << 40), "apart"),
    (dict(x=DEV + 2), "misaligned"), (dict(out=DEV + 1), "misaligned"), (dict(pos=DEV + 2), "misaligned"),
    (dict(out=DEV, os=520), "in place"),
))
def test_rope_refuses(change, msg):
    a = dict(R=rope(), ty=0, x=DEV, xs=512, out=2 * DEV, os=512, rows=4, heads=4, D=128, pos=DEV)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.rope(*a.values())


def cache(**kw):
    a = dict(pool=DEV, pages=8, page=32, kv_heads=2, head_len=64, err=None)
    a.update(kw)
    return hipkv.Cache(*a.values())


def batch(**kw):
    a = dict(nseq=2, rows=6, max_rows=4, max_len=64, row_start=DEV, len=DEV, table=DEV, table_stride=2)
    a.update(kw)
    return hipkv.Batch(*a.values())


BAD_ARGS = (
    (None, batch(), "NULL cache"), (cache(), None, "NULL cache"),
    (cache(page=33), batch(), "pages of"), (cache(head_len=80), batch(), "pages of"),
    (cache(kv_heads=0), batch(), "pages of"), (cache(pages=1 << 31), batch(), "pages"),
    (cache(pool=None), batch(), "NULL pool"), (cache(pool=DEV + 8), batch(), "misaligned"),
    (cache(err=DEV + 2), batch(), "misaligned"),
    (cache(), batch(nseq=65536), "sequences"), (cache(), batch(max_rows=7), "rows"),
    (cache(), batch(rows=1 << 31), "rows"), (cache(), batch(max_len=1 << 31), "below"),
    (cache(), batch(len=None), "NULL"), (cache(), batch(table=None), "NULL"),
    (cache(), batch(len=DEV + 1), "misaligned"), (cache(), batch(table=DEV + 2), "misaligned"),
    (cache(), batch(row_start=DEV + 2), "misaligned"),
    (cache(), batch(table_stride=1), "entries"), (cache(), batch(max_len=65), "entries"),
    (cache(), batch(row_start=None), "more than"),
    (cache(kv_heads=4096), batch(nseq=65535, rows=(1 << 31) - 1, max_rows=1 << 20), "too many"),
)


@pytest.mark.parametrize("C_,B,msg", BAD_ARGS)
def test_every_call_refuses_bad_caches_and_batches(C_, B, msg):
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.append(C_, B, 0, DEV, DEV, 4096 * 256)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.read(C_, B, 0, DEV, DEV, 4096 * 256)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.attn(C_, B, 0, DEV, 4096 * 256, 4096, DEV, 4096 * 256, 1.0, 0, DEV, 1 << 40)
    assert hipkv.attn_ws(C_, B, 4096) == 0 and re.search(msg, hipmoe.last_error())


@pytest.mark.parametrize("change,msg", (
    (dict(type=7), "type"), (dict(k=None), "NULL k"), (dict(v=None), "NULL v"),
    (dict(k=DEV + 8), "16-byte"), (dict(kv_stride=127), "apart"), (dict(kv_stride=130), "multiple of 16"),
    (dict(rope=rope(rot=66)), "rotated"), (dict(rope=None), "without a rotation"),
    (dict(heads=0), "query heads"), (dict(heads=70000), "query heads"), (dict(q_out=None), "NULL q_out"),
    (dict(q=DEV + 4), "16-byte"), (dict(q_stride=255), "apart"), (dict(q_out_stride=258), "multiple"),
    (dict(q_out=3 * DEV, q_out_stride=260), "in place"), (dict(pos=DEV + 1), "misaligned"),
))
def test_append_refuses(change, msg):
    a = dict(cache=cache(), batch=batch(), type=0, k=DEV, v=2 * DEV, kv_stride=128, rope=rope(), pos=None,
             q=3 * DEV, q_stride=256, heads=4, q_out=4 * DEV, q_out_stride=256)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.append(**a)


@pytest.mark.parametrize("change,msg", (
    (dict(type=3), "type"), (dict(k=None), "NULL k"), (dict(v=None), "NULL v"), (dict(stride=120), "apart"),
    (dict(type=1, stride=132), "multiple of 16"), (dict(v=DEV + 4), "16-byte"),
))
def test_read_refuses(change, msg):
    a = dict(cache=cache(), batch=batch(), type=0, k=DEV, v=DEV, stride=128)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.read(**a)


@pytest.mark.parametrize("change,msg", (
    (dict(type=3), "type"), (dict(heads=0), "query heads"), (dict(heads=3), "query heads"),
    (dict(heads=65538), "query heads"), (dict(q=None), "NULL q"), (dict(out=None), "NULL out"),
    (dict(q_stride=255), "apart"), (dict(out_stride=258), "multiple"), (dict(q=DEV + 8), "16-byte"),
    (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(out=DEV, out_stride=260), "in place"), (dict(ws=None), "workspace"), (dict(ws=DEV + 8), "workspace"),
    (dict(ws_bytes=15), "workspace"),
    (dict(batch=batch(rows=1 << 30, max_rows=1 << 30, nseq=1)), "too many"),
))
def test_attn_refuses(change, msg):
    b = batch(max_len=4096, table_stride=128)
    a = dict(cache=cache(), batch=b, type=0, q=DEV, q_stride=256, heads=4, out=2 * DEV, out_stride=256,
             scale=0.1, window=0, ws=DEV, ws_bytes=1 << 30)
    assert 16 < hipkv.attn_ws(a["cache"], b, 4) < 1 << 30
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipkv.attn(**a)


def test_without_a_device():
    if hipmoe.hip().device_count() > 0:
        pytest.skip("a GPU is visible")
    for call in (lambda: hipkv.rope(rope(), 0, DEV, 512, 2 * DEV, 512, 4, 4, 128, DEV),
                 lambda: hipkv.append(cache(), batch(), 0, DEV, DEV, 128),
                 lambda: hipkv.read(cache(), batch(), 0, DEV, DEV, 128),
                 lambda: hipkv.attn(cache(), batch(), 0, DEV, 256, 4, DEV, 256, 1.0, 0, DEV, 1 << 30)):
        with pytest.raises(hipmoe.HipMoeError, match="no HIP device"):
            call()


def test_calls_without_rows_do_nothing():
    for b in (batch(nseq=0), batch(rows=0, max_rows=0), batch(nseq=0, len=None, table=None)):
        hipkv.append(cache(), b, 0, None, None, 0)
        hipkv.read(cache(), b, 0, None, None, 0)
        hipkv.attn(cache(), b, 0, None, 0, 4, None, 0, 1.0)
        assert hipkv.attn_ws(cache(), b, 4) == 0
    hipkv.rope(rope(), 0, DEV, 512, 2 * DEV, 512, 0, 4, 128, DEV)


@pytest.mark.parametrize("D", (64, 128, 256))
@pytest.mark.parametrize("nseq,KH,G,rows", ((1, 8, 4, 1), (16, 8, 4, 1), (64, 8, 4, 1), (64, 8, 4, 4), (256, 2, 8, 2),
                                            (257, 2, 8, 1), (100, 16, 1, 16), (3, 1, 1, 5), (1000, 8, 4, 1)))
def test_a_workspace_serves_shorter_bounds(D, nseq, KH, G, rows):
    """What a step's attention needs grows with the bound of the lengths."""
    before = 0
    for max_len in list(range(1, 500, 31)) + list(range(500, 40000, 517)):
        c = cache(kv_heads=KH, head_len=D, page=64)
        b = batch(nseq=nseq, rows=nseq * rows, max_rows=rows, max_len=max_len, table_stride=700, row_start=None)
        ws = hipkv.attn_ws(c, b, KH * G)
        assert ws >= before, max_len
        before = ws
    assert before > 0
