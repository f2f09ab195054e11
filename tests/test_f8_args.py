"""What the calls of hip_f8.h refuse: on the CPU.  Every refusal comes before anything
is enqueued."""
import os
import re

import pytest

import hipf8
import hipmoe
from common import REPO

DEV = 1 << 20  # an aligned address that no call reads


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(REPO, "include", "hip_f8.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = {n for n in re.findall(r"\b(hip_[a-z_0-9]*)\s*\(", text)}
    assert len(names) == 5
    assert not [n for n in names if not hasattr(hipmoe.lib(), n)]


def rows(**kw):
    a = dict(codes=DEV, stride=256, scale=DEV, scale_stride=8, rows=8, k=256)
    a.update(kw)
    return hipf8.Rows(*a.values())


def mat(**kw):
    a = dict(codes=DEV, stride=256, scale=DEV, scale_stride=2, n=300, k=256, count=1, step=0, scale_step=0)
    a.update(kw)
    return hipf8.Mat(*a.values())


def mats(**kw):
    return mat(**dict(dict(count=4, step=300 * 256, scale_step=6), **kw))


BAD_ROWS = (
    (rows(k=0), "channels"), (rows(k=(1 << 20) + 1, stride=1 << 21), "channels"),
    (rows(rows=(1 << 31) - 65536, scale_stride=1 << 31), "rows"),
    (rows(codes=None), "NULL"), (rows(scale=None), "NULL"), (rows(stride=255), "apart"), (rows(stride=264), "apart"),
    (rows(stride=(1 << 24) + 16), "apart"), (rows(codes=DEV + 8), "16-byte"), (rows(scale=DEV + 2), "4-byte"),
    (rows(scale_stride=7), "scales of"), (rows(scale_stride=(1 << 31) + 1), "scales of"))

BAD_MATS = (
    (dict(n=0), "columns"), (dict(n=(1 << 31) - 65536), "columns"), (dict(k=0), "columns"),
    (dict(k=(1 << 20) + 1), "columns"), (dict(count=0), "matrices"), (dict(count=1025), "matrices"),
    (dict(codes=None), "NULL"), (dict(scale=None), "NULL"), (dict(stride=255), "apart"), (dict(stride=264), "apart"),
    (dict(codes=DEV + 4), "16-byte"), (dict(scale=DEV + 1), "4-byte"), (dict(scale_stride=1), "scales"),
    (dict(scale_stride=(1 << 31) + 1), "scales"), (dict(stride=(1 << 24) + 16), "apart"))


@pytest.mark.parametrize("X,msg", BAD_ROWS)
def test_every_call_refuses_bad_rows(X, msg):
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.quantize(0, DEV, 1 << 21, X)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.mul(X, mat(), None, 0, DEV, 512)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.group_mul(X, None, DEV, 4, mats(), None, 0, DEV, 512)


@pytest.mark.parametrize("change,msg", BAD_MATS)
def test_products_refuse_bad_matrices(change, msg):
    for W, U in ((mat(**change), None), (mat(), mat(**change))):
        with pytest.raises(hipmoe.HipMoeError, match=msg):
            hipf8.mul(rows(), W, U, 0, DEV, 512)
    for W, U in ((mats(**change), None), (mats(), mats(**change))):
        with pytest.raises(hipmoe.HipMoeError, match=msg):
            hipf8.group_mul(rows(), None, DEV, 4, W, U, 0, DEV, 512)


@pytest.mark.parametrize("change", (dict(step=300 * 256 + 8), dict(step=(1 << 40) + 16), dict(scale_step=(1 << 40) + 1)))
def test_group_mul_refuses_bad_steps(change):
    with pytest.raises(hipmoe.HipMoeError, match="apart"):
        hipf8.group_mul(rows(), None, DEV, 4, mats(**change), None, 0, DEV, 512)


def test_quantize_refuses():
    def call(**kw):
        a = dict(type=0, x=DEV, x_stride=256, rows=rows())
        a.update(kw)
        hipf8.quantize(**a)
    for change, msg in ((dict(type=3), "type"), (dict(rows=None), "NULL rows"), (dict(x=None), "NULL x"),
                        (dict(x_stride=252), "apart"), (dict(type=1, x_stride=260), "multiple of 16"),
                        (dict(x=DEV + 8), "16-byte"), (dict(x_stride=1 << 32), "apart"),
                        (dict(rows=rows(rows=1 << 28, scale_stride=1 << 28)), "too many")):
        with pytest.raises(hipmoe.HipMoeError, match=msg):
            call(**change)


@pytest.mark.parametrize("change,msg", (
    (dict(rows=None), "NULL"), (dict(mat=None), "NULL"), (dict(type=-1), "type"), (dict(mat=mat(k=255)), "columns"),
    (dict(up=mat(n=299)), "up of"), (dict(up=mat(k=255)), "up of"), (dict(mat=mats()), "matrices"),
    (dict(out=None), "NULL out"), (dict(out_stride=299), "apart"), (dict(out_stride=301), "multiple of 16"),
    (dict(out=DEV + 4), "16-byte"), (dict(add=DEV + 4), "16-byte"), (dict(add_stride=296), "apart"),
    (dict(add_stride=306), "multiple"), (dict(add=2 * DEV, add_stride=308), "in place"),
    (dict(add=2 * DEV, add_stride=0), "in place"), (dict(up=mat()), "addend"),
    (dict(rows=rows(rows=1 << 30, scale_stride=1 << 30), mat=mat(n=1 << 20), out_stride=1 << 20, add=None), "too many"),
))
def test_mul_refuses(change, msg):
    a = dict(rows=rows(), mat=mat(), up=None, type=0, out=2 * DEV, out_stride=304, add=3 * DEV, add_stride=300)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.mul(**a)


@pytest.mark.parametrize("change,msg", (
    (dict(rows=None), "NULL"), (dict(mat=None), "NULL"), (dict(type=9), "type"), (dict(mat=mats(k=200)), "columns"),
    (dict(up=mats(count=3)), "up of"), (dict(start=None), "misaligned rows"), (dict(start=DEV + 2), "misaligned rows"),
    (dict(from_=DEV + 1), "misaligned rows"), (dict(from_=None, n_rows=9), "9 rows of 8"),
    (dict(rows=rows(rows=0)), "of none"), (dict(n_rows=(1 << 31) - 65536), "below"), (dict(out=None), "NULL out"),
    (dict(out_stride=299), "apart"), (dict(out=DEV + 8), "16-byte"),
))
def test_group_mul_refuses(change, msg):
    a = dict(rows=rows(), from_=DEV, start=DEV, n_rows=30, mat=mats(), up=None, type=0, out=2 * DEV, out_stride=304)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.group_mul(**a)


@pytest.mark.parametrize("change,msg", (
    (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(topk=0), "slots"), (dict(topk=1025), "slots"),
    (dict(tokens=1 << 30), "pairs"), (dict(ids=None), "NULL"), (dict(start=None), "NULL"), (dict(from_=None), "NULL"),
    (dict(pos=None), "NULL"), (dict(tokens=0, start=None), "NULL"), (dict(ids=DEV + 2), "misaligned"),
    (dict(start=DEV + 1), "misaligned"), (dict(from_=DEV + 2), "misaligned"), (dict(pos=DEV + 3), "misaligned"),
))
def test_sort_refuses(change, msg):
    a = dict(ids=DEV, tokens=5, topk=2, experts=8, start=DEV, from_=DEV, pos=DEV)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.sort(**a)


@pytest.mark.parametrize("change,msg", (
    (dict(type=3), "type"), (dict(topk=0), "slots"), (dict(topk=1025), "slots"), (dict(tokens=1 << 30), "pairs"),
    (dict(n=0), "values"), (dict(n=(1 << 31) - 65536), "values"), (dict(y_rows=1 << 31), "rows"),
    (dict(pos=None), "NULL"), (dict(w=None), "NULL"), (dict(pos=DEV + 2), "misaligned"), (dict(w=DEV + 1), "misaligned"),
    (dict(y=None), "NULL y"), (dict(y_stride=299), "apart"), (dict(y=DEV + 8), "16-byte"), (dict(out=None), "NULL out"),
    (dict(out_stride=302), "multiple"), (dict(add=DEV + 8), "16-byte"), (dict(add_stride=200), "apart"),
    (dict(add=2 * DEV, add_stride=308), "in place"), (dict(add=2 * DEV, add_stride=0), "in place"),
    (dict(tokens=1 << 28, n=1 << 16, y_stride=1 << 16, out_stride=1 << 16, add=None), "too many"),
))
def test_combine_refuses(change, msg):
    a = dict(type=0, y=DEV, y_stride=300, y_rows=10, pos=DEV, w=DEV, tokens=5, topk=2, n=300, add=DEV, add_stride=300,
             out=2 * DEV, out_stride=304)
    a.update(change)
    with pytest.raises(hipmoe.HipMoeError, match=msg):
        hipf8.combine(**a)


CALLS = (lambda: hipf8.quantize(0, DEV, 256, rows()), lambda: hipf8.mul(rows(), mat(), mat(), 0, DEV, 304),
         lambda: hipf8.sort(DEV, 5, 2, 8, DEV, DEV, DEV),
         lambda: hipf8.group_mul(rows(), DEV, DEV, 30, mats(), None, 0, DEV, 304),
         lambda: hipf8.combine(0, DEV, 300, 10, DEV, DEV, 5, 2, 300, None, 0, DEV, 304))


def test_without_a_device():
    if hipmoe.hip().device_count() > 0:
        pytest.skip("a GPU is visible")
    for call in CALLS:
        with pytest.raises(hipmoe.HipMoeError, match="no HIP device"):
            call()


def test_calls_without_rows_do_nothing():
    none = rows(rows=0, codes=None, scale=None)
    hipf8.quantize(0, None, 0, none)
    hipf8.mul(none, mat(), None, 0, None, 0)
    hipf8.group_mul(none, None, None, 0, mats(), None, 0, None, 0)
    hipf8.combine(0, None, 0, 0, None, None, 0, 2, 300, None, 0, None, 0)
