"""Calls of hip_kv.h whose launches would have 2^32 threads and more along a dimension:
refused before anything is enqueued, over the fake runtime."""
import pytest

from test_host_paths import on_fake

BODY = """
import hipkv
A = 1 << 20  # addresses that no call reads
def batch(rows, max_len=1 << 20):
    return hipkv.Batch(1, rows, rows, max_len, A, A, A, 1 << 20)
cache = hipkv.Cache(A, 8, 32, {KH}, 64, None)
rope = hipkv.Rope(64, 0, A, 1.0)
W = {KH} * 64
calls = dict(
    rope=lambda n: hipkv.rope(rope, 0, A, 64, 2 * A, 64, n, 1, 64, A),
    append=lambda n: hipkv.append(cache, batch(n), 0, A, A, W, rope=rope, q=A, q_stride=W, heads={KH}, q_out=A,
                                  q_out_stride=W),
    read=lambda n: hipkv.read(cache, batch(n), 0, A, A, W),
    attn=lambda n: hipkv.attn(cache, batch(n), 0, A, W, {KH}, 2 * A, W, 0.1, 0, A, 1 << 40))
call = calls[{what!r}]
assert "k_kv" in kernels(lambda: call({most}))
def refused():
    try:
        call({most} + {more})
        raise SystemExit("taken")
    except hipmoe.HipMoeError as e:
        print(e)
assert "k_kv" not in kernels(refused)
"""


@pytest.mark.parametrize("what,KH,most,more", (
    ("rope", 1, (2 ** 24 - 1) * 8, 1),           # eight rows and 256 threads a workgroup
    ("append", 64, 32 * 2 ** 20, 32 * 2 ** 20),  # 4 * 32 rows of a tile in all heads, 512 threads
    ("read", 8, 32 * (2 ** 21 - 3), 32 * 4),     # a tile of a head, 256 threads
    ("attn", 16, 32 * (2 ** 19 - 1), 64)))       # 32 rows of a head, 512 threads at most
def test_too_many_threads(what, KH, most, more):
    on_fake(BODY.format(what=what, KH=KH, most=most, more=more))
