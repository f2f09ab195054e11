"""What the calls of hip_f8.h launch, over the fake runtime: one kernel each, nothing where
there are no rows, and nothing where a launch would have 2^32 threads or more."""
import pytest

from test_host_paths import on_fake

BODY = """
import hipf8
from hipf8 import F32, F16, BF16
A = 1 << 20  # an address that no call reads
def rows(n, k=128):
    return hipf8.Rows(A, -(-k // 16) * 16, A, max(n, 1), n, k)
def mat(n, k=128, count=1):
    return hipf8.Mat(A, -(-k // 16) * 16, A, -(-k // 128), n, k, count, n * -(-k // 16) * 16, 1 << 20)
def mul(n, ty=BF16, out=16, k=128, gated=False):
    hipf8.mul(rows(n, k), mat(out, k), mat(out, k) if gated else None, ty, A, -(-out // 8) * 8)
def group(n, ty=BF16, out=16, k=128, experts=4, gated=False):
    hipf8.group_mul(rows(n, k), None, A, n, mat(out, k, experts), mat(out, k, experts) if gated else None, ty, A,
                    -(-out // 8) * 8)
def quantize(n, ty=BF16, k=128):
    hipf8.quantize(ty, A, -(-k // 8) * 8, rows(n, k))
def combine(n, ty=BF16, topk=1, k=128):
    hipf8.combine(ty, A, k, n, A, A, n, topk, k, 0, 0, 2 * A, k)
def sort(n, topk=1, experts=8):
    hipf8.sort(A, n, topk, experts, A, 2 * A, 3 * A)
"""



@pytest.mark.parametrize("call,kernel", (
    ("quantize(5)", "k_f8_quantize"), ("sort(5)", "k_f8_sort"), ("sort(0)", "k_f8_sort"),
    ("combine(5)", "k_f8_combine"), ("mul(1)", "k_f8_few"), ("mul(16, F32)", "k_f8_few"),
    ("mul(100, BF16, 4096, 1024)", "k_f8_mid"), ("mul(9000, F16, 4096, 1024)", "k_f8_tile"),
    ("mul(9000, F16, 4096, 1024, True)", "k_f8_tile"), ("mul(9000, F32, 4096, 1024)", "k_f8_tile"),
    ("group(4)", "k_f8_few"), ("group(70)", "k_f8_few"), ("group(9000, BF16, 4096, 1024)", "k_f8_tile"),
    ("group(9000, F32, 4096, 1024, 64, True)", "k_f8_")))
def test_one_kernel_a_call(call, kernel):
    on_fake(BODY + f"""
names = kernels(lambda: {call})
print(names)
assert names.count("k_f8_") == 1 and {kernel!r} in names
""")


@pytest.mark.parametrize("call", ("quantize(0)", "combine(0)", "mul(0)", "group(0)"))
def test_no_rows_no_kernel(call):
    on_fake(BODY + f'assert "k_f8" not in kernels(lambda: {call})')


# 256 threads quantize four rows of 512 channels and sum up one of 2048 values in 16 bits
@pytest.mark.parametrize("call,most,more", (
    ("quantize({}, k=256)", 4 * (2 ** 24 - 1), 4), ("combine({}, k=2048)", 2 ** 24 - 1, 1),
    ("mul({}, out=200000, k=2000)", 100000, 2 ** 30),
    ("group({}, F32, out=40000, k=2000, experts=1000)", 3000, 2 ** 30)))
def test_too_many_threads(call, most, more):
    on_fake(BODY + f"""
assert "k_f8" in kernels(lambda: {call.format(most)})
def refused():
    try:
        {call.format(most + more)}
        raise SystemExit("taken")
    except hipmoe.HipMoeError as e:
        assert "too many rows" in str(e), e
assert "k_f8" not in kernels(refused)
""")
