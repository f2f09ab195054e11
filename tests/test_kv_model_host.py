"""The host side of models on 4-bit caches (hip_lm_batch_new_kv4): refusals, and
what a batch launches and allocates over the fake runtime."""
import pytest

import hiplm
from test_host_paths import TINY, on_fake


def test_refuses_no_model():
    for n in (0, 1, 4097):
        assert not hiplm._bind().hip_lm_batch_new_kv4(None, n)
        assert "lm_batch_new" in hiplm.last_error()


@pytest.mark.parametrize("n", (0, 4097))
def test_refuses_a_count_of_sequences(n):
    on_fake(f"""
    M = hiplm.LmModel({TINY}, 64)
    try:
        hiplm.LmBatch(M, {n}, kv4=True)
        raise SystemExit("taken")
    except hipmoe.HipMoeError as e:
        assert "1 .. 4096" in str(e), e
    """)


@pytest.mark.parametrize("context", (63, 64, 200))
def test_steps_prompts_and_the_context(context):
    """Decoding and generating go through the 4-bit kernels alone, up to the context
    and not past it."""
    on_fake(f"""
    M = hiplm.LmModel({TINY}, {context})
    B = hiplm.LmBatch(M, 3, kv4=True)
    ids = np.arange(3, dtype=np.int32)
    got = kernels(lambda: B.decode(ids))
    assert "k_kv_append" in got and "k_kv_attn" in got and "k_lm_attn" not in got, got
    B.reset()
    got = kernels(lambda: B.generate(np.tile(np.arange(50, dtype=np.int32), (3, 1)), {context} - 50))
    assert "k_kv_append" in got and "k_kv_attn" in got and "k_lm_pf" not in got, got
    for call in (lambda: B.decode(ids), lambda: B.generate(ids[:, None], 0)):
        try:
            call()
            raise SystemExit("went past the context")
        except hipmoe.HipMoeError as e:
            assert "do not fit" in str(e), e
    B.reset()
    B.decode(ids)
    B.free()
    M.free()
    """)


def test_allocations_that_fail():
    """Each allocation of a new batch and of its first prompts in turn: refused with
    a message, and the next try has what it needs."""
    on_fake(f"""
    M = hiplm.LmModel({TINY}, 640)
    ids = np.tile(np.arange(9, dtype=np.int32), (3, 1))
    def run():
        B = hiplm.LmBatch(M, 3, kv4=True)
        B.generate(ids, 2)
        B.free()
    hiplm.LmBatch(M, 2).free()
    F.fake_sizes()
    run()
    sizes = sorted({{int(n) for n in F.fake_sizes().split()}})
    assert len(sizes) > 8, sizes
    failed = 0
    for n in sizes:
        F.fake_fail_size(n)
        try:
            run()
        except hipmoe.HipMoeError as e:
            failed += 1
        F.fake_fail_size(0)
        run()
    assert failed > 6, (failed, sizes)
    """)
