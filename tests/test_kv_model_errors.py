"""What a batch on 4-bit caches says of the errors that its kernels leave in the step's
word: over the fake runtime, without page-locked memory, so that the word is read
by a copy."""
import pytest

from test_host_paths import TINY, on_fake


@pytest.mark.parametrize("word,says", ((1, "page or length"), (2, "page or length"), (3, "page or length"),
                                       (4, "out of polls"), (5, "out of polls")))
def test_errors_by_their_names(word, says):
    """HIP_KV_ERR_PAGE and _BATCH are not taken for a gather that ran out of polls; the
    word is cleared, and the next step runs."""
    on_fake(f"""
    F.fake_fail_host(1)
    M = hiplm.LmModel({TINY}, 64)
    B = hiplm.LmBatch(M, 3, kv4=True)
    F.fake_last_of.restype, F.fake_last_of.argtypes = C.c_void_p, [C.c_size_t]
    state = (C.c_int * 8).from_address(F.fake_last_of(32))
    assert list(state) == [0, 0, 0, 0, 0, 1, 0, 0], list(state)  # epoch 1
    ids = np.arange(3, dtype=np.int32)
    B.decode(ids)
    state[6] = {word}
    try:
        B.decode(ids)
        raise SystemExit("taken")
    except hipmoe.HipMoeError as e:
        assert {says!r} in str(e) and "({word})" in str(e), e
    assert state[6] == 0
    B.decode(ids)
    """)
