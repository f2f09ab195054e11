"""Whole models whose caches are in 4 bits (hip_lm_batch_new_kv4): every step and
prompt through the append, the rotation and the attention of hip_kv.h together,
against the same models in numpy (kv_model.py), whose caches take the same codes.

Tolerances.  Products and experts in fp32 leave logits about 1e-6 apart (relative
L2), but a key or value as far from a border between codes takes the next one: of the
100 000 codes and more of a sequence here a few do.  Such a step is an eighth of its
group's largest, about 0.3 sigma, in one component of 128: it moves one head's output
over n rows of like weight, sigma / sqrt(n), by 0.3 sigma / n: 0.027 / sqrt(n) of it
(0.3 / sqrt(128) = 0.027), and the logits by no more: three of them are left to a
step.  Caches in fp32 would be off by 0.1 and more (numpy both).  One layer has no
products before its codes but its own: one such step is left, or FEW over long caches.
Where the experts take f16 operands (more than a few rows) they are within 1e-3, as elsewhere.
The seeds' sequences have no two experts within 4e-3 of each other at the top-k border
(numpy), where such steps could choose another one.
"""
import numpy as np
import pytest

import hiplm
import hipmoe
import kv_model
from common import model_case, rel_l2

pytestmark = pytest.mark.gpu
FLIP = 0.027
FEW = 3e-3
EXPERTS = 1e-3


def prompts_of(md, seeds, n):
    return np.stack([hiplm.synth_prompt(s, n, md["V"]) for s in seeds])


@pytest.fixture
def made():
    """Frees what a test made, last first."""
    things = []
    yield lambda x: things.append(x) or x
    for x in reversed(things):
        x.free()


def small(arch, layers, window=0):
    if arch == "olmoe":
        return hiplm.synth_olmoe(5, layers, 512, 4, 300, 8, 2, 256, hipmoe.Q8_0)
    return hiplm.synth_mixtral(6, layers, 1024, 8, 4, 300, 8, 2, 256, hipmoe.Q4_0, window=window)


@pytest.mark.parametrize("arch,window,seeds", (("olmoe", 0, (1, 45)), ("mixtral", 20, (18, 12)),
                                               ("mixtral", 0, (11, 6))))
def test_steps(arch, window, seeds, made):
    """72 steps of two layers, into a second page, grouped heads and a window."""
    md = small(arch, 2, window)
    ids = prompts_of(md, seeds, 72)
    want = [kv_model.Sequence(md, r) for r in ids]
    assert min(s.gap.min() for s in want) > 4e-3
    M = made(hiplm.LmModel(md, 100))
    B = made(hiplm.LmBatch(M, len(seeds), kv4=True))
    off = np.zeros((len(seeds), 72))
    for i in range(72):
        _, lg = B.decode(ids[:, i])
        off[:, i] = [rel_l2(lg[s], want[s].logits[i]) for s in range(len(seeds))]
    print(f"{arch}: median {np.median(off):.2e}, worst {off.max():.2e}")
    rows = np.arange(1, 73) if window == 0 else np.minimum(np.arange(1, 73), window)
    assert (off <= 3 * FLIP / np.sqrt(rows)).all(), off


@pytest.mark.parametrize("arch,window,S,n,C", (
    ("olmoe", 0, 2, 100, 128), ("olmoe", 0, 1, 2, 70), ("mixtral", 0, 2, 33, 64),
    ("mixtral", 50, 3, 129, 200), ("mixtral", 0, 4, 512, 520),
    ("olmoe", 0, 3, 1000, 1024), ("mixtral", 200, 3, 1000, 1001),
    ("olmoe", 0, 1, 2200, 2210),    # steps in pieces
    ("mixtral", 0, 130, 20, 40)))   # prompts in two groups
def test_prompts(arch, window, S, n, C, made):
    """generate's prompts (a launch for up to 2048 rows) and the step after them."""
    md = small(arch, 1, window)
    M = made(hiplm.LmModel(md, C))
    B = made(hiplm.LmBatch(M, S, kv4=True))
    ids = prompts_of(md, range(40, 40 + S), n)
    toks, _ = B.generate(ids, 0)
    assert toks.shape == (S, 1)
    nxt, lg = B.decode(toks[:, 0])
    for s in range(S):
        r = kv_model.Sequence(md, np.append(ids[s], toks[s]), rows=(n - 1, n))
        scale = np.sqrt((r.logits ** 2).sum(1))
        few = EXPERTS + max(FEW, FLIP / np.sqrt(min(n, window or n)))
        # the prompt's pick is the largest logit, or as near as they are known
        if r.gap[n - 1] > 2e-3:
            assert r.logits[0, toks[s, 0]] >= r.logits[0].max() - 2 * few * scale[0], s
        if r.gap[n] > 2e-3:
            assert rel_l2(lg[s], r.logits[1]) <= few, s
            assert r.logits[1, nxt[s]] >= r.logits[1].max() - 2 * few * scale[1], s


@pytest.mark.parametrize("name", ("olmoe_small", "mixtral_small"))
def test_replayed_steps_equal_decoded(name, made):
    """generate's captured steps (one id of prompt: no rows at once) are decode's,
    twice, and decode goes on where they ended."""
    md, *_ = model_case(name)
    M = made(hiplm.LmModel(md, 80))
    S, n = 3, 70
    B = made(hiplm.LmBatch(M, S, kv4=True))
    start = prompts_of(md, (1, 2, 3), 1)
    toks = [start[:, 0]]
    for _ in range(n + 2):
        nxt, lg = B.decode(toks[-1])
        toks.append(nxt)
    for _ in range(2):
        B.reset()
        got, ms = B.generate(start, n)
        assert np.array_equal(got, np.stack(toks[1:n + 2], 1)) and ms > 0
        nxt, last = B.decode(toks[n + 1])
        assert np.array_equal(last, lg) and np.array_equal(nxt, toks[n + 2])


def test_beside_other_batches(made):
    """A batch in fp32 and the model's own run in between: each keeps its results."""
    md, *_ = model_case("mixtral_small")
    M = made(hiplm.LmModel(md, 64))
    ids = prompts_of(md, (1, 2), 24)
    alone = {}
    for kv4 in (False, True):
        B = hiplm.LmBatch(M, 2, kv4=kv4)
        alone[kv4] = [B.decode(ids[:, i])[1] for i in range(24)]
        B.free()
    B4, B32 = made(hiplm.LmBatch(M, 2, kv4=True)), made(hiplm.LmBatch(M, 2))
    for i in range(24):
        assert np.array_equal(B4.decode(ids[:, i])[1], alone[True][i])
        if i == 10:
            M.generate(ids[0], 4)
        assert np.array_equal(B32.decode(ids[:, i])[1], alone[False][i])
    assert not np.array_equal(alone[True][20], alone[False][20])


def test_a_full_cache_is_refused(made):
    md, *_ = model_case("olmoe_small")
    M = made(hiplm.LmModel(md, 40))
    B = made(hiplm.LmBatch(M, 2, kv4=True))
    ids = prompts_of(md, (1, 2), 40)
    with pytest.raises(hiplm.HipMoeError, match="do not fit"):
        B.generate(ids, 1)
    first = B.decode(ids[:, 0])[1]
    with pytest.raises(hiplm.HipMoeError, match="do not fit"):
        B.generate(ids[:, 1:31], 10)
    for i in range(1, 40):
        lg = B.decode(ids[:, i])[1]
    for _ in range(2):
        with pytest.raises(hiplm.HipMoeError, match="do not fit"):
            B.decode(ids[:, 0])
    B.reset()
    assert np.array_equal(B.decode(ids[:, 0])[1], first)
    for i in range(1, 40):
        again = B.decode(ids[:, i])[1]
    assert np.array_equal(again, lg)


def test_replayed_steps_over_long_caches(made):
    """Captured steps across the row counts at which the attention cuts a cache into
    pieces, against decoded ones, and two batches' graphs in turn."""
    md = small("olmoe", 1)
    M = made(hiplm.LmModel(md, 1100))
    A, B = made(hiplm.LmBatch(M, 2, kv4=True)), made(hiplm.LmBatch(M, 2, kv4=True))
    ids = prompts_of(md, (1, 2), 1000)
    steps = A.generate(ids, 0)[0][:, 0]
    want = [steps]
    for _ in range(60):
        want.append(A.decode(want[-1])[0])
    want = np.stack(want, 1)
    A.reset()
    for _ in range(2):
        for X in (A, B):
            assert np.array_equal(X.generate(ids, 30)[0], want[:, :31])
        for X in (B, A):
            assert np.array_equal(X.generate(want[:, 30:31], 29)[0], want[:, 31:])
            X.reset()
