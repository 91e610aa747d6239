"""Sequences that share a page, behind a step of a model that ended in an error."""
import numpy as np
import pytest

from tests.test_gpu_paged_model import cache_for, logits, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "int8"])
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 0, 2)])
def test_rows_of_forks_behind_a_step_that_failed(hip, dtype, order):
    """All layers were written when the sampler raises.  What comes next is to the bit what it is where the step never was: the same batch, lengths and keys."""
    cfg, llm = model()
    m, rng = llm.model, np.random.default_rng(8)
    prompt, more = rng.integers(0, cfg["vocab_size"], 45).astype(np.int32), rng.integers(0, cfg["vocab_size"], (3, 7)).astype(np.int32)

    class Broken:
        def check(self, rows):
            pass

        def pick(self, *args):
            raise RuntimeError("no numbers")

    after = []
    for fails in (False, True):
        cache = cache_for(llm, 24, dtype=dtype)
        whole = cache.add()
        m.forward_paged(cache, [whole], [prompt])
        seqs = [whole, cache.fork(whole, 34), cache.fork(whole, 40)]
        if fails:
            held = {s: list(p) for s, p in cache.pages.items()}, dict(cache.lengths), dict(cache.shared)
            with pytest.raises(RuntimeError, match="no numbers"):
                m.forward_paged(cache, [seqs[i] for i in order], [more[i] for i in order], sampler=Broken())
            assert held == (cache.pages, cache.lengths, cache.shared)
        m.forward_paged(cache, seqs, more[:, :1] + 1)
        after.append(logits(m, 3))
    assert np.array_equal(*after)


def test_a_fork_behind_a_window(hip):
    """What its next row would see was given away: refused, with the sequences as they were; a fork that has it goes on as the sequence does."""
    cfg, llm = model()
    m, rng = llm.model, np.random.default_rng(9)
    cache = cache_for(llm, 16)
    a = cache.add()
    m.forward_paged(cache, [a], [rng.integers(0, cfg["vocab_size"], 160).astype(np.int32)], 40)
    cache.slide(a, 40)
    back, beside = cache.fork(a, 80), cache.fork(a, 160)
    before = {s: list(p) for s, p in cache.pages.items()}, dict(cache.lengths), list(cache.free)
    for seqs, window in (([back], 40), ([a, back], 40), ([a], 60), ([a], 0)):
        with pytest.raises(ValueError, match="given away"):
            m.forward_paged(cache, seqs, [np.array([1])] * len(seqs), window)
        assert before == (cache.pages, cache.lengths, cache.free)
    m.forward_paged(cache, [a], [np.array([1])], 40)
    want = logits(m, 1)
    m.forward_paged(cache, [beside], [np.array([1])], 40)
    assert np.array_equal(want, logits(m, 1))
