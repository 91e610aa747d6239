"""The activations of steps over a paged cache grow and never shrink: prompts and steps of many sequences in turn take the same buffers."""
import numpy as np
import pytest

from tests.test_gpu_paged_model import cache_for, logits, model

pytestmark = pytest.mark.gpu


def test_prompts_and_steps_in_turn_keep_their_buffers(hip):
    cfg, llm = model()
    m = llm.model
    rng = np.random.default_rng(7)
    prompt, step = [rng.integers(0, cfg["vocab_size"], 60).astype(np.int32)], [rng.integers(0, cfg["vocab_size"], 1).astype(np.int32) for _ in range(16)]

    def run():
        cache = cache_for(llm)
        seqs = [cache.add() for _ in range(17)]
        m.forward_paged(cache, seqs[:1], prompt)
        a = logits(m, 1)
        m.forward_paged(cache, seqs[1:], step)
        return a, logits(m, 16)

    first = run()
    kept, ptrs = m._paged, [t.ptr for t in (m._paged.h, m._paged.g, m._paged.logits, m._paged.tokens)]
    assert kept.bsz >= 16 and kept.n >= 60
    for _ in range(2):
        assert all(np.array_equal(a, b) for a, b in zip(first, run()))
        assert m._paged is kept and ptrs == [t.ptr for t in (m._paged.h, m._paged.g, m._paged.logits, m._paged.tokens)]
