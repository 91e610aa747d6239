"""Transformer.forward_paged that ends in an error: the sequences are as they were, and go on as if the call had not been made."""
import numpy as np
import pytest

from denograd_amd import llama
from tests.test_gpu_paged_model import cache_for, logits, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["activations", "layer", "head", "tokens"])
@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_a_step_that_fails_leaves_lengths_and_pages(hip, monkeypatch, where, dtype):
    cfg, llm = model()
    m = llm.model
    rng = np.random.default_rng(4)
    first, more = [rng.integers(0, cfg["vocab_size"], n).astype(np.int32) for n in (20, 33)], [rng.integers(0, cfg["vocab_size"], n).astype(np.int32) for n in (50, 1)]

    def run(fail):
        cache = cache_for(llm, dtype=dtype)
        seqs = [cache.add() for _ in first]
        m.forward_paged(cache, seqs, first)
        if fail:
            before = ({s: list(p) for s, p in cache.pages.items()}, dict(cache.lengths), list(cache.free))

            def broken(*args, **kwargs):
                raise MemoryError("no room")

            with monkeypatch.context() as patch:
                if where == "activations":
                    patch.setattr(llama, "_PagedScratch", broken)
                    patch.setattr(m, "_paged", None)
                elif where == "layer":                          # the first layer has written its rows by then
                    patch.setattr(m.layers[-1].feed_forward, "call_rows", broken)
                elif where == "head":
                    patch.setattr(m, "output", None)
                else:
                    patch.setattr(m, "tok_embeddings", None)
                with pytest.raises((MemoryError, AttributeError)):
                    m.forward_paged(cache, seqs[::-1], more)
            assert before == (cache.pages, cache.lengths, cache.free)
        m.forward_paged(cache, seqs, more)
        return logits(m, 2), {s: list(p) for s, p in cache.pages.items()}

    (want, pages), (got, same) = run(False), run(True)
    assert np.array_equal(want, got) and pages == same
