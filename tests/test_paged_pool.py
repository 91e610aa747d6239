"""How many pages sequences need that grow behind a window (PageTable.pages_for): as many as the bookkeeping takes, and not one more."""
import numpy as np
import pytest

from denograd_amd.paged import PagedCache, PageTable


def run(n_pages, page, prompts, n_new, window, sinks):
    t = PageTable(n_pages, page)
    seqs = [t.add() for _ in prompts]
    most = 0
    for i in range(n_new):
        t.grow(seqs, prompts if i == 0 else [1] * len(seqs))
        most = max(most, n_pages - len(t.free))
        if window:
            for s in seqs:
                t.slide(s, window, sinks)
    return most


def test_pages_for_is_what_the_bookkeeping_takes():
    rng = np.random.default_rng(0)
    for _ in range(400):
        page, n_new = int(rng.choice([16, 32, 64])), int(rng.choice([1, 2, 40, 200]))
        prompts = rng.integers(1, 200, rng.integers(1, 5)).tolist()
        window, sinks = int(rng.choice([0, 1, 5, 16, 50, 1000])), int(rng.choice([0, 1, 16, 40]))
        n = PageTable.pages_for(prompts, n_new, page, window, sinks)
        assert run(n, page, prompts, n_new, window, sinks) == n
        if n > 1:
            with pytest.raises(MemoryError):
                run(n - 1, page, prompts, n_new, window, sinks)
    assert PageTable.pages_for([10], 1000, 16, 32, 4) == 4         # 63 pages without the window
    assert PageTable.pages_for([10], 1000, 16) == 64


@pytest.mark.gpu
def test_generating_behind_a_window_takes_the_pages_that_are_seen(hip, monkeypatch):
    from denograd_amd import paged
    from tests.test_gpu_paged_model import cache_for, model
    cfg, llm = model()
    prompts = [np.arange(n, dtype=np.int32) % cfg["vocab_size"] for n in (40, 3)]
    keep, want, toks = cache_for(llm, 64), [], prompts
    seqs = [keep.add() for _ in prompts]
    for _ in range(100):
        toks = llm.model.forward_paged(keep, seqs, toks, 20, 2).numpy()
        want.append(toks)
    made = []

    class Counted(PagedCache):
        def __init__(self, *args, **kwargs):
            super().__init__(*args, **kwargs)
            made.append(self)

    monkeypatch.setattr(paged, "PagedCache", Counted)
    got = llm.generate_paged(prompts, 100, page_size=16, window=20, sinks=2)
    assert np.array_equal(got, np.array(want).T)
    assert made[0].n_pages <= 7 and 64 - len(keep.free) == 9 + 7        # 139 and 102 positions
    for more in (dict(window=-1), dict(sinks=-1), dict(page_size=0)):
        with pytest.raises(ValueError):
            llm.generate_paged(prompts, 2, **more)
