"""A batch that cannot begin leaves its cache's sequences as they were; without a GPU."""
import numpy as np
import pytest

from denograd_amd.paged import PagedBatch, PagedCache, PageTable


class Plan:
    """Stands for the array that the device reads."""

    numel = 1 << 20

    def __init__(self):
        self.lazydata, self.full = self, False

    def view(self, *args):
        return self

    ensure_allocated = lambda self: self

    def copyin(self, plan):
        if self.full:
            raise MemoryError("no room")


def cache_of(n_pages=12):
    cache = PagedCache.__new__(PagedCache)                # the bookkeeping alone
    PageTable.__init__(cache, n_pages, 16)
    cache._plan, cache._batches = Plan(), 0
    return cache


def state(cache):
    return {s: list(p) for s, p in cache.pages.items()}, dict(cache.lengths), list(cache.free)


def test_a_batch_whose_arrays_cannot_be_written_leaves_lengths_and_pages():
    cache = cache_of()
    a, b, c = (cache.add() for _ in range(3))
    cache.begin([a, b], [40, 16])
    first = cache.begin([b, a], [1, 3])
    cache.slide(a, 20, 0)
    before = state(cache)
    cache._plan.full = True
    for seqs, counts in (([a], [1]), ([a, c, b], [30, 17, 15]), ([c], [64])):
        with pytest.raises(MemoryError, match="no room"):
            cache.begin(seqs, counts)
        assert state(cache) == before
    with pytest.raises(RuntimeError, match="another batch"):   # what its arrays hold now is not known
        first._args(0)
    cache._plan.full = False
    again = cache.begin([a, c, b], [30, 17, 15])
    assert isinstance(again, PagedBatch) and again.rows == 62 and cache.lengths == {a: 73, b: 32, c: 17}


def test_begins_and_cancels_at_random_keep_every_page_once():
    rng = np.random.default_rng(0)
    cache = cache_of(40)
    seqs = [cache.add() for _ in range(5)]
    for _ in range(300):
        some = [int(s) for s in rng.choice(seqs, 3, replace=False)]
        before = state(cache)
        try:
            batch = cache.begin(some, rng.integers(0, 40, 3) + [1, 0, 0])
        except MemoryError:
            assert state(cache) == before
            cache.drop(seqs.pop(0))
            seqs.append(cache.add())
            continue
        if rng.integers(2):
            batch._cancel()
            assert state(cache) == before
            batch._cancel()
            assert state(cache) == before
        assert sorted(cache.free + [p for v in cache.pages.values() for p in v if p >= 0]) == list(range(40))
