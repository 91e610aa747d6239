"""What sequences that share pages hold behind a batch that was cancelled between its layers; the bookkeeping, without a GPU."""
import numpy as np
import pytest

from tests.test_paged_begin import cache_of, state
from tests.test_paged_share import check_books


class Contents:
    """What the pages of a cache hold, position by position, as copies and writes leave it."""

    def __init__(self, n_pages=12):
        self.cache, self.at = cache_of(n_pages), np.full((n_pages, 16), -1)
        self.cache._copy = self.copy

    def copy(self, moves):
        for a, b, n in moves:
            self.at[b, :n] = self.at[a, :n]

    def write(self, seqs, counts, value):
        for s, c in zip(seqs, counts):
            for p in range(self.cache.lengths[s] - c, self.cache.lengths[s]):
                self.at[self.cache.pages[s][p // 16], p % 16] = value = value + 1

    def of(self, s):
        return [int(self.at[self.cache.pages[s][p // 16], p % 16]) for p in range(self.cache.lengths[s])]


@pytest.mark.parametrize("lengths", [(40, 34), (34, 40), (40, 40), (47, 33, 40), (33, 47, 47, 40)])
@pytest.mark.parametrize("counts", [1, 5, 20])
def test_forks_of_any_lengths_keep_their_rows_when_a_batch_is_cancelled(lengths, counts):
    """Holders of one begun page that all write: behind the batch as without it, in every order; and with it, each has its own rows."""
    for order in (list(range(len(lengths))), list(range(len(lengths)))[::-1], sorted(range(len(lengths)), key=lambda i: lengths[i])):
        c = Contents()
        whole = c.cache.add()
        c.cache.begin([whole], [47])
        c.write([whole], [47], 0)
        seqs = [c.cache.fork(whole, n) for n in lengths]
        c.cache.drop(whole)
        before = [c.of(s) for s in seqs], state(c.cache), dict(c.cache.shared)
        batch = c.cache.begin([seqs[i] for i in order], [counts] * len(seqs))
        check_books(c.cache)
        c.write([seqs[i] for i in order], [counts] * len(seqs), 100)
        assert [c.of(s)[:n] for s, n in zip(seqs, lengths)] == before[0]
        batch._cancel()
        check_books(c.cache)
        assert ([c.of(s) for s in seqs], dict(c.cache.pages), dict(c.cache.lengths), c.cache.shared) == (before[0], before[1][0], before[1][1], before[2])
        c.cache.begin([seqs[i] for i in order], [counts] * len(seqs))
        c.write([seqs[i] for i in order], [counts] * len(seqs), 1000)
        rows = [c.of(s) for s in seqs]
        assert [r[:n] for r, n in zip(rows, lengths)] == before[0] and len({v for r, n in zip(rows, lengths) for v in r[n:]}) == counts * len(seqs)


def test_random_batches_that_are_cancelled_or_not():
    rng = np.random.default_rng(1)
    for _ in range(40):
        c = Contents(int(rng.integers(6, 30)))
        want: dict[int, list[int]] = {c.cache.add(): []}
        for step in range(80):
            what = rng.integers(0, 6)
            seqs = list(want)
            if what == 0 and len(seqs) < 8:
                s = int(rng.choice(seqs))
                at = int(rng.integers(0, len(want[s]) + 1))
                want[c.cache.fork(s, at)] = want[s][:at]
            elif what == 1 and len(seqs) > 3:
                s = int(rng.choice(seqs))
                c.cache.drop(s)
                del want[s]
            else:
                some = [int(s) for s in rng.permutation(seqs)[:rng.integers(1, 6)]]
                counts = rng.integers(0, 20, len(some)).tolist()
                if not any(counts):
                    continue
                try:
                    batch = c.cache.begin(some, counts)
                except MemoryError:
                    continue
                c.write(some, counts, step * 1000)
                if rng.integers(0, 2):
                    gone = int(rng.choice(seqs)) if len(seqs) > 3 and rng.integers(0, 3) == 0 else None
                    if gone is not None:                      # an answer that ended while the batch was running
                        c.cache.drop(gone)
                        del want[gone]
                    batch._cancel()
                else:
                    for s in some:
                        want[s] = want[s] + c.of(s)[len(want[s]):]
            check_books(c.cache)
            assert {s: c.of(s) for s in want} == want
