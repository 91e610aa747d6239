"""Forks and windows that reach pages which were given away: refused before anything is computed; without a GPU."""
import numpy as np
import pytest

from tests.test_paged_begin import cache_of


def seen(cache, s, count, window, sinks):
    """Whether a batch of so many rows may attend."""
    batch = cache.begin([s], [count])
    try:
        batch._check_seen(window, sinks)
        return True
    except ValueError as e:
        assert f"sequence {s} " in str(e)
        return False
    finally:
        batch._cancel()


def test_a_fork_behind_the_window_of_its_sequence():
    cache = cache_of(40)
    a = cache.add()
    cache.begin([a], [512])
    cache.slide(a, 64)
    back = cache.fork(a, 256)
    assert cache.pages[back] == [-1] * 16
    assert not seen(cache, back, 1, 64, 0) and not seen(cache, back, 1, 0, 0) and not seen(cache, back, 20, 2, 0)
    assert seen(cache, back, 1, 1, 0)                        # its own position alone
    assert seen(cache, a, 1, 64, 0) and seen(cache, a, 1, 30, 0) and seen(cache, cache.fork(a), 3, 64, 0)
    assert not seen(cache, a, 1, 90, 0) and not seen(cache, a, 1, 64, 1) and not seen(cache, a, 1, 0, 0)


def test_what_is_refused_is_what_is_not_there():
    """Against the positions themselves, for every window and number of sinks of a slide and of the rows behind it."""
    rng = np.random.default_rng(0)
    for _ in range(3000):
        cache = cache_of(20)
        s = cache.add()
        length = int(rng.integers(1, 160))
        cache.begin([s], [length])
        for _ in range(int(rng.integers(0, 3))):
            cache.slide(s, int(rng.integers(1, 180)), int(rng.integers(0, 60)))
        if rng.integers(0, 2):
            try:
                s = cache.fork(s, int(rng.integers(0, length // 16 + 1)) * 16)
            except ValueError:
                continue
        length, count, window, sinks = cache.lengths[s], int(rng.integers(1, 40)), int(rng.integers(0, 180)), int(rng.integers(0, 60))
        if len(cache.free) * 16 < count + 16:
            continue
        want = all(cache.pages[s][j // 16] >= 0 for j in range(length) for p in (length,) if not window or j > p - window or j < sinks)
        assert seen(cache, s, count, window, sinks) == want


def test_sequences_without_new_rows_are_not_looked_at():
    cache = cache_of(40)
    a, b = cache.add(), cache.add()
    cache.begin([a, b], [200, 5])
    cache.slide(a, 16)
    batch = cache.begin([a, b], [0, 1])
    batch._check_seen(0, 0)
    assert batch._gaps == []
