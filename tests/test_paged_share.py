"""Sequences that share pages: forks, pages of one's own in front of a write, packing; the bookkeeping, without a GPU."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.paged import PagedCache, PageTable
from tests.test_paged_begin import cache_of, state


def check_books(t: PageTable) -> None:
    """Every page is free or held, and `shared` says by how many where that is more than one."""
    held: dict[int, int] = {}
    for pages in t.pages.values():
        for p in pages:
            if p >= 0:
                held[p] = held.get(p, 0) + 1
    assert sorted(t.free + list(held)) == list(range(t.n_pages))
    assert t.shared == {p: n for p, n in held.items() if n > 1}
    assert all(len(t.pages[s]) == -(-t.lengths[s] // t.page_size) for s in t.pages)


def test_a_fork_shares_pages_until_one_writes():
    t = PageTable(8, 16)
    a = t.add()
    assert t.grow([a], [40]) == []
    b, c = t.fork(a), t.fork(a, 32)
    assert t.pages[b] == t.pages[a] and t.pages[c] == t.pages[a][:2] and (t.lengths[b], t.lengths[c]) == (40, 32) and len(t.free) == 5
    check_books(t)
    assert t.grow([c], [1]) == []                            # a page of its own begins
    last = t.pages[a][2]
    assert t.grow([b, a], [1, 1]) == [(last, t.pages[b][2], 8)] and t.pages[a][2] == last     # the last holder writes into the page itself
    check_books(t)
    for s in (a, c, b):
        t.drop(s)
        check_books(t)
    assert len(t.free) == 8


def test_forks_inside_a_page_and_of_nothing():
    t = PageTable(4, 16)
    a = t.add()
    t.grow([a], [20])
    empty, inside, edge = t.fork(a, 0), t.fork(a, 5), t.fork(a, 16)
    assert t.pages[empty] == [] and t.pages[inside] == t.pages[a][:1] == t.pages[edge]
    first = t.pages[a][0]
    assert t.grow([inside, edge, a, empty], [1, 0, 1, 0]) == [(first, t.pages[inside][0], 5)]
    check_books(t)
    for at in (-1, 22):
        with pytest.raises(ValueError, match="fork"):
            t.fork(a, at)
    with pytest.raises(KeyError):
        t.fork(99)


def test_too_few_pages_for_pages_of_ones_own_change_nothing():
    t = PageTable(4, 16)
    a = t.add()
    t.grow([a], [20])
    forks = [t.fork(a) for _ in range(3)]
    before = {s: list(p) for s, p in t.pages.items()}, dict(t.lengths), list(t.free), dict(t.shared)
    with pytest.raises(MemoryError, match="3 pages"):
        t.grow([a, *forks], [1] * 4)
    assert before == (t.pages, t.lengths, t.free, t.shared)
    assert len(t.grow([a, forks[1]], [1] * 2)) == 2 and t.free == []
    check_books(t)


def test_a_batch_that_fails_gives_shared_pages_back():
    cache = cache_of()
    copied = []
    cache._copy = copied.append
    a = cache.add()
    cache.begin([a], [40])
    b = cache.fork(a)
    before, shared = state(cache), dict(cache.shared)
    cache._plan.full = True
    with pytest.raises(MemoryError, match="no room"):
        cache.begin([a, b], [30, 1])
    assert state(cache) == before and cache.shared == shared and len(copied) == 1
    cache._plan.full = False
    batch = cache.begin([a, b], [30, 1])
    check_books(cache)
    batch._cancel()
    assert state(cache) == before and cache.shared == shared
    # the other holder went while the batch was running: the page is the sequence's alone again
    batch = cache.begin([b], [1])
    cache.drop(a)
    batch._cancel()
    assert cache.lengths[b] == 40
    check_books(cache)

    def broken(moves):
        raise ffi.HipError("no copy")

    c = cache.fork(b)
    before, shared = state(cache), dict(cache.shared)
    cache._copy = broken
    with pytest.raises(ffi.HipError):
        cache.begin([c], [1])
    assert state(cache) == before and cache.shared == shared


def test_random_forks_drops_windows_and_packing():
    """The contents of pages, walked as a copy of every move and a write of every new position would leave them."""
    rng = np.random.default_rng(0)
    for _ in range(60):
        t = PageTable(int(rng.integers(6, 40)), 16)
        held = np.full((t.n_pages, 16), -1)
        want: dict[int, list[int]] = {}
        gone: dict[int, int] = {}                             # positions that were given away
        for step in range(120):
            seqs = list(t.pages)
            what = rng.integers(0, 7)
            if what == 0 or not seqs:
                s = t.add()
                want[s], gone[s] = [], 0
            elif what == 1 and len(seqs) > 1:
                s = int(rng.choice(seqs))
                t.drop(s)
                del want[s], gone[s]
            elif what == 2:
                s = int(rng.choice(seqs))
                at = int(rng.integers(0, t.lengths[s] + 1))
                if at % 16 and t.pages[s][at // 16] < 0:
                    with pytest.raises(ValueError, match="given away"):
                        t.fork(s, at)
                    continue
                n = t.fork(s, at)
                want[n], gone[n] = want[s][:at], gone[s]
            elif what == 3 and rng.integers(0, 3) == 0:
                for a, b, n in t._pack():
                    held[b, :n] = held[a, :n]
                assert sorted(t.free) == list(range(t.n_pages - len(t.free), t.n_pages))
            elif what == 4:
                s = int(rng.choice(seqs))
                w = int(rng.integers(1, 60))
                t.slide(s, w)
                gone[s] = max(gone[s], t.lengths[s] - w + 1)
            else:
                some = [int(s) for s in rng.permutation(seqs)[:rng.integers(1, 4)]]
                counts = rng.integers(0, 30, len(some)).tolist()
                try:
                    moves = t.grow(some, counts)
                except MemoryError:
                    check_books(t)
                    continue
                for a, b, n in moves:
                    held[b, :n] = held[a, :n]
                for s, c in zip(some, counts):
                    for i in range(c):
                        p = len(want[s])
                        want[s].append(int(rng.integers(1 << 30)))
                        held[t.pages[s][p // 16], p % 16] = want[s][-1]
            check_books(t)
            for s, values in want.items():
                for p in range(max(0, gone[s]), len(values)):
                    assert held[t.pages[s][p // 16], p % 16] == values[p]


@pytest.mark.parametrize("change,match", [
    (dict(host_pools=None), "null"), (dict(moves=None), "null"), (dict(n_pools=0), "0 pools"), (dict(n_pages=0), "pages"), (dict(n_moves=0), "moves"), (dict(moves=4098), "aligned"),
    (dict(data=None), "pool 1: null"), (dict(data=4104), "aligned"), (dict(segments=0), "pool 1"), (dict(positions=-1), "pool 1"), (dict(bytes=6), "multiple of 4"), (dict(bytes=0), "multiple of 4"),
    (dict(segments=1 << 20, positions=1 << 10), "1 GiB"), (dict(positions=1 << 30), "1 GiB"), ({}, "init"),
])
def test_copies_that_are_refused(change, match):
    lib = ffi.load()
    pools = (ffi.Pool * 2)(ffi.Pool(4096, 2, 16, 128), ffi.Pool(4096, 2, 16, 128))
    args = dict(host_pools=pools, n_pools=2, n_pages=4, moves=4096, n_moves=1)
    for k, v in change.items():
        if k in args:
            args[k] = v
        else:
            setattr(pools[1], k, v)
    if not change and __import__("os").path.exists("/dev/kfd"):
        pytest.skip("would run")
    assert lib.jsgrad_hip_paged_copy(*args.values()) != 0
    assert match in lib.jsgrad_hip_last_error().decode()


@pytest.mark.parametrize("change,match", [
    (dict(k_weight=None), "weights"), (dict(q_weight=None), "weights"), (dict(q=None, q_out=None), "weights"), (dict(q_weight=4100), "aligned"), (dict(k_weight=4104), "aligned"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(k=None), "null"), (dict(q_out=None), "together"), (dict(rope_rows=31), "rope"),
])
def test_normed_writes_that_are_refused(change, match):
    lib = ffi.load()
    desc = ffi.PagesDesc(ffi.W_F16, 4, 16, 2, 64, 2, 4096, 4096, None, None, 4096)
    args = dict(pages=desc, row_starts=4096, lengths=4096, n_seqs=1, rows=1, q=4096, k=4096, v=4096, q_weight=4096, k_weight=4096, eps=1e-5, rope=4096, rope_rows=32, q_out=4096, n_heads=4)
    args.update(change)
    assert lib.jsgrad_hip_paged_write_norm(*args.values()) != 0
    assert match in lib.jsgrad_hip_last_error().decode()


def test_pool_layout():
    assert C.sizeof(ffi.Pool) == 24
