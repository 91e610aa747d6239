"""Pages copied to pages, forks of running sequences, and a pool packed between steps."""
import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.ffi import check
from denograd_amd.paged import PagedCache
from denograd_amd.tensor import Tensor
from tests.test_gpu_paged_model import cache_for, logits, model

pytestmark = pytest.mark.gpu


def copied(pools, moves):
    out = [p.copy() for p in pools]
    for a, b, n in moves:
        for src, dst in zip(pools, out):
            if 0 <= a < len(src) and 0 <= b < len(src) and a != b and n > 0:
                dst[b, :, :n] = src[a, :, :n]
    return out


@pytest.mark.parametrize("n_pages,shapes,moves", [
    (5, [(2, 16, 128)], [(0, 3, 16)]), (5, [(2, 16, 128), (2, 16, 4), (1, 1, 516)], [(4, 0, 7), (1, 2, 1), (3, 3, 16)]),
    (9, [(8, 64, 256), (8, 64, 4)] * 3, [(0, 8, 64), (1, 7, 37), (2, 6, 63), (3, 5, 0), (-1, 4, 9), (4, 9, 9), (4, 1 << 30, 3)]),
    (6, [(3, 256, 128), (3, 256, 4), (1, 1, 12), (5, 7, 20), (2, 16, 4)], [(0, 5, 255), (1, 4, 1 << 30), (2, 3, -5)]),
    (300, [(1, 16, 16)] * 129, [(i, 299 - i, 1 + i % 16) for i in range(150)]),
    (3, [(1, 1, 3 << 20), (4, 200000, 4)], [(2, 0, 199999)]),
])
def test_copied_pages(hip, n_pages, shapes, moves):
    """Bytes are bytes: whole pages, the begun part of each segment, moves that are none."""
    rng = np.random.default_rng(n_pages)
    host = [rng.integers(-128, 128, (n_pages, *s)).astype(np.int8) for s in shapes]
    dev = [Tensor(h) for h in host]
    pools = (ffi.Pool * len(dev))(*[ffi.Pool(t.ptr, *s) for t, s in zip(dev, shapes)])
    m = Tensor(np.array(moves, np.int32))
    check(hip.jsgrad_hip_paged_copy(pools, len(dev), n_pages, m.ptr, len(moves)))
    for t, want in zip(dev, copied(host, moves)):
        assert np.array_equal(t.numpy(), want)


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_answers_that_share_a_prompt(hip, dtype):
    """A fork goes on as a sequence of its own with the same tokens does, whatever the others write: the same bits, as the rows of a batch are summed alike when batch and lengths are."""
    cfg, llm = model()
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, cfg["vocab_size"], 41).astype(np.int32)
    more = rng.integers(0, cfg["vocab_size"], (3, 9)).astype(np.int32)
    own, shared = cache_for(llm, 64, dtype=dtype), cache_for(llm, 16, dtype=dtype)
    so = [own.add() for _ in more]
    for s in so:
        llm.model.forward_paged(own, [s], [prompt])
    first = shared.add()
    llm.model.forward_paged(shared, [first], [prompt])
    ss = [first, shared.fork(first), shared.fork(first)]
    assert 16 - len(shared.free) == 3
    for i in range(more.shape[1]):
        llm.model.forward_paged(own, so, more[:, i:i + 1])
        want = logits(llm.model, 3)
        llm.model.forward_paged(shared, ss, more[:, i:i + 1])
        assert np.array_equal(want, logits(llm.model, 3))
        if i == 0:
            assert 16 - len(shared.free) == 5                # two whole pages together, a begun one each
        if i == 4:
            shared.drop(shared.fork(ss[1]))
    # a fork back inside the prompt: what it writes does not reach the others
    back = shared.fork(ss[0], 20)
    llm.model.forward_paged(shared, [back], [more[1, :5]])
    tok = more[:, 0]
    llm.model.forward_paged(own, so, tok[:, None])
    want = logits(llm.model, 3)
    llm.model.forward_paged(shared, ss, tok[:, None])
    assert np.array_equal(want, logits(llm.model, 3))


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_a_packed_pool_goes_on_as_before(hip, dtype):
    cfg, llm = model()
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, cfg["vocab_size"], n).astype(np.int32) for n in (30, 70, 5, 50)]
    a, b = cache_for(llm, 24, dtype=dtype), cache_for(llm, 24, dtype=dtype)
    for cache in (a, b):
        seqs = [cache.add() for _ in prompts]
        llm.model.forward_paged(cache, seqs, prompts)
        cache.drop(seqs[0])
        cache.drop(seqs[2])
        cache.fork(seqs[1], 40)
    live = [seqs[1], seqs[3], seqs[3] + 1]
    old = b.begin([live[0]], [1])
    b.drop(b.fork(live[1]))
    b.lengths[live[0]] -= 1                                  # the batch's one row was never written
    n = b.compact()
    assert n == 9 and sorted(b.free) == list(range(9, 24)) and max(p for v in b.pages.values() for p in v) == 8
    with pytest.raises(RuntimeError, match="another batch"):
        old.read(0)
    assert b.compact() == 9                                  # nothing left to move
    for _ in range(20):
        toks = rng.integers(0, cfg["vocab_size"], (3, 1)).astype(np.int32)
        llm.model.forward_paged(a, live, toks)
        want = logits(llm.model, 3)
        llm.model.forward_paged(b, live, toks)
        assert np.array_equal(want, logits(llm.model, 3))


def test_a_captured_copy_follows_its_moves(hip):
    """Replayed with other moves in the array, and the program's own copies between the replays."""
    import ctypes as C
    rng = np.random.default_rng(7)
    host = rng.integers(-128, 128, (6, 2, 16, 64)).astype(np.int8)
    t, m = Tensor(host), Tensor(np.array([[0, 5, 16], [1, 4, 3]], np.int32))
    pools = (ffi.Pool * 1)(ffi.Pool(t.ptr, 2, 16, 64))
    graph = C.c_void_p()
    check(hip.jsgrad_hip_graph_begin())
    check(hip.jsgrad_hip_paged_copy(pools, 1, 6, m.ptr, 2))
    check(hip.jsgrad_hip_graph_end(C.byref(graph)))
    for moves in ([[0, 5, 16], [1, 4, 3]], [[5, 1, 2], [2, 0, 16]], [[3, 3, 16], [9, 0, 1]], [[4, 2, 15], [0, 3, 1]]):
        m.lazydata.copyin(np.array(moves, np.int32).reshape(-1))
        check(hip.jsgrad_hip_graph_launch(graph))
        host = copied([host], moves)[0]
        assert np.array_equal(t.numpy(), host)
        back = [[moves[0][1], 1, 4]] if moves[0][1] != 1 else [[0, 2, 4]]
        k = Tensor(np.array(back, np.int32))
        check(hip.jsgrad_hip_paged_copy(pools, 1, 6, k.ptr, 1))
        host = copied([host], back)[0]
        assert np.array_equal(t.numpy(), host)
    check(hip.jsgrad_hip_graph_destroy(graph))


def test_a_cache_too_full_for_a_page_of_ones_own(hip):
    cfg, llm = model()
    cache = cache_for(llm, 2)
    s = cache.add()
    llm.model.forward_paged(cache, [s], [np.arange(20, dtype=np.int32)])
    f = cache.fork(s)
    with pytest.raises(MemoryError):
        llm.model.forward_paged(cache, [f], [np.array([1])])
    assert cache.lengths[f] == 20 and cache.pages[f] == cache.pages[s]
    cache.drop(s)
    llm.model.forward_paged(cache, [f], [np.array([1])])
    assert isinstance(cache, PagedCache) and cache.free == []
