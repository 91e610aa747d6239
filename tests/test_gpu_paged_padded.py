"""Attention of batches with many sequences that have no new rows, as a captured graph's batch is filled up: groups of 64 of them in front of, between and behind the others, and no more rows
than sequences."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd.ffi import check
from denograd_amd.tensor import Tensor
from tests.paged_ref import Case, attention
from tests.test_gpu_paged import compare, run_attention

pytestmark = pytest.mark.gpu


def batch(kind, hd, some, n_seqs, extra):
    """some: {sequence: (new rows, length)}."""
    news, lens = [0] * n_seqs, [0, 5, 40] * (n_seqs // 3) + [7] * (n_seqs % 3)
    for b, (n, l) in some.items():
        news[b], lens[b] = n, l
    rng = np.random.default_rng(n_seqs + hd)
    c = Case(rng, kind, hd, 2, 16, news, lens, extra_rows=extra)
    c.table = np.pad(c.table, ((0, 0), (0, 300)), constant_values=-1)      # room for more work than the batch has
    c.width = c.table.shape[1]
    c.device()
    return c, rng.standard_normal((c.rows, 8, hd)).astype(np.float16)


@pytest.mark.parametrize("kind,hd", [("float16", 64), ("float16", 128), ("int8", 64), ("int8", 128)])
@pytest.mark.parametrize("some,n_seqs,extra", [
    ({0: (150, 900)}, 200, 0), ({100: (150, 900)}, 200, 50), ({199: (150, 900)}, 200, 0), ({129: (1, 2000)}, 130, 0), ({63: (1, 300), 64: (60, 700), 200: (2, 50)}, 320, 7),
    ({5: (200, 200), 70: (1, 1500), 300: (8, 400), 511: (40, 41)}, 512, 0), ({64: (9, 3000)}, 65, 0), ({0: (1, 1), 319: (90, 700)}, 320, 229),
])
def test_sequences_without_new_rows(hip, kind, hd, some, n_seqs, extra):
    c, q = batch(kind, hd, some, n_seqs, extra)
    for window, sinks in ((0, 0), (70, 3)):
        ref, tol = attention(c, q, 8, window, sinks)
        compare(run_attention(hip, c, q, 8, window, sinks, times=2), ref, tol, int(c.starts[-1]))


def test_row_starts_that_fall_behind_sequences_without_rows(hip):
    """In the fifth group of 64, and the only sequence with rows in front of them: nothing is written, and the workspace serves the next call."""
    c, q = batch("float16", 64, {3: (40, 600)}, 300, 0)
    c.starts[290], c.starts[291] = 39, 20
    c.device()
    ws, tq, out = Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(8, 2, 64),), "uint8"), Tensor(q), Tensor.full(q.shape, 7.0, "float16")
    check(hip.jsgrad_hip_attn_paged(*c.batch, tq.ptr, out.ptr, 8, 0, 0, ws.ptr))
    assert np.all(out.numpy() == 7)
    c, q = batch("float16", 64, {3: (40, 600)}, 300, 0)
    ref, tol = attention(c, q, 8)
    compare(run_attention(hip, c, q, 8, 0, 0, ws), ref, tol, 40)


@pytest.mark.parametrize("kind,hd", [("float16", 64), ("int8", 64), ("float16", 128), ("int8", 128)])
def test_a_captured_launch_serves_prompts_and_single_rows(hip, kind, hd):
    """One graph for 130 sequences and 130 rows, replayed with a prompt, with a row each, with both and with nothing, another batch on the same workspace between the replays; each against an
    eager call."""
    n_seqs, rows, H = 130, 130, 8
    rng = np.random.default_rng(hd)
    lens = rng.integers(1, 200, n_seqs)
    lens[[3, 70]] = 1500, 700
    c = Case(rng, kind, hd, 2, 16, [1] * n_seqs, lens.tolist()).device()
    other, oq = batch(kind, hd, {1: (90, 800)}, 70, 0)
    q = rng.standard_normal((rows, H, hd)).astype(np.float16)
    ws = [Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(H, 2, hd),), "uint8") for _ in range(2)]
    tq, out, ref = Tensor(q), Tensor.full(q.shape, 7.0, "float16"), Tensor.full(q.shape, 7.0, "float16")
    graph = C.c_void_p()
    check(hip.jsgrad_hip_graph_begin())
    try:
        check(hip.jsgrad_hip_attn_paged(*c.batch, tq.ptr, out.ptr, H, 0, 0, ws[0].ptr))
    finally:
        check(hip.jsgrad_hip_graph_end(C.byref(graph)))
    for news in ({3: 130}, {b: 1 for b in range(n_seqs)}, {3: 60, 70: 9, 71: 1, 129: 1}, {}, {70: 128}, {b: 1 for b in range(0, n_seqs, 2)}):
        counts = [min(news.get(b, 0), int(lens[b])) for b in range(n_seqs)]
        c.t["starts"].lazydata.copyin(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        for t in (out, ref):
            t.lazydata.copyin(np.full(q.shape, 7, np.float16))
        check(hip.jsgrad_hip_graph_launch(graph))
        got = out.numpy()
        run_attention(hip, other, oq, H, 0, 0, ws[0])
        check(hip.jsgrad_hip_attn_paged(*c.batch, tq.ptr, ref.ptr, H, 0, 0, ws[1].ptr))
        assert np.array_equal(got, ref.numpy()) and np.all(got[sum(counts):] == 7) and not np.any(got[:sum(counts)] == 7)
        if sum(counts) in (130, 128):
            c.starts, c.news = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), counts
            want, tol = attention(c, q, H)
            compare(got, want, tol, sum(counts))
    check(hip.jsgrad_hip_graph_destroy(graph))
