"""Tokens of rows with min-p on what top-k and top-p leave, against float64."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.ffi import check
from denograd_amd.sampling import RowSampler
from denograd_amd.tensor import Tensor

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
NAMES = ("temperature", "top_k", "top_p", "min_p", "uniforms")


def last(x, temperature, top_k, top_p, min_p, u):
    """(token, share) of one row: the first top_k by value, of these those with less than top_p of their mass before them, of these the weights of min_p and more."""
    x = np.asarray(x).astype(np.float64)
    x[np.isnan(x)] = -np.inf
    T, p, m, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    best = int(np.argmax(x))
    if np.isneginf(x[best]):
        return -1, 0.0
    if T < float(np.float32(1e-6)):
        return best, 1.0
    rank = np.argsort(-x, kind="stable")
    if top_k > 0:
        rank = rank[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[rank] == x[best], 1.0, np.exp((x[rank] - x[best]) / T))
    if p < 1.0:
        upto = np.cumsum(w)
        n = 1 + int(np.count_nonzero(upto[:-1] < p * upto[-1]))
        rank, w = rank[:n], w[:n]
    held = w >= min(m, 1.0)
    at = np.argsort(rank[held])
    rank, w = rank[held][at], w[held][at]
    run = np.cumsum(w)
    i = int(np.argmax(run > u * run[-1]))
    return int(rank[i]), w[i] / run[-1]


def run(lib, x, order=ffi.MIN_P_LAST, **rows):
    R, n = x.shape
    t, dev = Tensor(x), {k: Tensor(np.ascontiguousarray(rows[k], np.int32 if k == "top_k" else np.float32)) for k in NAMES}
    tok, pr = Tensor.zeros((R,), "int32"), Tensor.zeros((R,), "float32")
    ws = Tensor.full((lib.jsgrad_hip_sample_rows_workspace_bytes(R, n) // 4,), float("nan"), "float32")
    at = [dev[k].ptr for k in NAMES]
    check(lib.jsgrad_hip_sample_rows_ordered(t.ptr, R, n, n, ffi.F16 if x.dtype == np.float16 else ffi.F32, *at[:4], order, at[4], tok.ptr, pr.ptr, ws.ptr))
    return tok.numpy(), pr.numpy()


def agree(lib, x, **rows):
    """Tokens are equal.  Shares: the weights are whole 2^-42 of the largest, so each is off by half of that and a total by as much for each entry; then one rounding to float."""
    got, share = run(lib, x, **rows)
    for r in range(x.shape[0]):
        want, p = last(x[r], *(rows[k][r] for k in NAMES))
        assert got[r] == want, (r, [rows[k][r] for k in NAMES], got[r], want)
        assert abs(share[r] - p) <= U32 * p + (x.shape[1] + 1) * 2.0 ** -43, (r, [rows[k][r] for k in NAMES], share[r], p)
    return got, share


def logits(rng, R, n, dtype):
    return (2 * rng.standard_normal((R, n)) + (rng.random((R, n)) < 0.002) * 9 * rng.random((R, n))).astype(dtype)


def settings(rng, R):
    return dict(temperature=rng.choice([0, 0.3, 0.7, 1, 1.7, 100], R), top_k=rng.choice([0, 1, 20, 256, 257, 1000, 5000, 1 << 30], R), top_p=rng.choice([0, 1e-3, 0.5, 0.9, 0.95, 0.999, 1], R),
                min_p=rng.choice([1e-7, 1e-4, 0.02, 0.1, 0.5, 1, 3], R), uniforms=np.where(rng.random(R) < 0.1, 1 - 2.0 ** -24, rng.random(R)))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [1, 2, 65, 1025, 4097, 32000, 128256])
def test_every_place_of_the_borders(hip, n, dtype):
    """The cut by min-p above, on and below the steps on which those by number and by mass are."""
    rng = np.random.default_rng(n)
    R = 48 if n <= 32000 else 24
    agree(hip, logits(rng, R, n, dtype), **settings(rng, R))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_the_place_makes_the_difference(hip, dtype):
    """Mass that min-p drops counts for top-p: other totals, and with them other tokens, than with min-p in front; the same where top-p is 1."""
    rng = np.random.default_rng(3)
    R, x = 64, logits(rng, 64, 128256, dtype)
    rows = dict(temperature=np.full(R, 1.0), top_k=rng.choice([0, 50, 1000], R), top_p=np.full(R, 0.9), min_p=np.full(R, 0.02), uniforms=rng.random(R))
    got, share = agree(hip, x, **rows)
    first = run(hip, x, ffi.MIN_P_FIRST, **rows)
    assert np.any(first[1] != share)
    rows["top_p"][:] = 1.0
    for a, b in zip(run(hip, x, ffi.MIN_P_FIRST, **rows), agree(hip, x, **rows)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("n", [700, 128256])
def test_flat_rows_ties_and_masked_entries(hip, n):
    """Few distinct values, so that steps hold more entries than a list; minus infinity, not numbers, and one infinity."""
    rng = np.random.default_rng(n)
    R = 24
    u = rng.random(R)
    few = rng.integers(0, 3, (R, n)).astype(np.float16)
    few[0], few[1, 0] = 0, np.inf
    few[2, ::2], few[3, 1::2], few[4] = np.nan, -np.inf, -np.inf
    few[4, n // 2] = -60000
    rows = dict(temperature=rng.choice([0.5, 1, 2], R), top_k=np.where(np.arange(R) % 2, 0, rng.integers(1, n + 1, R)), top_p=rng.choice([0.25, 0.5, 0.9, 1.0], R),
                min_p=rng.choice([np.exp(-1), np.exp(-2) * 1.01, 0.1, 0.9], R), uniforms=u)
    agree(hip, few, **rows)
    narrow = (100 + rng.integers(0, 3000, (R, n)) * 2.0 ** -17).astype(np.float32)
    rows["min_p"] = rng.choice([0.995, 0.99, 0.985], R)
    agree(hip, narrow, **rows)


def test_captured_and_replayed(hip):
    """One graph with other settings in the arrays at each replay, and eager calls between."""
    rng = np.random.default_rng(5)
    host = logits(rng, 6, 20000, np.float16)
    x, dev = Tensor(host), {k: Tensor(np.zeros(6, np.int32 if k == "top_k" else np.float32)) for k in NAMES}
    tok, pr = Tensor.zeros((6,), "int32"), Tensor.zeros((6,), "float32")
    ws = Tensor.empty((hip.jsgrad_hip_sample_rows_workspace_bytes(6, 20000),), "uint8")
    at = [dev[k].ptr for k in NAMES]
    graph = C.c_void_p()
    check(hip.jsgrad_hip_graph_begin())
    check(hip.jsgrad_hip_sample_rows_ordered(x.ptr, 6, 20000, 20000, ffi.F16, *at[:4], ffi.MIN_P_LAST, at[4], tok.ptr, pr.ptr, ws.ptr))
    check(hip.jsgrad_hip_graph_end(C.byref(graph)))
    for _ in range(4):
        rows = settings(rng, 6)
        for k, v in rows.items():
            dev[k].lazydata.copyin(np.ascontiguousarray(v, np.int32 if k == "top_k" else np.float32))
        check(hip.jsgrad_hip_graph_launch(graph))
        got, share = tok.numpy(), pr.numpy()
        eager = agree(hip, host, **rows)
        assert np.array_equal(got, eager[0]) and np.array_equal(share, eager[1])
    check(hip.jsgrad_hip_graph_destroy(graph))


def test_sampler_and_model(hip):
    """RowSampler and generate_paged pass the place on."""
    from tests.test_gpu_paged_model import cache_for, model
    rng = np.random.default_rng(6)
    x = logits(rng, 5, 3001, np.float16)
    s, numbers = RowSampler(1.0, 0, 0.9, 0.03, seed=11, min_p_last=True), np.random.default_rng(11)
    for _ in range(2):
        u = numbers.random(5, np.float32)
        want = [last(x[r], 1.0, 0, 0.9, 0.03, u[r]) for r in range(5)]
        assert np.array_equal(s.pick(Tensor(x)).numpy(), [w[0] for w in want]) and np.allclose(s.probs.numpy(), [w[1] for w in want], rtol=1e-6)
    cfg, llm = model()
    m, cache = llm.model, cache_for(llm, 16)
    settings_ = dict(temperature=1.5, top_k=300, top_p=0.8, min_p=0.05, seed=2, min_p_last=True)
    got = llm.generate_paged([np.arange(9)], 5, page_size=16, **settings_)
    seq, toks, sampler, numbers = cache.add(), np.arange(9, dtype=np.int32), RowSampler(**settings_), np.random.default_rng(2)
    for i in range(5):
        toks = m.forward_paged(cache, [seq], [toks], sampler=sampler).numpy()
        assert toks[0] == last(m._paged.logits.numpy()[0], 1.5, 300, 0.8, 0.05, numbers.random(1, np.float32)[0])[0] == got[0, i]
