"""Tokens of rows by temperature, min-p, top-k, top-p and given numbers, against float64."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.ffi import check
from denograd_amd.sampling import RowSampler
from denograd_amd.tensor import Tensor
from tests.sample_ref import sample

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def run(lib, x, n=None, stride=None, probs=True, **rows):
    """x: [rows, stride] host logits; rows: the five arrays, None for NULL."""
    R, n = x.shape[0], x.shape[1] if n is None else n
    t = Tensor(x)
    dev = {k: Tensor(np.ascontiguousarray(v, np.int32 if k == "top_k" else np.float32)) for k, v in rows.items() if v is not None}
    p = lambda k: dev[k].ptr if k in dev else None
    tok, pr = Tensor.full((R + 1,), 7.0, "float32"), Tensor.full((R + 1,), 7.0, "float32")
    ws = Tensor.full((lib.jsgrad_hip_sample_rows_workspace_bytes(R, n) // 4,), float("nan"), "float32")     # whatever it holds
    check(lib.jsgrad_hip_sample_rows(t.ptr, R, n, x.shape[1] if stride is None else stride, ffi.F16 if x.dtype == np.float16 else ffi.F32, p("temperature"), p("top_k"), p("top_p"), p("min_p"),
                                     p("uniforms"), tok.ptr, pr.ptr if probs else None, ws.ptr))
    got, share = tok.numpy().view(np.int32), pr.numpy()
    assert tok.numpy()[R] == 7 and share[R] == 7             # nothing behind the rows
    return got[:R], share[:R]


def agree(lib, x, n=None, **rows):
    """Tokens are equal.  Shares: the weights are whole 2^-42 of the largest, so each is off by half of that and a total by as much for each entry; then one rounding to float."""
    got, share = run(lib, x, n, **rows)
    n = x.shape[1] if n is None else n
    for r in range(x.shape[0]):
        one = {("u" if k == "uniforms" else k): v[r] for k, v in rows.items() if v is not None}
        want, p = sample(x[r, :n], **one)
        assert got[r] == want, (r, one, got[r], want)
        assert abs(share[r] - p) <= U32 * p + (n + 1) * 2.0 ** -43, (r, one, share[r], p)


def logits(rng, R, n, dtype, spread=2.0):
    x = spread * rng.standard_normal((R, n))
    x += (rng.random((R, n)) < 0.002) * 9 * rng.random((R, n))
    return x.astype(dtype)


def mixed(rng, R):
    return dict(temperature=rng.choice([0, 1e-3, 0.3, 0.7, 1, 1.7, 100], R), top_k=rng.choice([0, 1, 2, 20, 50, 512, 1000, 1025, 1 << 30], R), top_p=rng.choice([0, 1e-30, 0.1, 0.5, 0.9, 0.999, 1, 2], R),
                min_p=rng.choice([0, 0, 1e-4, 0.02, 0.5, 1, 3], R), uniforms=np.where(rng.random(R) < 0.1, rng.choice([0, 1 - 2.0 ** -24], R), rng.random(R)))


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 600, 1024, 1025, 4095, 4096, 4097, 32000, 50257, 128256, 131071, 1 << 20])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rows_with_settings_of_their_own(hip, n, dtype):
    rng = np.random.default_rng(n)
    R = 40 if n <= 50257 else 12
    agree(hip, logits(rng, R, n, dtype), **mixed(rng, R))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [20011, 128256, 1 << 19])
def test_borders_by_number_and_by_mass_in_one_row(hip, n, dtype):
    """Both on one step, on steps far apart, with all that is in front of the first in a list or too much for one, and entries that are alike at them."""
    rng = np.random.default_rng(n)
    ks, ps = [257, 1000, 5000, 8190, 9000, 19000], [1e-3, 0.3, 0.9, 0.999, 1 - 1e-6]
    R = len(ks) * len(ps)
    x = logits(rng, R, n, dtype)
    x[::3] = (x[::3] * 8).round() / 8
    agree(hip, x, temperature=rng.choice([0.5, 1, 1.5], R), top_k=np.repeat(ks, len(ps)), top_p=np.tile(ps, len(ks)), min_p=rng.choice([0, 0, 1e-5], R), uniforms=rng.random(R))


@pytest.mark.parametrize("alone", ["temperature", "top_k", "top_p", "min_p", None])
def test_settings_alone(hip, alone):
    rng = np.random.default_rng(1)
    rows = mixed(rng, 64)
    agree(hip, logits(rng, 64, 5003, np.float16), **{k: (v if k in (alone, "uniforms") else None) for k, v in rows.items()})


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n,stride", [(777, 780), (50257, 50264), (1000, 4321)])
def test_rows_inside_wider_ones(hip, n, stride, dtype):
    """What lies between rows is not read: it would win."""
    rng = np.random.default_rng(n)
    x = logits(rng, 20, stride, dtype)
    x[:, n:] = np.inf
    agree(hip, x, n, **mixed(rng, 20))


@pytest.mark.parametrize("n", [5, 4096, 128256])
def test_ties_borders_and_flat_rows(hip, n):
    """Equal logits: counts and shares of them end exactly, at the lowest indexes.  Few distinct values: borders inside a tie."""
    rng = np.random.default_rng(n)
    R = 24
    flat = np.zeros((R, n), np.float32)
    flat[1::2] = -0.0
    flat[2, ::2] = -0.0                                       # zeros of either sign are equal
    k = rng.integers(1, n + 1, R)
    p = rng.choice([0.25, 0.5, 0.75, 0.3, 1.0], R)
    u = rng.integers(0, 8, R) / 8
    agree(hip, flat, temperature=np.full(R, 0.7), top_k=k, top_p=p, uniforms=u)
    agree(hip, flat.astype(np.float16), temperature=np.full(R, 0.7), top_k=np.where(np.arange(R) % 3, 0, k), top_p=p, uniforms=u)
    few = rng.integers(0, 3, (R, n)).astype(np.float16)
    agree(hip, few, temperature=rng.choice([0.5, 1, 2], R), top_k=np.where(np.arange(R) % 2, 0, k), top_p=p, min_p=rng.choice([0, np.exp(-1), 0.1], R), uniforms=rng.random(R))
    narrow = (100 + rng.integers(0, 3000, (R, n)) * 2.0 ** -17).astype(np.float32)       # all of them within one part in forty of the same weight
    agree(hip, narrow, temperature=rng.choice([0.5, 1, 2], R), top_k=np.where(np.arange(R) % 2, 0, k), top_p=p, uniforms=rng.random(R))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [3, 700, 128256])
def test_masked_entries_infinities_and_nan(hip, n, dtype):
    rng = np.random.default_rng(n + 1)
    x = logits(rng, 16, n, dtype)
    low = np.finfo(dtype).min
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, n // 2] = low
    x[3] = low                                                # the lowest value is a value: all alike
    x[4, n - 1] = np.inf
    x[5, [0, n - 1]] = np.inf
    x[6, ::2] = np.nan
    x[6, 1] = 0.5
    x[7] = np.where(rng.random(n) < 0.9, low, x[7])
    x[8] = np.where(rng.random(n) < 0.9, -np.inf, x[8])
    x[8, 1] = 1.0
    x[9] = np.where(np.arange(n) == n - 1, 1.0, -np.inf)
    x[10] = np.nan
    x[10, 0] = -np.inf
    x[11] = np.finfo(dtype).tiny * rng.integers(-3, 4, n)
    rows = mixed(rng, 16)
    agree(hip, x, **rows)
    rows["temperature"][:] = 1.0
    agree(hip, x, **rows)
    rows["temperature"][:] = 0.0
    agree(hip, x, **rows)


def test_settings_that_are_no_settings(hip):
    """Not numbers, infinities, negative ones: a temperature below 1e-6 or not a number is greedy; numbers outside 0 to 1 count as the nearest inside."""
    rng = np.random.default_rng(2)
    x = logits(rng, 8, 999, np.float32)
    nan = np.nan
    base = dict(temperature=np.ones(8), top_k=np.zeros(8), top_p=np.ones(8), min_p=np.zeros(8), uniforms=rng.random(8))
    want = run(hip, x, **base)[0]
    for change in (dict(top_k=np.full(8, -5)), dict(top_p=np.full(8, nan)), dict(min_p=np.full(8, nan)), dict(min_p=np.full(8, -1))):
        assert np.array_equal(run(hip, x, **{**base, **change})[0], want)
    top = x.argmax(-1)
    for change in (dict(temperature=np.full(8, nan)), dict(temperature=np.full(8, -1)), dict(temperature=np.full(8, 9e-7)), dict(top_p=np.full(8, -1)), dict(top_p=np.zeros(8)),
                   dict(top_k=np.ones(8)), dict(min_p=np.full(8, 5))):
        assert np.array_equal(run(hip, x, **{**base, **change})[0], top)
    first, last = run(hip, x, **{**base, "uniforms": np.full(8, -3)})[0], run(hip, x, **{**base, "uniforms": np.full(8, 2)})[0]
    assert np.all(first == 0) and np.all(last == 998)
    assert np.array_equal(run(hip, x, **{**base, "uniforms": np.full(8, nan)})[0], first)
    hot = run(hip, x, **{**base, "temperature": np.full(8, np.inf)})[0]
    assert np.array_equal(hot, np.floor(base["uniforms"].astype(np.float32).astype(np.float64) * 999).astype(int))


def test_shares_are_drawn_as_often_as_they_say(hip):
    """Every entry of a row, over numbers spread evenly: as often as its share, to one."""
    rng = np.random.default_rng(3)
    x = np.repeat(logits(rng, 1, 40, np.float32), 4096, 0)
    rows = dict(temperature=np.full(4096, 0.9), top_k=np.full(4096, 30), top_p=np.full(4096, 0.98), uniforms=(np.arange(4096) + 0.5) / 4096)
    got, share = run(hip, x, **rows)
    for t in np.unique(got):
        assert abs((got == t).sum() - 4096 * share[got == t][0]) <= 1
    assert np.all(np.diff(got) >= 0)


def test_the_same_twice_and_beside_other_rows(hip):
    rng = np.random.default_rng(4)
    x, rows = logits(rng, 70, 40000, np.float16), mixed(rng, 70)
    a, pa = run(hip, x, **rows)
    b, pb = run(hip, x, **rows)
    assert np.array_equal(a, b) and np.array_equal(pa, pb)
    for i in (0, 33, 69):
        c, pc = run(hip, x[i:i + 1], **{k: v[i:i + 1] for k, v in rows.items()})
        assert c[0] == a[i] and pc[0] == pa[i]
    assert np.array_equal(run(hip, x, probs=False, **rows)[0], a)


def test_captured_and_replayed_with_other_settings(hip):
    """Two graphs with one workspace, eager calls between their replays, other numbers and settings in the arrays."""
    rng = np.random.default_rng(5)
    x = [Tensor(logits(rng, 6, 20000, np.float16)) for _ in range(2)]
    host = [t.numpy() for t in x]
    rows = mixed(rng, 6)
    dev = {k: Tensor(np.ascontiguousarray(v, np.int32 if k == "top_k" else np.float32)) for k, v in rows.items()}
    tok, pr = [Tensor.zeros((6,), "int32") for _ in range(2)], Tensor.zeros((6,), "float32")
    ws = Tensor.empty((hip.jsgrad_hip_sample_rows_workspace_bytes(6, 20000),), "uint8")
    call = lambda i: check(hip.jsgrad_hip_sample_rows(x[i].ptr, 6, 20000, 20000, ffi.F16, *(dev[k].ptr for k in ("temperature", "top_k", "top_p", "min_p", "uniforms")), tok[i].ptr, pr.ptr, ws.ptr))
    graphs = []
    for i in range(2):
        call(i)
        g = C.c_void_p()
        check(hip.jsgrad_hip_graph_begin())
        call(i)
        check(hip.jsgrad_hip_graph_end(C.byref(g)))
        graphs.append(g)
    for step in range(4):
        rows = mixed(rng, 6)
        for k, v in rows.items():
            dev[k].lazydata.copyin(np.ascontiguousarray(v, np.int32 if k == "top_k" else np.float32))
        check(hip.jsgrad_hip_graph_launch(graphs[step % 2]))
        check(hip.jsgrad_hip_graph_launch(graphs[1 - step % 2]))
        for i in range(2):
            want = [sample(host[i][r], *(rows[k][r] for k in ("temperature", "top_k", "top_p", "min_p", "uniforms")))[0] for r in range(6)]
            assert np.array_equal(tok[i].numpy(), want)
        call(step % 2)
        assert np.array_equal(run(hip, host[1 - step % 2], **rows)[0], tok[1 - step % 2].numpy())
    for g in graphs:
        check(hip.jsgrad_hip_graph_destroy(g))


def test_row_sampler(hip):
    rng = np.random.default_rng(6)
    x = logits(rng, 5, 3001, np.float16)
    t = Tensor(x)
    s = RowSampler([0.0, 0.7, 1.0, 1.3, 0.5], 40, 0.9, [0, 0, 0.1, 0, 0], seed=11)
    numbers = np.random.default_rng(11)
    for _ in range(3):
        u = numbers.random(5, np.float32)
        got = s.pick(t).numpy()
        want = [sample(x[r], [0.0, 0.7, 1.0, 1.3, 0.5][r], 40, 0.9, [0, 0, 0.1, 0, 0][r], u[r]) for r in range(5)]
        assert np.array_equal(got, [w[0] for w in want]) and np.allclose(s.probs.numpy(), [w[1] for w in want], rtol=1e-6)
    one = RowSampler(0.8, seed=1)
    for rows in (3, 5, 2, 5):                                 # one sampler, batches of any size
        assert one.pick(t, rows=rows).shape == (rows,)
    for bad in (lambda: s.pick(t, rows=4), lambda: one.pick(t, rows=6), lambda: one.pick(Tensor(x[0])), lambda: one.pick(t, Tensor.zeros((4,), "int32")), lambda: one.pick(Tensor.zeros((2, 8), "int32"))):
        with pytest.raises(ValueError):
            bad()


def test_answers_drawn_by_a_model(hip):
    """Each token is what the step's logits, the settings and the sampler's numbers give; several answers to a prompt, with and without a window."""
    from tests.test_gpu_paged_model import cache_for, logits as model_logits, model
    cfg, llm = model()
    m = llm.model
    prompts = [np.arange(n, dtype=np.int32) * 7 % cfg["vocab_size"] for n in (30, 1, 65)]
    got = llm.generate_paged(prompts, 6, page_size=16, samples=3, temperature=1.2, top_k=50, top_p=0.95, min_p=0.01, seed=4)
    assert got.shape == (9, 6) and len(np.unique(got[:3], axis=0)) > 1
    # the same, step by step, with a sequence of its own for each answer
    numbers, cache = np.random.default_rng(4), cache_for(llm, 64)
    seqs = [cache.add() for _ in range(9)]
    for s, p in zip(seqs, [p for p in prompts for _ in range(3)]):
        if p.size > 1:
            m.forward_paged(cache, [s], [p[:-1]])
    toks = [p[-1:] for p in prompts for _ in range(3)]
    sampler, step = RowSampler(1.2, 50, 0.95, 0.01, seed=4), []
    for i in range(6):
        toks = m.forward_paged(cache, seqs, toks, sampler=sampler).numpy()
        x, u = m._paged.logits.numpy()[:9], numbers.random(9, np.float32)
        assert np.array_equal(toks, [sample(x[r], 1.2, 50, 0.95, 0.01, u[r])[0] for r in range(9)])
        step.append(toks)
    # prompts that came in one batch there come one by one here: their rows may differ by roundings, and a token with them
    assert (np.array(step).T == got).mean() > 0.5
    greedy = llm.generate_paged(prompts, 6, page_size=16)
    assert np.array_equal(llm.generate_paged(prompts, 6, page_size=16, temperature=0.8, top_k=1), greedy)
    assert llm.generate_paged(prompts, 40, page_size=16, window=20, sinks=2, samples=2, temperature=1.0).shape == (6, 40)
    for bad in (dict(samples=0), dict(temperature=0.5, top_p=1.5), dict(temperature=0.5, top_k=-1), dict(temperature=float("inf"))):
        with pytest.raises(ValueError):
            llm.generate_paged(prompts, 2, **bad)
    with pytest.raises(ValueError, match="rows"):
        m.forward_paged(cache, seqs[:2], [[1], [2]], sampler=RowSampler([1.0, 1.0, 1.0]))
    assert cache.lengths[seqs[0]] == 35 and model_logits(m, 1).shape == (1, cfg["vocab_size"])
