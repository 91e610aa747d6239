"""Attention over pages that each row chooses: the pages' bounds and the choice, which are exact, and the attention against float64."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd.ffi import check
from denograd_amd.paged import PagedCache
from denograd_amd.tensor import Tensor
from tests import select_ref as ref
from tests.paged_ref import Case, attention as plain_attention
from tests.test_gpu_paged_model import cache_for, logits, model

pytestmark = pytest.mark.gpu

BATCHES = [  # kind, hd, H, KV, page, new rows, lengths, first, recent, top
    ("float16", 64, 4, 2, 16, [1], [1], 0, 1, 1), ("int8", 128, 8, 2, 16, [1], [200], 1, 2, 5), ("float16", 128, 32, 8, 64, [1, 0, 1, 3], [700, 9, 64, 65], 1, 1, 4),
    ("int8", 64, 32, 8, 32, [1, 1, 1], [1000, 31, 512], 0, 2, 9), ("float16", 64, 6, 2, 16, [33, 1], [90, 400], 2, 3, 7), ("int8", 128, 3, 1, 256, [5], [3000], 1, 1, 3),
    ("float16", 128, 7, 7, 128, [2] * 9, [2, 3, 127, 128, 129, 600, 900, 4, 5], 0, 1, 2), ("int8", 64, 64, 2, 16, [2, 1], [170, 300], 1, 1, 8), ("float16", 64, 40, 1, 32, [3], [500], 1, 2, 6),
    ("float16", 128, 4, 2, 16, [1] * 70, list(range(1, 1400, 20)), 1, 2, 10), ("int8", 128, 4, 1, 16, [1], [16000], 3, 5, 300),
]


def arrays(c, rng):
    """Bounds with something in them: what is not written stays."""
    codes = rng.integers(-100, 100, (c.n_pages, c.KV, 2, c.hd)).astype(np.int8)
    return codes, (2.0 ** rng.integers(-6, 3, (c.n_pages, c.KV))).astype(np.float32)


def everything(c, codes, scales):
    """Bounds of all pages of the case's sequences, as the steps before would have left them."""
    news, c.news = c.news, c.lens
    out = ref.bounds(c, codes, scales)
    c.news = news
    return out


def run_bounds(hip, c, codes, scales):
    tb, ts = Tensor(codes), Tensor(scales)
    check(hip.jsgrad_hip_paged_bounds(*c.batch, tb.ptr, ts.ptr))
    return tb.numpy(), ts.numpy()


def run_choose(hip, c, q, H, codes, scales, first, recent, top):
    tq, tb, ts, out = Tensor(q), Tensor(codes), Tensor(scales), Tensor(np.full((c.rows, c.KV, top), 77, np.int32))
    check(hip.jsgrad_hip_paged_select(*c.batch, tq.ptr, H, tb.ptr, ts.ptr, first, recent, top, out.ptr))
    return out.numpy()


_WS = {}


def run_attend(hip, c, q, H, selected, fill=7.0):
    key = (H, c.KV, c.hd)
    if key not in _WS:
        _WS[key] = Tensor.zeros((hip.jsgrad_hip_attn_selected_workspace_bytes(*key),), "uint8")
    tq, tsel, out = Tensor(q), Tensor(np.ascontiguousarray(selected, np.int32)), Tensor.full(q.shape, fill, "float16")
    check(hip.jsgrad_hip_attn_selected(*c.batch, tq.ptr, out.ptr, H, tsel.ptr, selected.shape[2], _WS[key].ptr))
    return out.numpy()


@pytest.mark.parametrize("kind,hd,H,KV,page,news,lens,first,recent,top", BATCHES)
def test_bounds_choice_and_attention(hip, kind, hd, H, KV, page, news, lens, first, recent, top):
    rng = np.random.default_rng(hd + H + page + top)
    c = Case(rng, kind, hd, KV, page, news, lens, extra_rows=2).device()
    codes, scales = everything(c, *arrays(c, rng))
    stale = codes.copy()
    for b, (n, l) in enumerate(zip(news, lens)):
        for i in {p // page for p in range(l - n, l)}:
            stale[c.table[b, i]] = 55
    want = ref.bounds(c, stale, scales)
    got = run_bounds(hip, c, stale, scales)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], codes)                      # whatever way the rows came
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    sel = run_choose(hip, c, q, H, *got, first, recent, top)
    assert np.array_equal(sel, ref.choose(c, q, H, *want, first, recent, top, np.full(sel.shape, 77, np.int32)))
    out = run_attend(hip, c, q, H, sel)
    n = int(c.starts[-1])
    exact, tol = ref.attention(c, q, H, sel)
    assert np.all(np.abs(out[:n].astype(np.float64) - exact[:n]) <= tol[:n]) and np.all(out[n:] == 7)


def test_scores_never_fall_short_of_a_key(hip):
    """What a page's score bounds: the largest product of a rounded query with a key of the page."""
    rng = np.random.default_rng(3)
    c = Case(rng, "float16", 64, 2, 16, [1], [800]).device()
    codes, scales = everything(c, *arrays(c, rng))
    q = rng.standard_normal((1, 4, 64)).astype(np.float16)
    k = c.values("k")
    for g in range(2):
        x = q[0, 2 * g:2 * g + 2].astype(np.float64)
        x = np.rint(x / ref.step(np.abs(x).max())) * ref.step(np.abs(x).max())
        for at in c.table[0]:
            bound = np.maximum(x[:, None] * codes[at, g, 0], x[:, None] * codes[at, g, 1]).sum(-1).max() * scales[at, g]
            assert (k[at, g] @ x.T).max() <= bound


@pytest.mark.parametrize("kind", ["float16", "int8"])
def test_keys_of_any_size_and_not_finite_ones(hip, kind):
    """Zeros, the least and largest halves, infinities and NaN on some pages; equal pages go to the lower one."""
    rng = np.random.default_rng(4)
    k = rng.standard_normal((30, 2, 16, 64)).astype(np.float16)
    k[1:6] = 0
    k[6] = np.float16(6e-8)
    k[7] = np.float16(65504)
    k[8, 0, 3, 9], k[9, 1, 0, 0], k[10, 0, 15, 63] = np.nan, np.inf, -np.inf
    k[11:16] = k[11]
    k[16] *= np.float16(1e-4)
    k[17] = np.float16(127)
    k[18] = np.float16(127.0625)
    k[19] = np.float16(-128)
    c = Case(rng, kind, 64, 2, 16, [400], [400], spare=5, k=k)
    if kind == "int8":
        c.sk[20:22] *= np.float32(1e-40)                      # products below the normal floats
        c.sk[22] = np.float32(1e36)
        c.sk[23] = np.float32(3e38)                           # and beyond the floats
    c.device()
    codes, scales = arrays(c, rng)
    want = ref.bounds(c, codes, scales)
    got = run_bounds(hip, c, codes, scales)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    q = rng.standard_normal((400, 4, 64)).astype(np.float16)
    q[0], q[1] = 0, np.float16(6e-8)
    q[2, 0, 5], q[3, 3, 1], q[399, 1, 2] = np.nan, np.inf, -np.inf
    for first, recent, top in ((0, 1, 4), (2, 2, 12), (0, 1, 30)):
        sel = run_choose(hip, c, q, 4, *got, first, recent, top)
        assert np.array_equal(sel, ref.choose(c, q, 4, *want, first, recent, top, np.full(sel.shape, 77, np.int32)))


def test_holes_short_tables_and_rows_outside(hip):
    """Entries that are no page of the pool, positions behind the table or below zero, sequences without rows."""
    rng = np.random.default_rng(5)
    c = Case(rng, "float16", 64, 2, 16, [1, 3, 0, 5, 2], [300, 100, 50, 3, 40], extra_rows=3)
    c.table[0, [2, 5, 6, 18]] = [-1, 1 << 30, c.n_pages, -7]
    c.table[1, :] = -1
    c.device()
    codes, scales = everything(c, *arrays(c, rng))
    want = ref.bounds(c, codes, scales)
    got = run_bounds(hip, c, codes, scales)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    q = rng.standard_normal((c.rows, 4, 64)).astype(np.float16)
    for top in (3, 17, 1024):
        sel = run_choose(hip, c, q, 4, codes, scales, 1, 2, top)
        assert np.array_equal(sel, ref.choose(c, q, 4, codes, scales, 1, 2, top, np.full(sel.shape, 77, np.int32)))
        out = run_attend(hip, c, q, 4, sel)
        n = int(c.starts[-1])
        exact, tol = ref.attention(c, q, 4, sel)
        assert np.all(np.abs(out[:n].astype(np.float64) - exact[:n]) <= tol[:n]) and np.all(out[n:] == 7)
    c.table = c.table[:, :10].copy()                          # the first sequence's last nine columns are not in the table
    c.device()
    sel = run_choose(hip, c, q, 4, codes, scales, 1, 2, 6)
    assert np.array_equal(sel, ref.choose(c, q, 4, codes, scales, 1, 2, 6, np.full(sel.shape, 77, np.int32)))


def test_lists_of_the_callers_own(hip):
    """Any order, holes between, no columns, later pages than the row's, a page twice."""
    rng = np.random.default_rng(6)
    for kind in ("float16", "int8"):
        c = Case(rng, kind, 128, 2, 32, [1, 2], [500, 77]).device()
        q = rng.standard_normal((3, 4, 128)).astype(np.float16)
        sel = np.full((3, 2, 9), -1, np.int32)
        sel[0, 0], sel[0, 1] = [7, -1, 3, 15, -1, 0, 1 << 30, -5, 16], [-1, -1, -1, -1, -1, -1, -1, -1, 4]
        sel[1, 0, :4], sel[1, 1] = [2, 1, 0, 3], -1          # column 3 is not there; nothing at all
        sel[2, 0, 4], sel[2, 1, :3] = 2, [1, 1, 0]
        out = run_attend(hip, c, q, 4, sel)
        exact, tol = ref.attention(c, q, 4, sel)
        assert np.all(np.abs(out.astype(np.float64) - exact) <= tol) and np.all(out[1, 2:] == 0)
        assert np.array_equal(out, run_attend(hip, c, q, 4, sel))


def test_values_that_are_not_finite_where_no_row_looks(hip):
    """On pages that are not chosen and behind the row's position they reach nothing; a key or value that is seen does."""
    rng = np.random.default_rng(7)
    c = Case(rng, "float16", 64, 1, 16, [1], [150])
    for i in (3, 5):
        c.k[c.table[0, i]], c.v[c.table[0, i]] = np.nan, np.inf
    c.k[c.table[0, 9], :, 6:], c.v[c.table[0, 9], :, 6:] = np.inf, np.nan
    c.device()
    q = rng.standard_normal((1, 4, 64)).astype(np.float16)
    sel = np.array([[[0, 1, 4, 8, 9]]], np.int32)
    out = run_attend(hip, c, q, 4, sel)
    exact, tol = ref.attention(c, q, 4, sel)
    assert np.all(np.abs(out.astype(np.float64) - exact) <= tol)
    c.v[c.table[0, 4], 0, 2, 7] = np.inf
    c.device()
    out = run_attend(hip, c, q, 4, sel)
    assert np.all(np.isposinf(out[0, :, 7])) and np.isfinite(np.delete(out, 7, -1)).all()


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
def test_all_pages_chosen_is_attention_over_everything(hip, kind, hd):
    rng = np.random.default_rng(8)
    c = Case(rng, kind, hd, 2, 16, [1, 40, 0, 1], [500, 40, 20, 3]).device()
    codes, scales = everything(c, *arrays(c, rng))
    q = rng.standard_normal((c.rows, 8, hd)).astype(np.float16)
    sel = run_choose(hip, c, q, 8, codes, scales, 0, 1, 40)
    out = run_attend(hip, c, q, 8, sel)
    exact, tol = plain_attention(c, q, 8)
    assert np.all(np.abs(out.astype(np.float64) - exact) <= tol)


def test_one_workspace_for_calls_of_any_size_and_two_graphs(hip):
    """Few rows cut into parts and many rows uncut, captured and eager ones in turn, over one workspace."""
    rng = np.random.default_rng(9)
    cases = [Case(rng, "float16", 64, 2, 16, news, lens).device() for news, lens in (([1], [2000]), ([200], [300]), ([1] * 5, [900, 20, 400, 1, 1500]))]
    tops = (100, 6, 33)
    ws = Tensor.zeros((hip.jsgrad_hip_attn_selected_workspace_bytes(8, 2, 64),), "uint8")
    data, graphs = [], []
    for c, top in zip(cases, tops):
        codes, scales = everything(c, *arrays(c, rng))
        t = [Tensor(rng.standard_normal((c.rows, 8, 64)).astype(np.float16)), Tensor(codes), Tensor(scales), Tensor.zeros((c.rows, 2, top), "int32"), Tensor.zeros((c.rows, 8, 64), "float16")]

        def call(c=c, t=t, top=top):
            check(hip.jsgrad_hip_paged_bounds(*c.batch, t[1].ptr, t[2].ptr))
            check(hip.jsgrad_hip_paged_select(*c.batch, t[0].ptr, 8, t[1].ptr, t[2].ptr, 1, 1, top, t[3].ptr))
            check(hip.jsgrad_hip_attn_selected(*c.batch, t[0].ptr, t[4].ptr, 8, t[3].ptr, top, ws.ptr))
        call()
        g = C.c_void_p()
        check(hip.jsgrad_hip_graph_begin())
        call()
        check(hip.jsgrad_hip_graph_end(C.byref(g)))
        data.append((t, call))
        graphs.append(g)
    for turn in range(3):
        for (c, (t, call), g, top) in zip(cases, data, graphs, tops):
            q = rng.standard_normal((c.rows, 8, 64)).astype(np.float16)
            t[0].lazydata.copyin(q.reshape(-1))
            check(hip.jsgrad_hip_graph_launch(g))
            sel, out = t[3].numpy(), t[4].numpy()
            exact, tol = ref.attention(c, q, 8, sel)
            assert np.all(np.abs(out.astype(np.float64) - exact) <= tol)
            data[turn][1]()
            call()
            assert np.array_equal(t[4].numpy(), out) and np.array_equal(t[3].numpy(), sel)
    for g in graphs:
        check(hip.jsgrad_hip_graph_destroy(g))
    assert not ws.numpy()[:4096].any()                        # counters are zero again


def test_a_wide_table(hip):
    """32768 columns, nearly all of them pages that the sequence has once each and again: scores repeat, ties go to the lower column."""
    rng = np.random.default_rng(10)
    c = Case(rng, "float16", 64, 1, 16, [1], [1000])
    pages = c.table[0, :62].copy()
    c.table = np.concatenate([np.tile(pages, 528), np.full(32, -1)]).astype(np.int32)[None, :32768]
    c.lens = [32736 * 16]
    c.device()
    codes, scales = arrays(c, rng)
    q = rng.standard_normal((1, 4, 64)).astype(np.float16)
    for top in (5, 1024):
        sel = run_choose(hip, c, q, 4, codes, scales, 2, 3, top)
        assert np.array_equal(sel, ref.choose(c, q, 4, codes, scales, 2, 3, top, np.full(sel.shape, 77, np.int32)))


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_a_model_over_chosen_pages(hip, dtype):
    """While all pages of a sequence fit the choice, the logits are those of attention over everything, to the rounding of its sums; beyond, prompts in pieces and forks go on alike."""
    cfg, llm = model()
    m, rng = llm.model, np.random.default_rng(11)
    prompts = [rng.integers(0, cfg["vocab_size"], n).astype(np.int32) for n in (40, 100, 3)]
    full = cache_for(llm, 64, dtype=dtype)
    cache = PagedCache(len(m.layers), m.n_kv_heads, m.dim // m.n_heads, 64, 16, dtype, bounds=True)
    sf, sc = [full.add() for _ in prompts], [cache.add() for _ in prompts]
    m.forward_paged(full, sf, prompts)
    want = logits(m, 3)
    m.forward_paged(cache, sc, prompts, choose=(1, 2, 10))
    assert np.max(np.abs(want - logits(m, 3))) <= 1e-2 * np.abs(want).max()
    for choose in ((1, 2, 10), (1, 1, 3)):
        toks = rng.integers(0, cfg["vocab_size"], (3, 1)).astype(np.int32)
        m.forward_paged(full, sf, toks)
        want = logits(m, 3)
        m.forward_paged(cache, sc, toks, choose=choose)
        off = np.max(np.abs(want - logits(m, 3)), -1) / np.abs(want).max(-1)
        assert off[2] <= 1e-2 and (off[1] <= 1e-2) == (choose[2] == 10)
    # a fork has the bounds of the pages that it shares, and a packed pool has them where the pages are
    f = cache.fork(sc[1])
    tok = [np.array([5], np.int32)]
    cache.compact()
    m.forward_paged(cache, [f], tok, choose=(1, 1, 3))
    a = logits(m, 1)
    m.forward_paged(cache, [sc[1]], tok, choose=(1, 1, 3))
    assert np.array_equal(a, logits(m, 1))
    for l in range(len(m.layers)):
        codes, scales = (t.numpy() for t in cache.bounds[l])
        pool = cache.pools[l].numpy()[0].astype(np.float32)
        if dtype == "int8":
            pool = pool * cache.scales[l].numpy()[0][..., None]
        for s in (*sc, f):
            for i, at in enumerate(cache.pages[s]):
                rows = pool[at, :, :min(16, cache.lengths[s] - 16 * i)]
                for g in range(2):
                    u = ref.step(np.abs(rows[g]).max())
                    assert scales[at, g] == u and np.array_equal(codes[at, g, 0], np.floor(rows[g].min(0) / u)) and np.array_equal(codes[at, g, 1], np.ceil(rows[g].max(0) / u))
    assert llm.generate_paged(prompts, 5, page_size=16, choose=(1, 1, 3), samples=2, temperature=0.7, dtype=dtype).shape == (6, 5)
    for bad in (lambda: m.forward_paged(full, sf, tok * 3, choose=(1, 1, 3)), lambda: m.forward_paged(cache, [f], tok, 5, choose=(1, 1, 3))):
        with pytest.raises(ValueError, match="bounds"):
            bad()
    before = dict(cache.lengths)
    with pytest.raises(Exception, match="recent"):
        m.forward_paged(cache, [f], tok, choose=(3, 1, 3))
    assert cache.lengths == before
