"""Normed writes, bounds, choice and attention over chosen pages where something is out of the ordinary: captured launches, arrays with anything in them, pools beyond 32-bit offsets, lists that are kept."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.ffi import check
from denograd_amd.paged import PagedCache
from denograd_amd.tensor import Tensor
from tests.paged_ref import Case
from tests.test_gpu_paged_model import model

pytestmark = pytest.mark.gpu

EPS = 1e-5


def normed(x, w):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w.astype(np.float64)


class Step:
    """What a serving step calls on a batch, over pools of its own or given ones."""

    def __init__(self, hip, desc, starts, lens, n_seqs, rows, H, KV, hd, bounds, choose, guard=2):
        self.hip, self.args, self.H, self.choose, self.bounds, self.rows = hip, (desc, starts.ptr, lens.ptr, n_seqs, rows), H, choose, bounds, rows
        self.keep = starts, lens
        most = rows + guard
        self.q, self.k, self.v = (Tensor.zeros((most, h, hd), "float16") for h in (H, KV, KV))
        self.w = Tensor((1 + 0.25 * np.cos(np.arange(hd))).astype(np.float16))
        self.q_out, self.out = Tensor.full((most, H, hd), 7.0, "float16"), Tensor.full((most, H, hd), 7.0, "float16")
        self.sel = Tensor(np.full((most, KV, choose[2]), 77, np.int32))
        self.ws = Tensor.zeros((hip.jsgrad_hip_attn_selected_workspace_bytes(H, KV, hd),), "uint8")

    def fill(self, rng):
        self.host = [rng.standard_normal(t.shape).astype(np.float16) for t in (self.q, self.k, self.v)]
        for t, x in zip((self.q, self.k, self.v), self.host):
            t.lazydata.copyin(x.reshape(-1))

    def __call__(self):
        check(self.hip.jsgrad_hip_paged_write_norm(*self.args, self.q.ptr, self.k.ptr, self.v.ptr, self.w.ptr, self.w.ptr, EPS, None, 0, self.q_out.ptr, self.H))
        check(self.hip.jsgrad_hip_paged_bounds(*self.args, self.bounds[0].ptr, self.bounds[1].ptr))
        check(self.hip.jsgrad_hip_paged_select(*self.args, self.q_out.ptr, self.H, self.bounds[0].ptr, self.bounds[1].ptr, *self.choose, self.sel.ptr))
        check(self.hip.jsgrad_hip_attn_selected(*self.args, self.q_out.ptr, self.out.ptr, self.H, self.sel.ptr, self.choose[2], self.ws.ptr))

    def results(self):
        return [t.numpy() for t in (self.q_out, self.sel, self.out)]


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_captured_step_follows_its_arrays(hip, kind, hd):
    """One graph, replayed with other rows, row starts, lengths and tables, a batch filled up among them, and eager calls between; every replay against the eager calls on pools that hold the same."""
    rng = np.random.default_rng(hd)
    cases = [Case(np.random.default_rng(9), kind, hd, 2, 16, [3, 9, 0], [40, 130, 20], extra_rows=0).device() for _ in range(2)]
    steps = []
    for c in cases:
        bounds = Tensor(np.zeros((c.n_pages, 2, 2, hd), np.int8)), Tensor(np.ones((c.n_pages, 2), np.float32))
        steps.append(Step(hip, c.desc, c.t["starts"], c.t["lens"], 3, 12, 8, 2, hd, bounds, (1, 1, 4)))
    graph = C.c_void_p()
    for s in steps:
        s.fill(np.random.default_rng(1))
    steps[0](), steps[1]()
    check(hip.jsgrad_hip_graph_begin())
    steps[0]()
    check(hip.jsgrad_hip_graph_end(C.byref(graph)))
    for starts, lens, swap in (([0, 3, 12, 12], [40, 130, 20], False), ([0, 1, 2, 3], [41, 131, 21], False), ([0, 0, 10, 12], [0, 140, 23], True), ([0, 12, 12, 12], [48, 3, 2], False)):
        seed = int(rng.integers(1 << 30))
        table = cases[0].table.copy()
        if swap:
            table[[0, 2]] = table[[2, 0]]
        for c, s in zip(cases, steps):
            s.fill(np.random.default_rng(seed))
            for name, x in (("starts", starts), ("lens", lens), ("table", table.reshape(-1))):
                c.t[name].lazydata.copyin(np.array(x, np.int32))
        check(hip.jsgrad_hip_graph_launch(graph))
        steps[1]()
        for a, b in zip(steps[0].results(), steps[1].results()):
            assert np.array_equal(a, b)
        for name in ("k", "v") + (("sk", "sv") if kind == "int8" else ()):
            assert np.array_equal(cases[0].t[name].numpy(), cases[1].t[name].numpy())
        n = starts[-1]
        got = steps[0].results()[0][:n].astype(np.float64)
        want = normed(steps[0].host[0][:n], steps[0].w.numpy())
        assert np.all(np.abs(got - want) <= (2.0 ** -11 + 2.0 ** -24 * (hd / 2 + 9)) * np.abs(want) + 2.0 ** -25)
        for i in (0, 1):
            assert np.array_equal(steps[0].bounds[i].numpy(), steps[1].bounds[i].numpy())
    check(hip.jsgrad_hip_graph_destroy(graph))


@pytest.mark.parametrize("rows", [9, 2100])
def test_arrays_with_anything_in_them_reach_no_other_memory(hip, rows):
    """Row starts that fall or lie outside, lengths below zero and behind the table, entries of the table that are no pages: the calls return and leave what is behind their outputs as it was; rows of no
    sequence keep what they had."""
    n = rows // 3
    for kind, hd in (("float16", 64), ("int8", 128)):
        for starts, lens in (([0, 5, 3, rows], [5, 7, 6]), ([0, 100 * rows, rows, rows], [3, 2, 1]), ([-4, 2, 10 * rows, -1], [-3, 2 ** 31 - 1, 50]), ([0, n, 2 * n, 3 * n], [1, 0, -2 ** 31]),
                             ([0, n, 2 * n, rows], [400, 2, 33]), ([rows, rows, rows, rows], [9, 9, 9]), ([2 ** 31 - 1, -2 ** 31, 7, 5], [30, 40, 50])):
            rng = np.random.default_rng(4)
            c = Case(rng, kind, hd, 2, 16, [3, 3, 3], [30, 40, 50])
            c.starts, c.lens = np.array(starts, np.int32), lens
            c.table[1, 1], c.table[2, 0] = c.n_pages, -2 ** 31
            c.device()
            # a page more than the pool has: it stays as it is
            bounds = Tensor(np.full((c.n_pages + 1, 2, 2, hd), 55, np.int8)), Tensor(np.full((c.n_pages + 1, 2), 3.0, np.float32))
            s = Step(hip, c.desc, c.t["starts"], c.t["lens"], 3, rows, 8, 2, hd, bounds, (1, 1, 3))
            s.fill(rng)
            s()
            q_out, sel, out = s.results()
            assert np.all(q_out[rows:] == 7) and np.all(sel[rows:] == 77) and np.all(out[rows:] == 7)
            assert np.all(bounds[0].numpy()[c.n_pages] == 55) and np.all(bounds[1].numpy()[c.n_pages] == 3)
            assert np.all((sel == 77) | ((sel >= -1) & (sel < c.width)))
            if starts[0] == rows:
                assert np.all(q_out == 7) and np.all(sel == 77) and np.all(out == 7)
            if lens == [1, 0, -2 ** 31]:                      # one row alone is at a position that is there
                assert np.all(sel[:n - 1] == -1) and not out[:n - 1].any() and np.all(sel[n:3 * n] == -1) and not out[n:3 * n].any() and np.all(sel[n - 1] == [0, -1, -1])
            assert not s.ws.numpy()[:4096].any()


def test_pools_beyond_32_bit_offsets(hip):
    """int8 pages of 4.6 GB: rows written to, looked over, chosen, attended and copied at both ends give what they give in a small pool."""
    hd, KV, page, H, n = 128, 8, 256, 16, 600
    many = (4600 << 20) // (KV * page * hd)
    results = []
    for n_pages, ids in ((many, [many - 1, 3, many - 2]), (5, [0, 1, 2])):
        pools, scales = [Tensor.zeros((n_pages, KV, page, hd), "int8") for _ in range(2)], [Tensor.zeros((n_pages, KV, page), "float32") for _ in range(2)]
        bounds = Tensor.zeros((n_pages, KV, 2, hd), "int8"), Tensor.zeros((n_pages, KV), "float32")
        table, starts, lens = Tensor(np.array([ids], np.int32)), Tensor(np.array([0, n], np.int32)), Tensor(np.array([n], np.int32))
        desc = ffi.PagesDesc(ffi.W_I8, n_pages, page, KV, hd, 3, pools[0].ptr, pools[1].ptr, scales[0].ptr, scales[1].ptr, table.ptr)
        s = Step(hip, desc, starts, lens, 1, n, H, KV, hd, bounds, (0, 1, 2))
        s.fill(np.random.default_rng(2))
        s()
        first = s.results()
        # the first page to another place, and everything again without a write
        to = n_pages - 3 if n_pages == many else 4
        held = [ffi.Pool(t.ptr, KV, page, b) for t, b in zip((*pools, *scales), (hd, hd, 4, 4))] + [ffi.Pool(bounds[0].ptr, 1, 1, KV * 2 * hd), ffi.Pool(bounds[1].ptr, 1, 1, KV * 4)]
        moves = Tensor(np.array([[ids[0], to, page]], np.int32))
        check(hip.jsgrad_hip_paged_copy((ffi.Pool * 6)(*held), 6, n_pages, moves.ptr, 1))
        table.lazydata.copyin(np.array([to, *ids[1:]], np.int32))
        s.out.lazydata.copyin(np.zeros(s.out.numel, np.float16))
        check(hip.jsgrad_hip_paged_select(*s.args, s.q_out.ptr, H, bounds[0].ptr, bounds[1].ptr, 0, 1, 2, s.sel.ptr))
        check(hip.jsgrad_hip_attn_selected(*s.args, s.q_out.ptr, s.out.ptr, H, s.sel.ptr, 2, s.ws.ptr))
        again = s.results()
        assert np.array_equal(first[1][:n], again[1][:n]) and np.array_equal(first[2][:n], again[2][:n])
        results.append(first)
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    assert np.isfinite(results[0][2].astype(np.float32)).all() and np.abs(results[0][2][:n].astype(np.float32)).max() > 0.1


def test_lists_that_are_kept(hip):
    """Every choice has an array of its own, or the caller's."""
    rng = np.random.default_rng(3)
    cache = PagedCache(1, 2, 64, 12, 16, bounds=True)
    a = cache.add()
    batch = cache.begin([a], [150])
    rows = [Tensor(rng.standard_normal((150, h, 64)).astype(np.float16)) for h in (2, 2, 4)]
    batch.write(0, rows[0], rows[1])
    lists, outs = [], []
    for i in range(2):
        q = Tensor(rng.standard_normal((150, 4, 64)).astype(np.float16))
        lists.append(batch.choose(0, q, 4, 1, 1, 3))
        outs.append((lists[-1].numpy(), batch.attend_chosen(0, q, 4, 1, 1, 3).numpy(), batch.attend_pages(0, q, 4, lists[-1]).numpy()))
    assert not np.array_equal(outs[0][0], outs[1][0])
    for t, (sel, chosen, pages) in zip(lists, outs):
        assert np.array_equal(t.numpy(), sel) and np.array_equal(chosen, pages)
    mine = Tensor.zeros((150, 2, 3), "int32")
    assert batch.choose(0, q, 4, 1, 1, 3, mine) is mine and np.array_equal(mine.numpy(), outs[1][0])
    with pytest.raises(ValueError, match="out"):
        batch.choose(0, q, 4, 1, 1, 4, mine)
    with pytest.raises(Exception, match="pages"):
        batch.choose(0, q, 4, 1, 1, 0)


def test_settings_that_no_row_can_have(hip):
    llm = model()[1]
    for bad in (dict(temperature=-1.0), dict(temperature=np.nan), dict(top_p=1.5), dict(min_p=-0.1), dict(top_k=-1), dict(samples=0)):
        with pytest.raises(ValueError):
            llm.generate_paged([[1, 2, 3]], 2, page_size=16, **bad)
