"""The paged KV cache against float64: rows written (rotated, fp16 or int8), read back, and attention of ragged batches over them."""
import numpy as np
import pytest

from denograd_amd.ffi import check
from denograd_amd.tensor import Tensor
from tests.paged_ref import U16, U32, Case, attention, quantise

pytestmark = pytest.mark.gpu


def rope_table(n, hd, rng):
    angle = np.outer(np.arange(n), 500000.0 ** (-np.arange(0, hd, 2) / hd))
    return np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float16)


def rotate(x, cs):
    """float32 with the rounding of every product, as the framework's other rotary epilogues have it.  x [rows, heads, hd], cs [rows, hd/2, 2]."""
    x, c, s = x.astype(np.float32), cs[:, None, :, 0].astype(np.float32), cs[:, None, :, 1].astype(np.float32)
    e, o = x[..., 0::2], x[..., 1::2]
    return np.stack([e * c - o * s, e * s + o * c], -1).reshape(x.shape)


WRITES = [  # kind, hd, H, KV, page, new rows, lengths
    ("float16", 64, 4, 2, 16, [1], [1]), ("int8", 64, 4, 2, 16, [1], [40]), ("float16", 128, 32, 8, 64, [5, 0, 17, 1], [5, 9, 200, 64]),
    ("int8", 128, 32, 8, 64, [5, 0, 17, 1], [5, 9, 200, 64]), ("int8", 128, 3, 1, 32, [33], [97]), ("float16", 64, 7, 7, 256, [2] * 9, [2, 3, 255, 256, 257, 258, 600, 4, 5]),
    ("int8", 64, 24, 8, 128, [1] * 130, list(range(1, 131))), ("int8", 128, 64, 8, 16, [700, 3], [700, 1000]),
]


@pytest.mark.parametrize("kind,hd,H,KV,page,news,lens", WRITES)
def test_rows_written_and_read_back(hip, kind, hd, H, KV, page, news, lens):
    """fp16 rows are exact: the same float operations, rounded once.  int8: a scale is off by its division's rounding, a code by half a step and what
    the quotient's rounding adds, U32 of up to 127."""
    rng = np.random.default_rng(hd + H + page + len(news))
    c = Case(rng, kind, hd, KV, page, news, lens, extra_rows=2).device()
    n = int(c.starts[-1])
    q, k, v = (rng.standard_normal((c.rows, h, hd)).astype(np.float16) for h in (H, KV, KV))
    k *= np.float16(3)
    v[0, 0] = 0
    cs = rope_table(c.width * page, hd, rng)
    tq, tk, tv, tc, to = Tensor(q), Tensor(k), Tensor(v), Tensor(cs), Tensor.full(q.shape, 7.0, "float16")
    check(hip.jsgrad_hip_paged_write(*c.batch, tq.ptr, tk.ptr, tv.ptr, tc.ptr, cs.shape[0], to.ptr, H))
    pos = np.concatenate([np.arange(l - m, l) for m, l in zip(news, lens)])
    place = [c.places(b, l - m, l) for b, (m, l) in enumerate(zip(news, lens))]
    ids, slots = (np.concatenate([p[i] for p in place]) for i in (0, 1))
    want_q, want_k, want_v = rotate(q[:n], cs[pos]), rotate(k[:n], cs[pos]), v[:n].astype(np.float32)
    got_q = to.numpy()
    assert np.array_equal(got_q[:n], want_q.astype(np.float16)) and np.all(got_q[n:] == 7)
    rk, rv = Tensor.full(k.shape, 7.0, "float16"), Tensor.full(v.shape, 7.0, "float16")
    check(hip.jsgrad_hip_paged_read(*c.batch, rk.ptr, rv.ptr))
    for name, want, before, read in (("k", want_k, c.k, rk.numpy()), ("v", want_v, c.v, rv.numpy())):
        pool = c.t[name].numpy()
        got = pool[ids, :, slots]
        if kind == "float16":
            assert np.array_equal(got, want.astype(np.float16))
            assert np.array_equal(read[:n], got)
        else:
            scales = c.t["s" + name].numpy()
            s, top = scales[ids, :, slots], np.abs(want).max(-1)
            assert np.all(np.abs(s - np.where(top == 0, 1, top / 127.0)) <= 2 * U32 * np.maximum(s, top / 127.0))
            assert np.all(np.abs(got - want / s[..., None]) <= 0.5 + 2 * 127 * U32)
            assert np.array_equal(read[:n], (got.astype(np.float32) * s[..., None]).astype(np.float16))
            old = c.sk if name == "k" else c.sv
            old, new = old.copy(), scales.copy()
            old[ids, :, slots] = new[ids, :, slots] = 0
            assert np.array_equal(old, new)
        untouched = (before if kind == "float16" else (c.ck if name == "k" else c.cv)).copy()
        pool = pool.copy()
        untouched[ids, :, slots] = 0
        pool[ids, :, slots] = 0
        assert np.array_equal(pool, untouched)              # nothing beside the batch's places
        assert np.all(read[n:] == 7)


@pytest.mark.parametrize("kind,hd,KV,page,news,lens", [
    ("float16", 64, 2, 16, [12800], [13000]), ("int8", 128, 2, 32, [5000, 0, 3, 8000, 1], [5000, 3, 3, 9000, 77]), ("int8", 64, 3, 256, [100] * 130 + [0] * 9, [120] * 130 + [5] * 9),
    ("float16", 128, 1, 16, [1] * 20 + [12500] + [2] * 70, [9] * 20 + [12500] + [600] * 70),
])
def test_many_rows_read(hip, kind, hd, KV, page, news, lens):
    """More than 12288 rows: eight to a block, of one sequence or several, some without a page, some that no sequence has."""
    rng = np.random.default_rng(hd + KV)
    c = Case(rng, kind, hd, KV, page, news, lens, extra_rows=13)
    c.table[0, c.width // 2] = c.n_pages + 5
    c.table[-1, 0] = -9
    c.device()
    out = [Tensor.full((c.rows + 1, KV, hd), 7.0, "float16") for _ in range(2)]
    check(hip.jsgrad_hip_paged_read(*c.batch, out[0].ptr, out[1].ptr))
    place = [c.places(b, l - m, l) for b, (m, l) in enumerate(zip(news, lens))]
    ids, slots = (np.concatenate([p[i] for p in place]) for i in (0, 1))
    n = int(c.starts[-1])
    for name, t in zip("kv", out):
        got = t.numpy()
        if kind == "int8":
            codes, scales = (c.ck, c.sk) if name == "k" else (c.cv, c.sv)
            want = (codes[ids, :, slots].astype(np.float32) * scales[ids, :, slots][..., None]).astype(np.float16)
        else:
            want = getattr(c, name)[ids, :, slots]
        assert np.array_equal(got[:n], np.where((ids < 0)[:, None, None], np.float16(0), want)) and np.all(got[n:] == 7)


def test_a_write_without_rotation_queries_or_pages(hip):
    """No rope table: rows as they are.  No q: only the cache.  q_out may be q.  Rows without a page leave no trace and read as zeros; their queries are
    rotated all the same where the table has the position."""
    rng = np.random.default_rng(3)
    c = Case(rng, "float16", 64, 2, 16, [40, 4], [40, 6])
    c.table[0, 1], c.table[0, 2], c.table[1, 0] = -1, c.n_pages, 0x7fffffff
    c.device()
    k, v, q = (rng.standard_normal((c.rows, h, 64)).astype(np.float16) for h in (2, 2, 4))
    tk, tv, tq = Tensor(k), Tensor(v), Tensor(q)
    check(hip.jsgrad_hip_paged_write(*c.batch, None, tk.ptr, tv.ptr, None, 0, None, 0))
    rk, rv = Tensor.full(k.shape, 7.0, "float16"), Tensor.full(v.shape, 7.0, "float16")
    check(hip.jsgrad_hip_paged_read(*c.batch, rk.ptr, rv.ptr))
    for got, x, name, before in ((rk, k, "k", c.k), (rv, v, "v", c.v)):
        want = x.copy()
        want[16:] = 0
        assert np.array_equal(got.numpy(), want)
        pool = c.t[name].numpy().copy()
        assert np.array_equal(pool[c.table[0, 0]].transpose(1, 0, 2), x[:16])
        pool[c.table[0, 0]] = before[c.table[0, 0]]
        assert np.array_equal(pool, before)
    cs = rope_table(c.width * 16, 64, rng)
    tc = Tensor(cs)
    check(hip.jsgrad_hip_paged_write(*c.batch, tq.ptr, tk.ptr, tv.ptr, tc.ptr, cs.shape[0], tq.ptr, 4))
    pos = np.concatenate([np.arange(40), np.arange(2, 6)])
    assert np.array_equal(tq.numpy(), rotate(q, cs[pos]).astype(np.float16))


def test_arrays_with_anything_in_them_reach_no_other_memory(hip):
    """Row starts that fall or lie outside, lengths below zero and behind the table, more new rows than positions: what has a place is written, all
    else stays.  (Which rows those are is not promised for falling starts; that the calls return and leave their surroundings is.)"""
    rng = np.random.default_rng(4)
    for starts, lens in (([0, 5, 3, 9], [5, 7, 6]), ([0, 100, 9, 9], [3, 2, 1]), ([-4, 2, 1000, -1], [-3, 2 ** 31 - 1, 50]), ([0, 3, 6, 9], [1, 0, -2 ** 31]), ([0, 3, 6, 9], [400, 2, 33])):
        c = Case(rng, "int8", 64, 2, 16, [3, 3, 3], [30, 40, 50])
        c.starts, c.lens = np.array(starts, np.int32), lens
        c.rows = 9
        c.device()
        k, v, q = (rng.standard_normal((11, h, 64)).astype(np.float16) for h in (2, 2, 4))
        tk, tv, tq, to = Tensor(k), Tensor(v), Tensor(q), Tensor.full((11, 4, 64), 7.0, "float16")
        cs = rope_table(c.width * 16, 64, rng)
        tc = Tensor(cs)
        check(hip.jsgrad_hip_paged_write(*c.batch, tq.ptr, tk.ptr, tv.ptr, tc.ptr, cs.shape[0], to.ptr, 4))
        rk, rv = Tensor.full(k.shape, 7.0, "float16"), Tensor.full(v.shape, 7.0, "float16")
        check(hip.jsgrad_hip_paged_read(*c.batch, rk.ptr, rv.ptr))
        out, ws = Tensor.full((11, 4, 64), 7.0, "float16"), Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(4, 2, 64),), "uint8")
        check(hip.jsgrad_hip_attn_paged(*c.batch, tq.ptr, out.ptr, 4, 0, 0, ws.ptr))
        for t in (to, rk, rv, out):
            assert np.all(t.numpy()[9:] == 7)
        if starts == [0, 3, 6, 9] and lens[0] == 1:           # rows at -2, -1, 0; -3 .. -1; -3 .. -1
            got = out.numpy()
            assert not got[[0, 1, 3, 4, 5, 6, 7, 8]].any() and got[2].any()
            assert np.all(to.numpy()[[0, 1, 3, 4, 5, 6, 7, 8]] == 7)


def test_rows_of_zeros_and_rows_that_are_not_finite(hip):
    rng = np.random.default_rng(5)
    for hd in (64, 128):
        c = Case(rng, "int8", hd, 2, 16, [6], [6]).device()
        k, v = (rng.standard_normal((6, 2, hd)).astype(np.float16) for _ in range(2))
        k[0], k[1, 0, 5], k[2, 1, hd - 1], v[3, 0, 0], v[4] = 0, np.nan, np.inf, -np.inf, np.float16(6e-8)
        v[5, 0], v[5, 0, 7] = 0, np.float16(-65504)
        tk, tv = Tensor(k), Tensor(v)
        check(hip.jsgrad_hip_paged_write(*c.batch, None, tk.ptr, tv.ptr, None, 0, None, 0))
        rk, rv = Tensor.zeros(k.shape, "float16"), Tensor.zeros(v.shape, "float16")
        check(hip.jsgrad_hip_paged_read(*c.batch, rk.ptr, rv.ptr))
        for got, x in ((rk.numpy(), k), (rv.numpy(), v)):
            bad = ~np.isfinite(x).all(-1)
            assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
            codes, scales = quantise(x)
            assert np.array_equal(got[~bad], (codes.astype(np.float32) * scales[..., None]).astype(np.float16)[~bad])
        assert np.array_equal(c.t["sk"].numpy()[c.table[0, 0], :, 0], [1, 1])


ATTN = [  # kind, hd, H, KV, page, new rows, lengths, window, sinks
    ("float16", 64, 4, 2, 16, [1], [1], 0, 0), ("int8", 64, 4, 2, 16, [1], [1], 0, 0),
    ("float16", 128, 8, 2, 64, [1, 1, 1], [1, 64, 65], 0, 0), ("int8", 128, 8, 2, 64, [1, 1, 1], [63, 640, 1000], 0, 0),
    ("float16", 64, 32, 8, 32, [1], [700], 0, 0), ("int8", 64, 32, 8, 256, [1] * 5, [700, 3, 33, 1500, 257], 0, 0),
    ("float16", 128, 4, 1, 16, [37], [37], 0, 0), ("int8", 128, 4, 1, 16, [37], [137], 0, 0),
    ("float16", 64, 6, 2, 128, [130, 0, 1, 65], [130, 10, 300, 65], 0, 0), ("int8", 64, 6, 2, 128, [130, 0, 1, 65], [130, 10, 300, 65], 0, 0),
    ("float16", 128, 3, 3, 64, [200], [321], 0, 0), ("int8", 128, 3, 3, 64, [200], [321], 0, 0),
    ("float16", 64, 8, 1, 16, [40], [90], 0, 0), ("int8", 64, 16, 1, 16, [40], [90], 0, 0), ("float16", 64, 24, 1, 32, [3, 20], [90, 20], 0, 0),
    ("float16", 64, 4, 2, 16, [70, 1], [200, 150], 1, 0), ("int8", 64, 4, 2, 16, [70, 1], [200, 150], 1, 3),
    ("float16", 128, 4, 2, 32, [100, 1, 1], [400, 500, 20], 50, 4), ("int8", 128, 4, 2, 32, [100, 1, 1], [400, 500, 20], 50, 4),
    ("float16", 64, 4, 2, 64, [150, 2], [600, 700], 128, 130), ("int8", 64, 4, 2, 64, [150, 2], [600, 700], 64, 64),
    ("float16", 64, 8, 2, 16, [1] * 3, [1500, 1200, 77], 300, 65), ("int8", 128, 8, 2, 64, [1] * 3, [1500, 1200, 77], 300, 65),
    ("float16", 64, 4, 2, 16, [2], [2], 2 ** 31 - 1, 2 ** 31 - 1),
]


def run_attention(hip, c, q, H, window, sinks, ws=None, times=1):
    ws = ws if ws is not None else Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(H, c.KV, c.hd),), "uint8")
    tq = Tensor(q)
    got = None
    for _ in range(times):
        out = Tensor.full((c.rows + 1, H, c.hd), 7.0, "float16")
        check(hip.jsgrad_hip_attn_paged(*c.batch, tq.ptr, out.ptr, H, window, sinks, ws.ptr))
        one = out.numpy()
        assert np.all(one[c.starts[-1]:] == 7)
        assert got is None or np.array_equal(one, got, equal_nan=True)      # the workspace is left as it was found
        got = one
    return got[:c.rows]


def compare(got, ref, tol, rows):
    bad = np.abs(got[:rows].astype(np.float64) - ref[:rows]) > tol[:rows]
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got[:rows] - ref[:rows])[bad].max())


@pytest.mark.parametrize("kind,hd,H,KV,page,news,lens,window,sinks", ATTN)
def test_attention_of_a_ragged_batch(hip, kind, hd, H, KV, page, news, lens, window, sinks):
    rng = np.random.default_rng(hd * 7 + H + page + sum(lens))
    c = Case(rng, kind, hd, KV, page, news, lens, extra_rows=1).device()
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    ref, tol = attention(c, q, H, window, sinks)
    got = run_attention(hip, c, q, H, window, sinks, times=2)
    compare(got, ref, tol, int(c.starts[-1]))


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd,H,KV,news,lens", [(64, 8, 2, [1], [300]), (128, 8, 2, [1, 1], [70, 200]), (64, 8, 2, [3, 0, 40], [3, 9, 700]), (128, 4, 4, [16], [90]), (128, 4, 4, [17, 16], [90, 400]),
                                                (64, 34, 2, [1, 1], [200, 50])])
def test_a_batch_filled_up_with_rows_that_no_sequence_has(hip, kind, hd, H, KV, news, lens):
    """As a captured graph's batch is: many more rows than the sequences have, and sequences with none; both kinds of blocks in a launch."""
    rng = np.random.default_rng(hd + len(news))
    c = Case(rng, kind, hd, KV, 16, news + [0] * 5, lens + [0, 7, 0, 100, 1], extra_rows=200).device()
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    ref, tol = attention(c, q, H)
    compare(run_attention(hip, c, q, H, 0, 0, times=2), ref, tol, int(c.starts[-1]))


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd,news,lens", [(64, [1, 1], [900, 64]), (128, [90, 1], [400, 33])])
def test_large_scores_and_values_of_every_size(hip, kind, hd, news, lens):
    """Scores up to several hundred: one key has all the weight.  Values over eight orders of magnitude, those of int8 pages with scales as far apart."""
    rng = np.random.default_rng(hd)
    c = Case(rng, kind, hd, 2, 16, news, lens)
    size = (10.0 ** rng.uniform(-5, 3, c.v.shape[:3]))[..., None]
    c = Case(np.random.default_rng(hd), kind, hd, 2, 16, news, lens, k=(c.k * np.float16(6)).astype(np.float16), v=(c.v * size).astype(np.float16)).device()
    q = (rng.standard_normal((c.rows, 4, hd)) * 4).astype(np.float16)
    ref, tol = attention(c, q, 4)
    compare(run_attention(hip, c, q, 4, 0, 0), ref, tol, c.rows)


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd,H,news,lens,window,sinks", [(64, 4, [70, 1], [300, 77], 0, 0), (128, 2, [1, 1, 5], [65, 130, 500], 40, 3), (128, 6, [140], [140], 0, 0)])
def test_what_a_row_does_not_see_does_not_reach_it(hip, kind, hd, H, news, lens, window, sinks):
    """Places behind a sequence's end, other sequences' pages, positions outside the window and later rows of the chunk hold what is not a number."""
    rng = np.random.default_rng(hd + H)
    c = Case(rng, kind, hd, 2, 16, news, lens)
    mine = np.zeros(c.k.shape[:3], bool)
    for b, l in enumerate(lens):
        ids, slots = c.places(b, 0, l)
        if window:                                            # only what the last row sees; earlier rows lose keys that they had
            j = np.arange(l)
            ids, slots = ids[(j > l - 1 - window) | (j < sinks)], slots[(j > l - 1 - window) | (j < sinks)]
        mine[ids, :, slots] = True
    k, v = c.k.copy(), c.v.copy()
    k[~mine], v[~mine] = np.nan, np.inf
    c2 = Case(np.random.default_rng(hd + H), kind, hd, 2, 16, news, lens, k=k, v=v).device()
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    ref, tol = attention(c2, q, H, window, sinks)
    got = run_attention(hip, c2, q, H, window, sinks)
    fine = np.isfinite(ref).all(-1)
    assert fine[c.starts[1:] - 1].all()
    assert np.all(np.abs(got.astype(np.float64) - ref)[fine] <= tol[fine])
    if window == 0:
        # the last row of the first sequence's chunk is not a number: the rows before it are what they are without it
        ids, slots = c.places(0, lens[0] - 1, lens[0])
        k[ids[0], :, slots[0]], v[ids[0], :, slots[0]] = np.nan, np.nan
        c3 = Case(np.random.default_rng(hd + H), kind, hd, 2, 16, news, lens, k=k, v=v).device()
        again = run_attention(hip, c3, q, H, 0, 0)
        last = news[0] - 1
        assert np.isnan(again[last]).all()
        if last:
            assert np.all(np.abs(again[:last].astype(np.float64) - ref[:last]) <= tol[:last])


@pytest.mark.parametrize("kind", ["float16", "int8"])
def test_pages_that_are_not_there(hip, kind):
    """Entries outside the pool hold no keys, in the middle and everywhere; a row that sees nothing is zeros."""
    rng = np.random.default_rng(9)
    c = Case(rng, kind, 64, 2, 16, [20, 1, 1, 3], [200, 150, 40, 3])
    c.table[0, 2:5], c.table[1, 0], c.table[2, :], c.table[3, 0] = [-1, c.n_pages, -2 ** 31], 2 ** 31 - 1, -1, -7
    c.device()
    q = rng.standard_normal((c.rows, 4, 64)).astype(np.float16)
    for window, sinks in ((0, 0), (30, 4)):
        ref, tol = attention(c, q, 4, window, sinks)
        got = run_attention(hip, c, q, 4, window, sinks, times=2)
        compare(got, ref, tol, c.rows)
        assert not got[21:].any()


def in_chunks(c, H):
    """Room for more rows and positions than the batch has, as in a captured graph: a launch for so many has chunks for the sequences with more than a few rows."""
    c.rows += 24000 // H
    c.table = np.pad(c.table, ((0, 0), (0, -(-1100 // c.page))), constant_values=-1)
    c.width = c.table.shape[1]
    return c.device()


def padded(c, q):
    return np.concatenate([q, np.zeros((c.rows - q.shape[0], *q.shape[1:]), np.float16)])


@pytest.mark.parametrize("kind,hd,H,KV,page,news,lens,window,sinks", [a for a in ATTN if max(a[5]) * a[2] > 32 * a[3]])
def test_attention_of_a_ragged_batch_in_chunks(hip, kind, hd, H, KV, page, news, lens, window, sinks):
    rng = np.random.default_rng(hd * 7 + H + page + sum(lens))
    c = in_chunks(Case(rng, kind, hd, KV, page, news, lens), H)
    q = padded(c, rng.standard_normal((int(c.starts[-1]), H, hd)).astype(np.float16))
    ref, tol = attention(c, q, H, window, sinks)
    compare(run_attention(hip, c, q, H, window, sinks, times=2), ref, tol, int(c.starts[-1]))


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
def test_large_scores_and_values_of_every_size_in_chunks(hip, kind, hd):
    rng = np.random.default_rng(hd)
    news, lens = [90, 1, 40], [400, 33, 40]
    c = Case(rng, kind, hd, 2, 16, news, lens)
    size = (10.0 ** rng.uniform(-5, 3, c.v.shape[:3]))[..., None]
    c = in_chunks(Case(np.random.default_rng(hd), kind, hd, 2, 16, news, lens, k=(c.k * np.float16(6)).astype(np.float16), v=(c.v * size).astype(np.float16)), 4)
    q = padded(c, (rng.standard_normal((131, 4, hd)) * 4).astype(np.float16))
    ref, tol = attention(c, q, 4)
    compare(run_attention(hip, c, q, 4, 0, 0), ref, tol, 131)


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd,H,news,lens,window,sinks", [(64, 4, [70, 1], [300, 77], 0, 0), (128, 4, [33, 60], [130, 500], 40, 3), (128, 6, [140], [140], 0, 0)])
def test_what_a_row_does_not_see_does_not_reach_it_in_chunks(hip, kind, hd, H, news, lens, window, sinks):
    """Places that no row of the batch sees, and keys behind a row of its own chunk."""
    rng = np.random.default_rng(hd + H)
    c = Case(rng, kind, hd, 2, 16, news, lens)
    mine = np.zeros(c.k.shape[:3], bool)
    for b, (n, l) in enumerate(zip(news, lens)):
        ids, slots = c.places(b, 0, l)
        if window:
            j = np.arange(l)
            ids, slots = ids[(j > l - n - window) | (j < sinks)], slots[(j > l - n - window) | (j < sinks)]
        mine[ids, :, slots] = True
    k, v = c.k.copy(), c.v.copy()
    k[~mine], v[~mine] = np.nan, np.inf
    many = lambda: in_chunks(Case(np.random.default_rng(hd + H), kind, hd, 2, 16, news, lens, k=k, v=v), H)
    c2, n = many(), sum(news)
    q = padded(c2, rng.standard_normal((n, H, hd)).astype(np.float16))
    ref, tol = attention(c2, q, H, window, sinks)
    got = run_attention(hip, c2, q, H, window, sinks)
    assert np.isfinite(ref[:n]).all()
    compare(got, ref, tol, n)
    # a row in the middle of the first chunk is not a number: the rows before it are what they are without it, it and those that see it are not numbers
    at = news[0] // 2
    ids, slots = c.places(0, lens[0] - news[0] + at, lens[0] - news[0] + at + 1)
    k[ids[0], :, slots[0]], v[ids[0], :, slots[0]] = np.nan, np.nan
    again = run_attention(hip, many(), q, H, window, sinks)
    compare(again, ref, tol, at)
    assert np.isnan(again[at:at + 1]).all() and (window or np.isnan(again[at:news[0]]).all())
    # infinite values reach those that see them
    k[ids[0], :, slots[0]], v[ids[0], :, slots[0]] = c.k[ids[0], :, slots[0]], np.inf
    if kind == "float16":
        again = run_attention(hip, many(), q, H, window, sinks)
        compare(again, ref, tol, at)
        assert not np.isfinite(again[at:at + 1]).any()


@pytest.mark.parametrize("kind", ["float16", "int8"])
def test_pages_that_are_not_there_in_chunks(hip, kind):
    rng = np.random.default_rng(9)
    c = Case(rng, kind, 64, 2, 16, [50, 1, 20, 30], [200, 150, 40, 30])
    c.table[0, 2:5], c.table[1, 0], c.table[2, :], c.table[3, 0] = [-1, c.n_pages, -2 ** 31], 2 ** 31 - 1, -1, -7
    in_chunks(c, 4)
    q = padded(c, rng.standard_normal((101, 4, 64)).astype(np.float16))
    for window, sinks in ((0, 0), (30, 4)):
        ref, tol = attention(c, q, 4, window, sinks)
        got = run_attention(hip, c, q, 4, window, sinks, times=2)
        compare(got, ref, tol, 101)
        assert not got[51:71].any() and not got[71:87].any() and got[87:101].any()


@pytest.mark.parametrize("kind,hd", [("float16", 64), ("int8", 128)])
@pytest.mark.parametrize("news,lens", [([2] * 70, list(range(2, 702, 10))), ([8] * 5, [8, 9, 200, 500, 64]), ([1] * 65 + [9], [30] * 65 + [400]), ([2] * 40 + [300], [50] * 40 + [900]),
                                       ([17, 0, 0, 1], [1000, 0, 3, 40])])
def test_which_blocks_a_batch_has_is_found_on_the_device(hip, kind, hd, news, lens):
    """Around 32 pairs to a sequence, and more sequences than lanes, under a table with room for much more than they fill."""
    rng = np.random.default_rng(len(news) + hd)
    c = Case(rng, kind, hd, 2, 16, news, lens)
    c.table = np.pad(c.table, ((0, 0), (0, 5000)), constant_values=-1)
    c.width = c.table.shape[1]
    c.device()
    q = rng.standard_normal((c.rows, 8, hd)).astype(np.float16)
    ref, tol = attention(c, q, 8)
    compare(run_attention(hip, c, q, 8, 0, 0, times=2), ref, tol, c.rows)


def test_row_starts_that_fall_leave_the_workspace_as_it_was(hip):
    """512 sequences that all claim rows 0 to 3, and a long one behind them: a grid made for four rows has blocks for a part of that one's parts alone.
    Nothing is written, and the next call on this workspace gives what it would have."""
    rng = np.random.default_rng(12)
    c = Case(rng, "float16", 64, 2, 64, [0] * 1025, [20] * 1024 + [2000])
    c.starts, c.rows = np.array([0, 4] * 513, np.int32), 4
    c.device()
    ws, q, out = Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(4, 2, 64),), "uint8"), Tensor.zeros((4, 4, 64), "float16"), Tensor.full((4, 4, 64), 7.0, "float16")
    check(hip.jsgrad_hip_attn_paged(*c.batch, q.ptr, out.ptr, 4, 0, 0, ws.ptr))
    assert np.all(out.numpy() == 7)
    for news in ([1], [300]):
        good = Case(rng, "float16", 64, 2, 64, news, [2000]).device()
        x = rng.standard_normal((good.rows, 4, 64)).astype(np.float16)
        ref, tol = attention(good, x, 4)
        compare(run_attention(hip, good, x, 4, 0, 0, ws), ref, tol, good.rows)


@pytest.mark.parametrize("kind,hd,H,KV,news,lens,window,sinks", [
    ("float16", 128, 8, 2, [1], [20011], 0, 0), ("int8", 64, 8, 2, [1, 1], [9000, 30], 0, 0), ("int8", 128, 8, 2, [3], [9000], 0, 0), ("float16", 64, 4, 2, [60], [6000], 0, 0),
    ("int8", 128, 32, 8, [100, 1, 1, 1], [2500, 4000, 5, 1200], 0, 0), ("float16", 64, 8, 2, [1], [20000], 9000, 100), ("float16", 128, 32, 8, [1] * 70, list(range(1, 1401, 20)), 0, 0),
    ("int8", 64, 32, 8, [1] * 140, list(range(1, 1401, 10)), 0, 0), ("float16", 128, 32, 8, [300] + [1, 2, 4] * 7, [3000] + list(range(50, 2150, 100)), 0, 0),
    ("int8", 128, 8, 2, [1, 900, 4, 40] + [1] * 66, [9000, 900, 4, 3000] + [77] * 66, 500, 70), ("float16", 64, 8, 8, [2] * 65 + [40], list(range(2, 132, 2)) + [700], 0, 0),
])
def test_long_contexts_and_many_sequences(hip, kind, hd, H, KV, news, lens, window, sinks):
    """Keys in parts and their merge; more sequences than a wavefront has lanes.  A few rows and heads against float64, everything twice on one workspace."""
    rng = np.random.default_rng(len(lens) + lens[0])
    c = Case(rng, kind, hd, KV, 64, news, lens).device()
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    got = run_attention(hip, c, q, H, window, sinks, times=2)
    ref, tol = attention(c, q, H, window, sinks)
    compare(got, ref, tol, c.rows)


def test_a_pool_beyond_32_bit_offsets(hip):
    """int8 pages of 4.6 GB: rows written to and attended from the last page."""
    hd, KV, page, H = 128, 8, 256, 16
    n_pages = (4600 << 20) // (KV * page * hd)
    rng = np.random.default_rng(1)
    pools = [Tensor.zeros((n_pages, KV, page, hd), "int8") for _ in range(2)]
    scales = [Tensor.zeros((n_pages, KV, page), "float32") for _ in range(2)]
    from denograd_amd import ffi
    table = np.array([[n_pages - 1, 3, n_pages - 2]], np.int32)
    tt, st, ln = Tensor(table), Tensor(np.array([0, 600], np.int32)), Tensor(np.array([600], np.int32))
    desc = ffi.PagesDesc(ffi.W_I8, n_pages, page, KV, hd, 3, pools[0].ptr, pools[1].ptr, scales[0].ptr, scales[1].ptr, tt.ptr)
    k, v, q = (rng.standard_normal((600, h, hd)).astype(np.float16) for h in (KV, KV, H))
    tk, tv, tq = Tensor(k), Tensor(v), Tensor(q)
    check(hip.jsgrad_hip_paged_write(desc, st.ptr, ln.ptr, 1, 600, None, tk.ptr, tv.ptr, None, 0, None, 0))
    rk, rv = Tensor.zeros(k.shape, "float16"), Tensor.zeros(v.shape, "float16")
    check(hip.jsgrad_hip_paged_read(desc, st.ptr, ln.ptr, 1, 600, rk.ptr, rv.ptr))
    for got, x in ((rk, k), (rv, v)):
        codes, sc = quantise(x)
        assert np.all(np.abs(got.numpy().astype(np.float64) - x) <= sc[..., None] * (0.5 + 2 * 127 * U32) + U16 * np.abs(got.numpy()))
    small = Case(rng, "int8", hd, KV, page, [600], [600], spare=0)
    small.table = np.array([[0, 1, 2]], np.int32)
    for name in ("k", "v"):
        codes, sc = quantise(k if name == "k" else v)
        full, fs = np.zeros((3, KV, page, hd), np.int8), np.ones((3, KV, page), np.float32)
        for i in range(600):
            full[i // page, :, i % page], fs[i // page, :, i % page] = codes[i], sc[i]
        setattr(small, "c" + name, full), setattr(small, "s" + name, fs)
    ws, out = Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(H, KV, hd),), "uint8"), Tensor.zeros((600, H, hd), "float16")
    check(hip.jsgrad_hip_attn_paged(desc, st.ptr, ln.ptr, 1, 600, tq.ptr, out.ptr, H, 0, 0, ws.ptr))
    ref, tol = attention(small, q, H)
    # codes at the border of two steps may differ by one between the two quantisers: their share of the result
    tol = tol + 2.0 ** -20 * np.abs(v).max()
    assert np.mean(np.abs(out.numpy().astype(np.float64) - ref) <= tol) > 0.999
