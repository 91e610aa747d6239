"""Pages chosen for thousands of rows and attention over them: rows share tiles of the choice, and each wavefront of the attention has a row of its own."""
import numpy as np
import pytest

from tests import select_ref as ref
from tests.paged_ref import Case
from tests.test_gpu_paged_select import arrays, everything, run_attend, run_bounds, run_choose

pytestmark = pytest.mark.gpu

BATCHES = [  # kind, hd, H, KV, page, new rows, lengths, first, recent, top; the choice has tiles of 16 / (H / KV) rows, and with heads of 128 takes four of them at a time
    ("float16", 64, 32, 8, 16, [1500, 0, 33, 567], [2000, 100, 33, 5000], 1, 2, 12), ("int8", 128, 16, 2, 64, [4023, 77], [4023, 4999], 1, 1, 5),
    ("float16", 128, 16, 1, 32, [3001, 1100], [3001, 1900], 0, 1, 9), ("int8", 64, 6, 2, 16, [8201], [8300], 2, 3, 20), ("float16", 128, 16, 8, 256, [4099], [4200], 0, 1, 3),
    ("float16", 64, 16, 16, 128, [4001, 1, 95], [4001, 700, 800], 1, 1, 4), ("int8", 128, 20, 1, 16, [2050], [2100], 1, 1, 17), ("float16", 64, 40, 1, 16, [1400], [1500], 1, 1, 7),
    ("int8", 64, 3, 1, 64, [1] * 4100, [1 + 7 * i % 300 for i in range(4100)], 1, 1, 3), ("float16", 64, 8, 2, 16, [2055], [2055], 1, 2, 64), ("float16", 64, 8, 2, 16, [2055], [2055], 1, 2, 65),
]


@pytest.mark.parametrize("kind,hd,H,KV,page,news,lens,first,recent,top", BATCHES)
def test_many_rows(hip, kind, hd, H, KV, page, news, lens, first, recent, top):
    rng = np.random.default_rng(hd + H + page + top)
    c = Case(rng, kind, hd, KV, page, news, lens, extra_rows=3)
    c.table[0, c.width // 2 if len(lens) < 100 else 0] = -1   # a hole: rows of one page have none
    c.device()
    codes, scales = everything(c, *arrays(c, rng))
    got = run_bounds(hip, c, codes, scales)                   # again, in one call for all rows
    assert np.array_equal(got[0], codes) and np.array_equal(got[1], scales)
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    q[5], q[c.rows // 2, 0, 3], q[7, H - 1, 0] = 0, np.nan, np.inf
    sel = run_choose(hip, c, q, H, codes, scales, first, recent, top)
    want = ref.choose_many(c, q, H, codes, scales, first, recent, top, np.full(sel.shape, 77, np.int32))
    assert np.array_equal(sel, want)
    q[c.rows // 2], q[7] = q[1], q[2]
    out = run_attend(hip, c, q, H, sel)
    n, every = int(c.starts[-1]), max(1, c.rows * H // 16384)
    exact, tol = ref.attention(c, q, H, sel, every)
    for b, m in enumerate(news):
        rows = np.arange(c.starts[b], c.starts[b] + m, every)
        assert np.all(np.abs(out[rows].astype(np.float64) - exact[rows]) <= tol[rows])
    assert np.all(out[n:] == 7) and np.isfinite(out[:n].astype(np.float32)).all()
    assert np.array_equal(out, run_attend(hip, c, q, H, sel))


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd,H", [(64, 8), (128, 32)])
def test_values_that_are_not_finite_among_many_rows(hip, kind, hd, H):
    """Where a row looks they reach it; on other pages, behind its position and behind the sequence they reach nothing."""
    rng = np.random.default_rng(hd + H)
    c = Case(rng, kind, hd, 2, 16, [2100], [2150])
    at = c.table[0]
    if kind == "int8":
        c.sk[at[3]], c.sv[at[3]] = np.nan, np.inf
        c.sv[at[20], :, 5] = np.nan
        c.sk[at[134], :, 6:], c.sv[at[134], :, 6:] = np.inf, np.nan
    else:
        c.k[at[3]], c.v[at[3]] = np.nan, np.inf
        c.v[at[20], :, 5, 7] = np.inf
        c.k[at[134], :, 6:], c.v[at[134], :, 6:] = np.inf, np.nan
    c.device()
    q = rng.standard_normal((2100, H, hd)).astype(np.float16)
    last = (50 + np.arange(2100)) // 16
    sel = np.stack([last - 1, np.where(np.arange(2100) % 5 == 0, 20, 21), last, np.full(2100, -1)], -1)[:, None].repeat(2, 1).astype(np.int32)
    sel[sel == 3] = 4
    out = run_attend(hip, c, q, H, sel)
    keys = sel * 16 + 5
    hit = ((sel == 20) & (keys <= (50 + np.arange(2100))[:, None, None])).any(-1).repeat(H // 2, 1)          # rows and heads that see it
    assert 100 < hit[:, 0].sum() < 600
    if kind == "int8":
        assert np.isnan(out[hit]).all()
    else:
        assert np.all(np.isposinf(out[hit][:, 7])) and np.isfinite(np.delete(out[hit], 7, -1)).all()
    exact, tol = ref.attention(c, q, H, sel)
    assert np.all(np.abs(out[~hit].astype(np.float64) - exact[~hit]) <= tol[~hit])
    sel[9, 0, 0] = 3                                          # keys that are not numbers
    again = run_attend(hip, c, q, H, sel)
    assert np.isnan(again[9, :H // 2]).all() and np.array_equal(np.delete(again, 9, 0), np.delete(out, 9, 0), equal_nan=True) and np.array_equal(again[9, H // 2:], out[9, H // 2:])


def test_a_large_score_among_many_rows(hip):
    """Scores far apart and far from zero: weights of one key alone, keys that count for nothing, all of it at any place of the list."""
    rng = np.random.default_rng(13)
    c = Case(rng, "float16", 64, 2, 16, [2048], [2048])
    c.k[c.table[0, ::7]] *= np.float16(60)
    c.device()
    q = (rng.standard_normal((2048, 8, 64)) * 30).astype(np.float16)
    sel = rng.integers(-1, 130, (2048, 2, 6)).astype(np.int32)
    out = run_attend(hip, c, q, 8, sel)
    exact, tol = ref.attention(c, q, 8, sel)
    assert np.all(np.abs(out.astype(np.float64) - exact) <= tol)


def test_more_rows_than_positions(hip):
    """A sequence with fewer positions than rows: rows in front of position 0 choose nothing and give zeros."""
    rng = np.random.default_rng(14)
    c = Case(rng, "float16", 64, 2, 16, [2100], [2000]).device()
    codes, scales = arrays(c, rng)
    q = rng.standard_normal((2100, 8, 64)).astype(np.float16)
    sel = run_choose(hip, c, q, 8, codes, scales, 1, 1, 5)
    assert np.array_equal(sel, ref.choose_many(c, q, 8, codes, scales, 1, 1, 5, np.full(sel.shape, 77, np.int32))) and np.all(sel[:100] == -1)
    out = run_attend(hip, c, q, 8, sel)
    exact, tol = ref.attention(c, q, 8, sel, 3)
    assert np.all(out[:100] == 0) and np.all(np.abs(out[::3].astype(np.float64) - exact[::3]) <= tol[::3])


@pytest.mark.parametrize("hd,H,width", [(128, 4, 32768), (128, 20, 32768), (128, 4, 16385), (128, 4, 16384), (64, 4, 16400)])
def test_the_widest_tables(hip, hd, H, width):
    """As many columns as a choice takes, and those at which a block has fewer rows and wavefronts; pages come again and again, ties go to the lower column."""
    rng = np.random.default_rng(width + H)
    for rows in (1, 3):
        c = Case(rng, "int8", hd, 1, 16, [rows], [1000])
        c.table = np.resize(c.table[0, :62], width).astype(np.int32)[None]
        c.lens = [width * 16 - 5]
        c.device()
        codes, scales = arrays(c, rng)
        q = rng.standard_normal((rows, H, hd)).astype(np.float16)
        for top in (5, 1024):
            sel = run_choose(hip, c, q, H, codes, scales, 2, 3, top)
            assert np.array_equal(sel, ref.choose_many(c, q, H, codes, scales, 2, 3, top, np.full(sel.shape, 77, np.int32)))
