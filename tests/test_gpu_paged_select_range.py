"""The choice of pages and their bounds at both ends of the floats: scales of int8 pages may be any finite number, and scores of different pages stay different."""
import numpy as np
import pytest

from tests import select_ref as ref
from tests.paged_ref import Case
from tests.test_gpu_paged_select import run_bounds, run_choose

pytestmark = pytest.mark.gpu

# kv heads, query heads, new rows, lengths: one row to a block, rows side by side, and more than 16 heads to a kv head
FORMS = [(2, 8, [1], [640]), (1, 4, [40], [400]), (1, 40, [2], [300])]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("KV,H,news,lens", FORMS)
@pytest.mark.parametrize("least,most", [(100, 123), (-126, -110), (-126, 123)])
def test_units_of_any_size(hip, hd, KV, H, news, lens, least, most):
    """Bounds as whole numbers up to 127 in units from 2^-126 to 2^122, the largest that a page of finite keys has: the largest scores are past the floats, and all are in their order."""
    rng = np.random.default_rng(hd + H + least + 126)
    c = Case(rng, "int8", hd, KV, 16, news, lens).device()
    box = np.sort(rng.integers(-127, 128, (c.n_pages, c.KV, 2, hd)), 2).astype(np.int8)
    scales = (2.0 ** rng.integers(least, most, (c.n_pages, c.KV))).astype(np.float32)
    q = rng.standard_normal((c.rows, H, hd)).astype(np.float16)
    sel = run_choose(hip, c, q, H, box, scales, 0, 1, 6)
    assert np.array_equal(sel, ref.choose(c, q, H, box, scales, 0, 1, 6, np.full(sel.shape, 77, np.int32)))
    # two pages, the better one behind the other
    c = Case(rng, "int8", hd, 1, 16, [1], [48]).device()
    box, scales = np.full((c.n_pages, 1, 2, hd), 64, np.int8), np.ones((c.n_pages, 1), np.float32)
    for a, b in ((most - 2, most - 1), (least, least + 1)):
        scales[c.table[0, 0]], scales[c.table[0, 1]] = 2.0 ** a, 2.0 ** b
        for x, want in ((1.0, 1), (-1.0, 0)):
            assert run_choose(hip, c, np.full((1, 4, hd), x, np.float16), 4, box, scales, 0, 1, 2).tolist() == [[[want, 2]]]


@pytest.mark.parametrize("hd", [64, 128])
def test_from_keys_to_choices(hip, hd):
    """Keys of int8 pages in units from 2^-140 to 2^120."""
    rng = np.random.default_rng(hd)
    c = Case(rng, "int8", hd, 2, 16, [300], [300])
    c.sk = (2.0 ** np.broadcast_to(rng.integers(-140, 121, (c.n_pages, 1, 1)), c.sk.shape)).astype(np.float32)
    c.device()
    none = np.zeros((c.n_pages, 2, 2, hd), np.int8), np.ones((c.n_pages, 2), np.float32)
    got, want = run_bounds(hip, c, *none), ref.bounds(c, *none)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    q = rng.standard_normal((300, 8, hd)).astype(np.float16)
    sel = run_choose(hip, c, q, 8, *got, 1, 1, 5)
    assert np.array_equal(sel, ref.choose(c, q, 8, *want, 1, 1, 5, np.full(sel.shape, 77, np.int32)))


@pytest.mark.parametrize("hd", [64, 128])
def test_keys_far_apart_on_one_page(hip, hd):
    """A key that is less than the last bit of a float in the page's unit is rounded outwards all the same: to -1 below zero, to 1 above it."""
    rng = np.random.default_rng(hd + 1)
    c = Case(rng, "int8", hd, 2, 16, [160], [160])
    c.sk = (2.0 ** rng.integers(-149, 119, c.sk.shape)).astype(np.float32)
    c.sk[c.table[0, 0], :, 0], c.sk[c.table[0, 0], :, 1:] = 2.0 ** 100, 2.0 ** -140
    c.ck[c.table[0, 0], :, 0, 0], c.ck[c.table[0, 0], :, 1:, 1], c.ck[c.table[0, 0], :, 1:, 2] = 64, 3, -3
    c.ck[c.table[0, 0], :, 0, 1:] = 0
    c.device()
    none = np.zeros((c.n_pages, 2, 2, hd), np.int8), np.ones((c.n_pages, 2), np.float32)
    got, want = run_bounds(hip, c, *none), ref.bounds(c, *none)
    at = c.table[0, 0]
    assert want[0][at, 0, :, 1].tolist() == [0, 1] and want[0][at, 0, :, 2].tolist() == [-1, 0] and want[1][at, 0] == 2.0 ** 100
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
