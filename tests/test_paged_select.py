"""Refusals of the calls on chosen pages; without a GPU."""
import numpy as np
import pytest

from denograd_amd import ffi

BASE = dict(kind=ffi.W_F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, table_width=8, pages_k=4096, pages_v=4096, scales_k=None, scales_v=None, page_table=4096)


def refused(call, args, change, match):
    desc = {k: change.get(k, v) for k, v in BASE.items()}
    args = {k: change.get(k, v) for k, v in args.items()}
    lib = ffi.load()
    assert getattr(lib, call)(ffi.PagesDesc(*desc.values()), 4096, 4096, change.get("n_seqs", 1), change.get("rows", 1), *args.values()) != 0
    text = lib.jsgrad_hip_last_error().decode()
    assert match in text and call in text


@pytest.mark.parametrize("change,match", [(dict(bounds=None), "null"), (dict(scales=None), "null"), (dict(bounds=4104), "aligned"), (dict(scales=4098), "aligned"), (dict(page_size=24), "page_size"),
                                          (dict(head_dim=96), "head_dim"), (dict(rows=0), "rows"), (dict(pages_k=None), "null")])
def test_bounds(change, match):
    refused("jsgrad_hip_paged_bounds", dict(bounds=4096, scales=4096), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(q=None), "null"), (dict(q=4104), "aligned"), (dict(n_heads=3), "n_heads"), (dict(n_heads=0), "n_heads"), (dict(n_heads=130), "at most 64"), (dict(bounds=None), "null"), (dict(scales=4097), "aligned"),
    (dict(first=-1), "first"), (dict(recent=0), "recent"), (dict(top=0), "pages"), (dict(top=1025), "pages"), (dict(first=3, recent=2), "first 3"), (dict(first=0x7fffffff), "first"),
    (dict(recent=0x7fffffff), "recent"), (dict(selected=None), "selected"), (dict(selected=4098), "selected"), (dict(table_width=32769), "table_width"), (dict(rows=1 << 24), "rows"),
    (dict(rows=(1 << 24) - 1, n_heads=128), "rows"),
])
def test_choice(change, match):
    refused("jsgrad_hip_paged_select", dict(q=4096, n_heads=4, bounds=4096, scales=4096, first=1, recent=1, top=4, selected=4096), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(selected=None), "null"), (dict(workspace=None), "null"), (dict(out=8200), "aligned"), (dict(workspace=4104), "aligned"), (dict(selected=4098), "aligned"),
    (dict(out=4096), "out must not be q"), (dict(n_heads=5), "n_heads"), (dict(top=0), "pages"), (dict(top=1025), "pages"), (dict(rows=(1 << 24) - 1, n_heads=62), "rows"),
])
def test_attention(change, match):
    refused("jsgrad_hip_attn_selected", dict(q=4096, out=8192, n_heads=4, selected=4096, top=4, workspace=4096), change, match)


def test_references_against_each_other():
    """The reference's unit of bounds: halves and powers of two land where 127 times it just holds them."""
    from tests.select_ref import step
    for most, want in ((127.0, 1.0), (127.0625, 2.0), (128.0, 2.0), (63.5, 0.5), (0.0, 1.0), (6e-8, 2.0 ** -30), (65504.0, 1024.0), (1e-42, 2.0 ** -126)):
        assert step(most) == want
        assert most == 0 or want == 2.0 ** -126 or np.float64(127) * want >= most > 127 * want / 2


def test_the_choice_for_many_rows_at_once():
    from tests import select_ref as ref
    from tests.paged_ref import Case
    rng = np.random.default_rng(0)
    c = Case(rng, "float16", 64, 2, 16, [60, 0, 7], [300, 5, 7])
    c.table[0, 4] = -1
    codes, scales = ref.bounds(c, np.zeros((c.n_pages, 2, 2, 64), np.int8), np.ones((c.n_pages, 2), np.float32))
    scales[c.table[0, 16]] = np.inf
    q = rng.standard_normal((67, 8, 64)).astype(np.float16)
    q[3, 2, 1], q[4] = np.nan, 0
    for top in (3, 30):
        before = np.full((67, 2, top), 77, np.int32)
        assert np.array_equal(ref.choose(c, q, 8, codes, scales, 1, 2, top, before), ref.choose_many(c, q, 8, codes, scales, 1, 2, top, before))
