"""The paged cache without a GPU: arguments that are refused, the descriptor's layout, the bookkeeping of pages."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.ffi import check
from denograd_amd.paged import PagedCache, PageTable

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
cpu_only = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="the addresses are made up")
A = 1 << 20     # some 16-byte aligned address


def desc(**more):
    d = dict(kind=ffi.W_I8, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, table_width=3, pages_k=A, pages_v=A, scales_k=A, scales_v=A, page_table=A)
    d.update(more)
    return ffi.PagesDesc(*[d[n] for n, _ in ffi.PagesDesc._fields_])


def write(d, starts=A, lens=A, n=1, rows=1, q=A, k=A, v=A, rope=A, rope_rows=48, q_out=A, heads=4):
    check(ffi.load().jsgrad_hip_paged_write(d, starts, lens, n, rows, q, k, v, rope, rope_rows, q_out, heads))


def read(d, starts=A, lens=A, n=1, rows=1, k=A, v=A):
    check(ffi.load().jsgrad_hip_paged_read(d, starts, lens, n, rows, k, v))


def attend(d, starts=A, lens=A, n=1, rows=1, q=A, out=2 * A, heads=4, window=0, sinks=0, ws=A):
    check(ffi.load().jsgrad_hip_attn_paged(d, starts, lens, n, rows, q, out, heads, window, sinks, ws))


BAD_PAGES = [(dict(kind=ffi.W_NF4), "kind 3"), (dict(kind=ffi.W_F32), "kind 0"), (dict(head_dim=96), "head_dim 96"), (dict(page_size=8), "page_size 8"), (dict(page_size=48), "page_size 48"),
             (dict(page_size=512), "page_size 512"), (dict(page_size=0), "page_size 0"), (dict(page_size=-16), "page_size -16"), (dict(n_pages=0), "n_pages 0"), (dict(n_kv_heads=0), "n_kv_heads 0"),
             (dict(table_width=0), "table_width 0"), (dict(table_width=(1 << 26) + 1), "table_width"), (dict(pages_k=None), "null pointer"), (dict(page_table=None), "null pointer"),
             (dict(scales_v=None), "without scales"), (dict(pages_v=A + 8), "16-byte aligned"), (dict(scales_k=A + 4), "16-byte aligned"), (dict(page_table=A + 2), "4-byte aligned")]
BAD_BATCH = [(dict(starts=None), "null pointer"), (dict(lens=None), "null pointer"), (dict(n=0), "0 sequences"), (dict(n=65536), "65536 sequences"), (dict(rows=0), "0 rows"),
             (dict(rows=-3), "-3 rows"), (dict(starts=A + 1), "4-byte aligned"), (dict(rows=(1 << 24) + 1), "rows")]


@cpu_only
@pytest.mark.parametrize("call", [write, read, attend])
def test_every_call_refuses_bad_pages_and_batches(call):
    for more, says in BAD_PAGES:
        with pytest.raises(ffi.HipError, match=says):
            call(desc(**more))
    for more, says in BAD_BATCH:
        with pytest.raises(ffi.HipError, match=says):
            call(desc(), **more)
    with pytest.raises(ffi.HipError, match="null pointer"):
        call(None)
    # nothing is wrong with these, so that the next question is for a device
    for fine in (desc(), desc(kind=ffi.W_F16, scales_k=None, scales_v=None), desc(head_dim=128, page_size=256, table_width=1)):
        with pytest.raises(ffi.HipError, match="jsgrad_hip_init has not been called"):
            call(fine, **(dict(rope_rows=256) if call is write else {}))


@cpu_only
def test_what_each_call_refuses_of_its_own():
    for more, says in ((dict(k=None), "null"), (dict(v=None), "null"), (dict(q=None), "go together"), (dict(q_out=None), "go together"), (dict(heads=0), "n_heads 0"),
                       (dict(k=A + 2), "aligned"), (dict(rope=A + 8), "aligned"), (dict(rope_rows=47), "rope table of 47 positions, the page table has 48")):
        with pytest.raises(ffi.HipError, match=says):
            write(desc(), **more)
    for more, says in ((dict(k=None), "null"), (dict(v=A + 4), "aligned")):
        with pytest.raises(ffi.HipError, match=says):
            read(desc(), **more)
    for more, says in ((dict(q=None), "null"), (dict(out=None), "null"), (dict(ws=None), "null"), (dict(out=A), "must not be q"), (dict(heads=3), "n_heads 3"), (dict(heads=0), "n_heads 0"),
                       (dict(window=-1), "window -1"), (dict(sinks=-1), "sinks -1"), (dict(q=A + 8), "aligned"), (dict(ws=A + 8), "aligned")):
        with pytest.raises(ffi.HipError, match=says):
            attend(desc(), **more)


@cpu_only
def test_more_rows_than_a_launch_has_blocks_are_refused():
    """A grid's threads are counted in 32 bits, 256 to a block: fewer than 2^24 blocks."""
    for call in (write, read, attend):
        with pytest.raises(ffi.HipError, match="16777216 rows"):
            call(desc(), rows=1 << 24)
        with pytest.raises(ffi.HipError, match="jsgrad_hip_init has not been called"):
            call(desc(), rows=(1 << 24) - 1)
    # 2^25 pairs of each of 64 kv heads in q tiles of 128: 2^24 blocks, and those of the parts
    with pytest.raises(ffi.HipError, match="2097152 rows of 1024 heads"):
        attend(desc(n_kv_heads=64), rows=1 << 21, heads=1024)


def test_descriptor_layout(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "jsgrad_hip.h"\nint main(void){printf("%zu %zu %zu", sizeof(jsgrad_hip_pages_t), offsetof(jsgrad_hip_pages_t, pages_k),'
                   'offsetof(jsgrad_hip_pages_t, page_table));return 0;}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(ffi.PagesDesc), ffi.PagesDesc.pages_k.offset, ffi.PagesDesc.page_table.offset] == [64, 24, 56]
    assert int(re.search(r"PAGES_BYTES = (\d+)", open(os.path.join(ROOT, "integration", "jsgrad", "runtime", "hip_bindings.ts")).read()).group(1)) == 64


def test_page_table_keeps_every_page_once():
    rng = np.random.default_rng(0)
    t, seqs = PageTable(50, 16), []

    def all_pages():
        return sorted(t.free + [p for v in t.pages.values() for p in v if p >= 0])

    for _ in range(300):
        op = rng.integers(0, 4)
        if op == 0 or not seqs:
            seqs.append(t.add())
        elif op == 1 and len(seqs) > 2:
            t.drop(seqs.pop(int(rng.integers(len(seqs)))))
        elif op == 2:
            some = list(rng.choice(seqs, size=min(len(seqs), 2), replace=False))
            counts = rng.integers(0, 60, len(some))
            before = {s: (t.lengths[s], len(t.pages[s])) for s in seqs}
            try:
                t.grow(some, counts)
                assert all(t.lengths[s] == before[s][0] + c and len(t.pages[s]) == -(-t.lengths[s] // 16) for s, c in zip(some, counts))
            except MemoryError:
                assert {s: (t.lengths[s], len(t.pages[s])) for s in seqs} == before
        else:
            t.slide(seqs[0], int(rng.integers(1, 40)), int(rng.integers(0, 30)))
        assert all_pages() == list(range(50))


def test_slide_keeps_what_the_next_row_sees_and_gives_the_rest():
    for page in (16, 32):
        for length in (1, 15, 16, 17, 64, 100):
            for window in (1, 2, 16, 17, 50, 200):
                for sinks in (0, 1, 16, 20):
                    t = PageTable(20, page)
                    s = t.add()
                    t.grow([s], [length])
                    n = t.slide(s, window, sinks)
                    held = {j // page for j in range(length) if j > length - window or j < sinks}
                    gone = {i for i, p in enumerate(t.pages[s]) if p < 0}
                    assert n == len(gone) and not gone & held
                    whole = {i for i in range(len(t.pages[s])) if (i + 1) * page <= length}
                    assert gone == whole - held - {i for i in whole if i * page < sinks}
                    assert t.slide(s, window, sinks) == 0


def test_page_table_refuses():
    for args in ((0, 16), (4, 8), (4, 24), (4, 512)):
        with pytest.raises(ValueError):
            PageTable(*args)
    t = PageTable(4, 16)
    s = t.add()
    for seqs, counts in (([s, s], [1, 1]), ([s], [-1]), ([s], [1, 2])):
        with pytest.raises(ValueError):
            t.grow(seqs, counts)
    with pytest.raises(ValueError):
        t.slide(s, 0)
    with pytest.raises(MemoryError, match="5 pages are needed and 4 of 4 are free"):
        t.grow([s], [65])


def test_paged_cache_refuses():
    for args in ((1, 2, 96, 4), (1, 2, 64, 0), (0, 2, 64, 4), (1, 0, 64, 4), (1, 1025, 64, 4), (1, 2, 64, 4, 24), (1, 2, 64, 4, 16, "float32")):
        with pytest.raises(ValueError):
            PagedCache(*args)
    cache = PagedCache.__new__(PagedCache)                # the bookkeeping alone: these come before anything on a device
    PageTable.__init__(cache, 4, 16)
    s = cache.add()
    for seqs, counts in (([], []), ([s], [0]), ([s], [1 << 24]), ([s] * 65536, [1] * 65536), ([s], [1, 1]), ([s, s], [1, 1])):
        with pytest.raises(ValueError):
            cache.begin(seqs, counts)
    assert cache.lengths[s] == 0 and len(cache.free) == 4
