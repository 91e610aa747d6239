"""What the kernels of the paged cache go by (denograd_amd/csrc/paged.h), compiled for the host: whatever row starts, lengths and page tables hold, no index
leaves its buffer, every visible key is in one part of its q tile's tiles, and the parts of a launch fit the workspace and the grid."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r'''
#include <assert.h>
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "paged.h"
using namespace jsg;
static uint64_t state = 88172645463325252ull;
static uint64_t rnd() { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return state; }
static int range(int lo, int hi) { return lo + (int)(rnd() % (uint64_t)((int64_t)hi - lo + 1)); }
static int any() { switch (range(0, 5)) { case 0: return (int)rnd(); case 1: return range(-5, 5); case 2: return 0x7fffffff; case 3: return (int)0x80000000; default: return range(0, 3000); } }

int main() {
  long rows_seen = 0, cut_items = 0;
  for (int round = 0; round < 3000; round++) {
    const bool sane = round % 3 != 0;
    PagedBatch p;
    p.page_shift = range(4, 8);
    p.width = range(1, range(0, 9) ? 12 : 3000);
    p.n_seqs = range(1, range(0, 3) ? 5 : 200);
    p.n_pages = range(1, 50);
    const int room = paged_room(p);
    std::vector<int32_t> starts(p.n_seqs + 1), lens(p.n_seqs), table((size_t)p.n_seqs * p.width);
    int at = 0;
    for (int b = 0; b < p.n_seqs; b++) {
      starts[b] = at;
      const int len = range(0, room), n = range(0, range(0, 2) ? 3 : len < 300 ? len : 300);
      at += n;
      lens[b] = len > n ? len : n;
    }
    starts[p.n_seqs] = at;
    p.rows = at + range(0, 2) > 0 ? at + range(0, 2) : 1;
    if (p.rows < 1) p.rows = 1;
    if (!sane) {
      for (auto &x : starts) if (range(0, 1)) x = any();
      for (auto &x : lens) if (range(0, 1)) x = any();
    }
    for (auto &x : table) x = range(0, 3) ? range(0, p.n_pages - 1) : any();
    p.row_starts = starts.data(); p.lengths = lens.data(); p.table = table.data();
    const int n_rep = range(1, 9), KV = range(1, 9), window = range(0, 1) ? 0 : range(1, range(0, 1) ? 200 : 1 << 30), sinks = range(0, 1) ? 0 : range(1, range(0, 4) ? 200 : 1 << 30);
    struct Shape { int q_rows, blocks, least; } shapes[] = {SHAPES};
    for (Shape sh : shapes) {
      auto div = [&](int x) { return x / n_rep; };
      float pairs = 0;
      int longest = 0;
      for (int b = 0; b < p.n_seqs; b++) {
        const PagedSeq s = paged_seq(p, b);
        assert(s.start >= 0 && s.n >= 0 && s.start + s.n <= p.rows && s.len >= 0);
        const PagedShare h = paged_share(s, n_rep, div, sh.q_rows, room, window, sinks);
        assert((int64_t)h.q_tiles * sh.q_rows >= (int64_t)s.n * n_rep && (s.n > 0) == (h.q_tiles > 0));
        pairs += (float)h.q_tiles * (float)h.key_tiles;
        if (h.key_tiles > longest) longest = h.key_tiles;
      }
      const int target = paged_target(pairs * (float)KV, sh.blocks, sh.least) * range(8, 16) / 8;
      int64_t slots = 0, blocks = 0;
      for (int b = 0; b < p.n_seqs; b++) {
        const PagedSeq s = paged_seq(p, b);
        const PagedShare h = paged_share(s, n_rep, div, sh.q_rows, room, window, sinks);
        const int parts = paged_parts(h.key_tiles, target, 1.0f / (float)target, (int)sqrtf((float)h.key_tiles) * (round % 2 ? 1 : 100));
        assert(parts >= 1 && (parts == 1 || h.key_tiles > target) && parts <= (h.key_tiles - 1) / target + 2);
        blocks += (int64_t)KV * h.q_tiles * parts;
        if (parts > 1) slots += (int64_t)KV * h.q_tiles * parts, cut_items++;
        assert(parts == 1 || (room + PAGED_KEYS - 1) / PAGED_KEYS > sh.least);
        const int n_rows = s.n * n_rep, p0 = paged_pos(s, 0);
        for (int qt = 0; qt < h.q_tiles; qt++) {
          if (qt > 2 && qt < h.q_tiles - 2) continue;
          const int q0 = qt * sh.q_rows, q1 = q0 + sh.q_rows < n_rows ? q0 + sh.q_rows : n_rows;
          const PagedKeys k = paged_keys(p0 + div(q0), p0 + div(q1 - 1), room, window, sinks);
          assert(k.n >= 0 && (k.n <= h.key_tiles || window));
          int last = -1;
          for (int i = 0; i < k.n; i++) {
            if (i > 5 && i < k.n - 5 && k.n > 100) { last = k.tile(i); continue; }
            const int t = k.tile(i);
            assert(t > last && t >= 0 && (int64_t)t * PAGED_KEYS < room);
            last = t;
            for (int pos = t * PAGED_KEYS; pos < (t + 1) * PAGED_KEYS; pos += 16) {
              const int id = paged_page(p, b, pos);
              assert(id >= -1 && id < p.n_pages);
              const size_t row = paged_row(p, KV, id < 0 ? 0 : id, KV - 1, pos), all = (size_t)p.n_pages * KV << p.page_shift;
              assert(row + 16 <= all);
            }
          }
          // every key that a row sees is in a tile
          for (int i = 0; i < 6; i++) {
            const int r = range(q0, q1 - 1), pos = p0 + div(r);
            if (pos < 0) continue;
            rows_seen++;
            for (int j = 0; j < 40; j++) {
              const int key = j < 20 ? pos - j * j : range(0, pos);
              if (key < 0 || key >= room || !(window == 0 || key > pos - window || key < sinks)) continue;
              bool in = key / PAGED_KEYS < k.n_sink || (key / PAGED_KEYS >= k.t_lo && key / PAGED_KEYS < k.t_lo + k.n - k.n_sink);
              assert(in);
            }
          }
        }
      }
      assert(slots <= 2 * sh.blocks);
      if (sane) assert(blocks <= (int64_t)KV * ((int64_t)p.rows * n_rep / sh.q_rows + (p.n_seqs < p.rows ? p.n_seqs : p.rows)) + (longest > sh.least ? 2 * sh.blocks : 0));
    }
  }
  printf("%ld %ld", rows_seen, cut_items);
  return 0;
}
'''


def test_indices_and_shares_of_any_batch(tmp_path):
    import re
    text = open(os.path.join(ROOT, "denograd_amd", "csrc", "paged_attn.hip")).read()
    shapes = re.findall(r"constexpr int \w+_THREADS = \d+, \w+_QROWS = (\d+);\nconstexpr int \w+_BLOCKS = (\d+), \w+_LEAST = (\d+);", text)
    assert shapes
    src = tmp_path / "plan.cpp"
    src.write_text(SOURCE.replace("SHAPES", ", ".join("{%s, %s, %s}" % s for s in shapes)))
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "denograd_amd", "csrc"), str(src), "-o", str(tmp_path / "plan")], check=True)
    r = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    rows_seen, cut = (int(v) for v in r.stdout.split())
    assert rows_seen > 100000 and cut > 1000


FALLS = r'''
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "paged.h"
using namespace jsg;
int main() {
  srand(1);
  int fell = 0;
  for (int round = 0; round < 20000; round++) {
    PagedBatch p = {};
    p.n_seqs = rand() % 9 + 1;
    p.rows = rand() % 20 + 1;
    std::vector<int32_t> starts(p.n_seqs + 1), lens(p.n_seqs, 5);
    for (int b = 0; b <= p.n_seqs; b++) starts[b] = rand() % 3 ? (b ? starts[b - 1] : 0) + rand() % 4 : rand() % 6 == 0 ? (int32_t)((uint32_t)rand() * 2u) : rand() % 30;
    p.row_starts = starts.data(); p.lengths = lens.data();
    long all = 0;
    bool falls = false;
    for (int b = 0; b < p.n_seqs; b++) {
      all += paged_seq(p, b).n;
      falls |= paged_falls(p, b);
      if (paged_falls(p, b) && starts[b + 1] >= starts[b]) return 1;
    }
    if (!falls && all > p.rows) return 2;
    fell += falls;
  }
  return fell > 1000 && fell < 19000 ? 0 : 3;
}
'''


def test_rows_are_shared_out_where_row_starts_do_not_fall(tmp_path):
    """Which the grid of an attention launch rests on; a batch whose first rows fall is not worked on."""
    src = tmp_path / "falls.cpp"
    src.write_text(FALLS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "denograd_amd", "csrc"), str(src), "-o", str(tmp_path / "falls")], check=True)
    assert subprocess.run([str(tmp_path / "falls")]).returncode == 0
