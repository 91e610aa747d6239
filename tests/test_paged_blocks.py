"""What an attention launch over the paged cache says of its batch without looking at it (denograd_amd/csrc/paged.h, compiled for the host): however the rows are dealt out to the
sequences, there are blocks for all, those that nothing is left for know it, and the few-row kernel is launched only where no sequence has many rows or the work is little."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r'''
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "paged.h"
using namespace jsg;
static uint64_t state = 88172645463325252ull;
static int range(int lo, int hi) { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return lo + (int)(state % (uint64_t)(hi - lo + 1)); }
#define CHECK(x) do { if (!(x)) { printf("round %d: %s\n", round, #x); return 1; } } while (0)

int main() {
  int only = 0, cut = 0;
  for (int round = 0; round < 20000; round++) {
    const int seqs = range(1, round % 3 ? 8 : 300), n_rep = range(0, 1) ? 1 << range(0, 5) : range(1, 40), KV = range(1, 8), rows = range(1, round % 5 ? 40 : 2000);
    const int shift = range(4, 8), width = range(1, range(0, 1) ? 12 : 2000), room = width << shift, least_part = range(1, 4);
    // rows in one sequence, one in each, or anyhow; the sequences have no more than `rows`, the others none
    std::vector<int> n(seqs, 0);
    const int how = range(0, 2);
    int used = how == 0 ? range(1, rows) : 0;
    if (how == 0) n[range(0, seqs - 1)] = used;
    else if (how == 1) for (int b = 0; b < seqs && used < rows; b++, used++) n[b] = 1;
    else while (used < rows && range(0, 50)) { const int m = range(1, rows - used < 30 ? rows - used : 30); n[range(0, seqs - 1)] += m; used += m; }
    const int most_seqs = seqs < rows ? seqs : rows, room_tiles = (room + PAGED_KEYS - 1) / PAGED_KEYS;
    const size_t few_items = KV * paged_most_tiles(rows, n_rep, most_seqs, PF_QROWS, PF_QROWS, 1), items = KV * paged_most_tiles(rows, n_rep, most_seqs, PC_QROWS, PF_QROWS, PF_PAIRS / PF_QROWS);
    const float little = range(0, 1) ? 6100.0f : 12288.0f;
    size_t few_tiles = 0, tiles = 0;
    float pairs = 0, all = 0;
    bool many = false;
    std::vector<PagedShare> shares;
    for (int b = 0; b < seqs; b++) {
      PagedSeq s = {0, n[b], range(n[b] < room ? n[b] : room, room)};
      auto div = [&](int x) { return x / n_rep; };
      const PagedShare f = paged_share(s, n_rep, div, PF_QROWS, room, 0, 0), c = paged_share(s, n_rep, div, PC_QROWS, room, 0, 0);
      few_tiles += f.q_tiles;
      pairs += (float)f.q_tiles * f.key_tiles * KV;
      all += (float)f.q_tiles * KV;
      shares.push_back(f);
      const bool small = n[b] * n_rep <= PF_PAIRS;
      many |= !small;
      tiles += small ? f.q_tiles : c.q_tiles;
    }
    CHECK(KV * few_tiles <= few_items);
    CHECK(KV * tiles <= items);
    if (paged_few_only(rows, n_rep, PF_PAIRS, few_items, room_tiles, little)) {
      only++;
      CHECK(!many || pairs <= little);
    }
    const int target = paged_target(pairs, 512, least_part) * range(8, 16) / 8;
    size_t blocks = 0;
    for (auto &h : shares) {
      const int parts = paged_parts(h.key_tiles, target, 1.0f / (float)target, range(0, 1) ? 64 : 1 << 20);
      blocks += (size_t)KV * h.q_tiles * parts;
      cut += parts > 1;
    }
    CHECK((float)blocks <= paged_most_blocks(pairs, all, 1.0f / (float)target));
  }
  return only > 500 && cut > 500 ? 0 : 2;
}
'''


def test_blocks_and_kernels_of_any_batch(tmp_path):
    text = open(os.path.join(ROOT, "denograd_amd", "csrc", "paged_attn.hip")).read()
    consts = "\n".join(f"#define {n} {v}" for n, v in re.findall(r"\b(P[CF]_QROWS|PF_PAIRS) = (\d+)", text))
    assert consts.count("#define") == 3
    src = tmp_path / "blocks.cpp"
    src.write_text(consts + SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "denograd_amd", "csrc"), str(src), "-o", str(tmp_path / "blocks")], check=True)
    r = subprocess.run([str(tmp_path / "blocks")], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout[-500:], r.stderr[-2000:])
