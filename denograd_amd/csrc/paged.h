// Where things are in a paged KV cache and a ragged batch: what the kernels of paged.hip and paged_attn.hip go by, in plain C++ so that
// a host compiler takes it too (tests/test_paged_plan.py walks it over batches and tables with anything in them).
//
// row_starts, lengths and page_table are device memory that the host does not look at.  Whatever they hold, no address outside the buffers is made
// of it: first rows are brought into [0, rows], lengths into [0, 2^30], and a position whose table entry is no page of the pool, or that
// lies behind the table, has no page: nothing is written there and no query sees it.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define JSG_BOTH __host__ __device__ __forceinline__
#else
#define JSG_BOTH inline
#endif

namespace jsg {

struct PagedBatch {
  const int32_t *row_starts, *lengths;   // [n_seqs + 1], [n_seqs]
  const int32_t *table;                  // [n_seqs][width]
  int n_seqs, rows, width, n_pages, page_shift;
};
struct PagedSeq {
  int start, n, len;                     // first row of the batch, new rows, positions with them
};
JSG_BOTH int paged_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
JSG_BOTH PagedSeq paged_seq(int start, int end, int len, int rows) {
  PagedSeq s;
  s.start = paged_clamp(start, 0, rows);
  s.n = paged_clamp(end, s.start, rows) - s.start;
  s.len = paged_clamp(len, 0, 1 << 30);  // no table has more positions
  return s;
}
// Whether first rows fall here.  Where they do not, the sequences share the rows out among them, and a grid made for `rows` rows has blocks for all.
JSG_BOTH bool paged_falls(const PagedBatch &p, int b) { return paged_clamp(p.row_starts[b + 1], 0, p.rows) < paged_clamp(p.row_starts[b], 0, p.rows); }
JSG_BOTH PagedSeq paged_seq(const PagedBatch &p, int b) { return paged_seq(p.row_starts[b], p.row_starts[b + 1], p.lengths[b], p.rows); }
// position of row i of a sequence: below zero where there are more new rows than positions
JSG_BOTH int paged_pos(const PagedSeq &s, int i) { return s.len - s.n + i; }
JSG_BOTH int paged_room(const PagedBatch &p) { return p.width << p.page_shift; }
// the page that holds a position, or -1
JSG_BOTH int paged_page(const PagedBatch &p, int b, int pos) {
  if (pos < 0 || pos >= paged_room(p)) return -1;
  const int id = p.table[(size_t)b * p.width + (pos >> p.page_shift)];
  return id >= 0 && id < p.n_pages ? id : -1;
}
// row of pages_k / pages_v ([n_pages][n_kv_heads][page_size] rows of head_dim) of a position on that page; scales have one value per row
JSG_BOTH size_t paged_row(const PagedBatch &p, int n_kv_heads, int id, int g, int pos) {
  return (((size_t)id * n_kv_heads + g) << p.page_shift) + (size_t)(pos & ((1 << p.page_shift) - 1));
}

constexpr int PAGED_GRID = 1 << 24;      // a launch has fewer blocks of 256 threads: it counts its threads in 32 bits

// ---- the work of an attention launch
constexpr int PAGED_KEYS = 64;           // keys of a tile
// Key tiles that rows at positions p_lo .. p_hi look at: [0, n_sink), then from t_lo on, n in all.
struct PagedKeys {
  int n_sink, t_lo, n;
  JSG_BOTH int tile(int i) const { return i < n_sink ? i : t_lo + (i - n_sink); }
};
JSG_BOTH PagedKeys paged_keys(int p_lo, int p_hi, int room, int window, int sinks) {
  PagedKeys k = {0, 0, 0};
  const int hi = p_hi < room ? p_hi : room - 1, t_end = hi < 0 ? 0 : hi / PAGED_KEYS + 1;
  if (window > 0 && p_lo >= window) k.t_lo = (p_lo - window + 1) / PAGED_KEYS;
  if (window > 0 && sinks > 0) k.n_sink = paged_clamp((sinks - 1) / PAGED_KEYS + 1, 0, k.t_lo < t_end ? k.t_lo : t_end);
  k.n = k.n_sink + (t_end > k.t_lo ? t_end - k.t_lo : 0);
  return k;
}
// A sequence's share of a launch with blocks of q_rows (row, query head) pairs, the heads of a kv head side by side: q tiles, and the key tiles of the last one.
struct PagedShare {
  int q_tiles, key_tiles;
};
// rows * n_rep is below 2^30; div: x / n_rep
template <typename Div> JSG_BOTH PagedShare paged_share(const PagedSeq &s, int n_rep, Div div, int q_rows, int room, int window, int sinks) {
  PagedShare h;
  h.q_tiles = (s.n * n_rep + q_rows - 1) / q_rows;
  h.key_tiles = s.n > 0 ? paged_keys(paged_pos(s, div((h.q_tiles - 1) * q_rows)), paged_pos(s, s.n - 1), room, window, sinks).n : 0;
  return h;
}
// q tiles per kv head that a batch of `rows` rows of `seqs` sequences has at most, however the rows are dealt out: of q_rows pairs, or of `least` where a sequence has no more than `few` of those.
JSG_BOTH size_t paged_most_tiles(int rows, int n_rep, int seqs, int q_rows, int least, int few) {
  const size_t by_pairs = (size_t)rows * n_rep / q_rows + (size_t)few * seqs, by_rows = (size_t)rows * ((n_rep + least - 1) / least);
  return by_pairs < by_rows ? by_pairs : by_rows;
}
// Whether no such batch has a sequence of more than most_pairs pairs, or more than `little` pairs of a q tile and a key tile of all heads: few_items q tiles over room_tiles key tiles.
JSG_BOTH bool paged_few_only(int rows, int n_rep, int most_pairs, size_t few_items, int room_tiles, float little) {
  return (size_t)rows * n_rep <= (size_t)most_pairs || (double)few_items * room_tiles <= little;
}
// Key tiles of a part where `blocks` parts have the same share of the launch's pairs of a q tile and a key tile.  An item of key_tiles > target, for a target of that and more,
// is cut into ceil(key_tiles / target) parts, one more at most, or fewer; the parts of cut items are no more than 2 * blocks, as each has half a target's pairs at least.
JSG_BOTH int paged_target(float pairs, int blocks, int least) {
  const float t = pairs * (1.002f / (float)blocks);            // a little more than the share, for the rounding here and in the next
  return t < (float)least ? least : t < 1e9f ? (int)t + 1 : 1000000000;
}
// inv: 1.0f / target
JSG_BOTH int paged_parts(int key_tiles, int target, float inv, int most) {
  const int n = key_tiles <= target ? 1 : (int)((float)(key_tiles - 1) * inv + 1e-3f) + 1;
  return n > most ? (most < 1 ? 1 : most) : n;
}
// No more blocks than this: an item's parts are one and less than one more for every target of its key tiles; the rest is for the rounding, there and here.
JSG_BOTH float paged_most_blocks(float pairs, float items, float inv) { return 1.01f * (items + pairs * inv) + 8.0f; }

}  // namespace jsg
