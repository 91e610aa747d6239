// Where things are in a paged KV cache and a ragged batch: what the kernels of paged.hip and paged_attn.hip go by, in plain C++ so that
// a host compiler takes it too (tests/test_paged_plan.py walks it over batches and tables with anything in them).
//
// row_starts, lengths and page_table are device memory that the host does not look at.  Whatever they hold, no address outside the buffers is made
// of it: first rows are brought into [0, rows], a negative length counts as zero, and a position whose table entry is no page of the pool, or that
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
  s.len = len < 0 ? 0 : len;
  return s;
}
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

}  // namespace jsg
