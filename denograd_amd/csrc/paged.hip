// Rows into and out of a paged KV cache: rotary embedding + write (fp16, or int8 with a float scale per position and head), and the read back.
//
// Reference semantics of what is written: apply_rotary_emb and the cache assign (jsgrad/models/llama.ts:17-32,61-87); the pages,
// their int8 form and ragged batches have no counterpart there.
//
// int8, for the row x of one position and head (keys behind the rotation, in float): scale = max |x| / 127, code = rint(x / scale), so that code * scale is
// within scale / 2 of x.  A row of zeros has scale 1; one with a value that is not finite has scale NaN and reads as NaN.  Scales are float: an
// fp16 one would be off by 2^-11 and would lose rows below 7.6e-6.
#include <type_traits>

#include "gemm.h"
#include "paged.h"

namespace jsg {

constexpr int PR_THREADS = 256, PR_ROWS = 8;

struct PagedArgs {
  PagedBatch pb;
  void *pages[2];                        // k, v
  float *scales[2];
  const _Float16 *x[3];                  // k, v, q rows in
  _Float16 *y[3];                        // k, v, q rows out
  const _Float16 *rope;                  // [positions][HD/2][2] or null
  int n_kv_heads, n_heads;               // n_heads 0: no q
  Divisor pieces;                        // of a row that is read: 8 elements of a head each
};

// Sequence of row r: the first one that ends behind it.  Called by whole wavefronts with a uniform r: 64 first rows at a time.
__device__ __forceinline__ int paged_find(const PagedBatch &pb, int r) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0;; b0 += 64) {
    const int b = b0 + lane;
    const uint64_t behind = __builtin_amdgcn_ballot_w64(b >= pb.n_seqs || pb.row_starts[b + 1] > r);
    if (behind) return b0 + __builtin_ctzll(behind);         // n_seqs: no sequence has the row
  }
}

template <int LANES> __device__ __forceinline__ uint32_t group_max(uint32_t v) {   // over 8 or 16 neighbouring lanes
  auto step = [&](auto c) { const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(c)::value, 0xf, 0xf, true); v = v > o ? v : o; };
  step(std::integral_constant<int, 0xB1>());
  step(std::integral_constant<int, 0x4E>());
  step(std::integral_constant<int, 0x141>());
  if (LANES == 16) step(std::integral_constant<int, 0x140>());
  return v;
}

// Bound by memory: 32768 rows of 32 and 8 heads of 128, fp16 159 us = 5.1 TB/s, int8 170 (the quotients are divided out, so that a code is the nearest one: fp16 rows have many
// that lie in the middle).  One block per row of the batch, a thread per 8 elements of a head: its heads are n_kv_heads of k, as many of v, then n_heads of q.
template <int HD, bool I8> __global__ __launch_bounds__(PR_THREADS) void paged_write_kernel(PagedArgs a) {
  constexpr int G = HD / 8;
  const int r = blockIdx.x, KV = a.n_kv_heads, heads = 2 * KV + a.n_heads;
  const int b = paged_find(a.pb, r);
  if (b >= a.pb.n_seqs) return;
  const PagedSeq s = paged_seq(a.pb, b);
  const int pos = paged_pos(s, r - s.start);
  if (r < s.start || pos < 0 || pos >= paged_room(a.pb)) return;
  const int id = paged_page(a.pb, b, pos);
  for (int i = threadIdx.x; i < heads * G; i += PR_THREADS) {        // heads * G is a multiple of G: the lanes of a head stay together
    const int h = i / G, e0 = i % G * 8, which = h < KV ? 0 : h < 2 * KV ? 1 : 2, n = which == 2 ? a.n_heads : KV, g = h - which * KV;
    const h8_t x = *(const h8_t *)(a.x[which] + ((size_t)r * n + g) * HD + e0);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = (float)x[e];
    if (which != 1 && a.rope) {
      const h8_t cs = *(const h8_t *)(a.rope + (size_t)pos * HD + e0);   // cos, sin of four pairs
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const float ev = (float)x[2 * p], od = (float)x[2 * p + 1], c = (float)cs[2 * p], d = (float)cs[2 * p + 1];
        f[2 * p] = ev * c - od * d;
        f[2 * p + 1] = ev * d + od * c;
      }
    }
    h8_t o;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = (_Float16)f[e];
    if (which == 2) {
      *(h8_t *)(a.y[2] + ((size_t)r * n + g) * HD + e0) = o;
    } else if (id >= 0) {
      const size_t row = paged_row(a.pb, KV, id, g, pos);
      if constexpr (!I8) {
        *(h8_t *)((_Float16 *)a.pages[which] + row * HD + e0) = o;
      } else {
        uint32_t top = 0;                                     // as bits: what is not a number is above infinity, and that above everything else
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
        top = group_max<G>(top);
        const bool finite = top < 0x7f800000u;
        const float amax = __uint_as_float(top), scale = top == 0 ? 1.0f : finite ? __fdiv_rn(amax, 127.0f) : NAN;
        uint32_t c[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) c[e / 4] |= (uint32_t)((finite ? (int)rintf(__fdiv_rn(f[e], scale)) : 0) & 255) << (e % 4 * 8);
        *(uint2 *)((int8_t *)a.pages[which] + row * HD + e0) = make_uint2(c[0], c[1]);
        if (e0 == 0) a.scales[which][row] = scale;
      }
    }
  }
}

// The same rows back: RN16(code * scale), zeros where there is no page.
template <int HD, bool I8> __global__ __launch_bounds__(PR_THREADS) void paged_read_kernel(PagedArgs a) {
  constexpr int G = HD / 8;
  const int r = blockIdx.x, KV = a.n_kv_heads;
  const int b = paged_find(a.pb, r);
  if (b >= a.pb.n_seqs) return;
  const PagedSeq s = paged_seq(a.pb, b);
  const int pos = paged_pos(s, r - s.start);
  if (r < s.start) return;
  const int id = paged_page(a.pb, b, pos);
  for (int i = threadIdx.x; i < 2 * KV * G; i += PR_THREADS) {
    const int h = i / G, e0 = i % G * 8, which = h < KV ? 0 : 1, g = h - which * KV;
    h8_t o = {};
    if (id >= 0) {
      const size_t row = paged_row(a.pb, KV, id, g, pos);
      if constexpr (I8) {
        const uint2 c = *(const uint2 *)((const int8_t *)a.pages[which] + row * HD + e0);
        const float scale = a.scales[which][row];
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = mul_rn16((float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3))), scale);
      } else {
        o = *(const h8_t *)((const _Float16 *)a.pages[which] + row * HD + e0);
      }
    }
    *(h8_t *)(a.y[which] + ((size_t)r * KV + g) * HD + e0) = o;
  }
}

// Where a block's rows are.
struct PagedRows {
  size_t row[PR_ROWS];                   // of the pages, kv head 0
  int pos[PR_ROWS];                      // -1: no sequence has the row, or its position lies outside the table
  int id[PR_ROWS];                       // -1: no page
};

// Filled by a wavefront for itself: the sequences' arrays, one to a lane and 64 at a time, then a lane per row.  Two round trips to memory, the page numbers being the second.
__device__ __forceinline__ void paged_rows(const PagedBatch &pb, int n_kv_heads, int r0, int n, PagedRows &to) {
  const int lane = threadIdx.x & 63;
  int b = -1, pos = -1;
  for (int b0 = 0, done = 0; b0 < pb.n_seqs && done < n; b0 += 64) {
    PagedSeq s = {0, 0, 0};
    int end = 0x7fffffff;                                    // lanes past the last sequence
    if (b0 + lane < pb.n_seqs) {
      end = pb.row_starts[b0 + lane + 1];
      s = paged_seq(pb.row_starts[b0 + lane], end, pb.lengths[b0 + lane], pb.rows);
    }
    for (; done < n; done++) {                               // the first sequence that ends behind the row
      const uint64_t behind = __builtin_amdgcn_ballot_w64(end > r0 + done);
      if (!behind) break;                                    // in the next 64
      const int l = __builtin_ctzll(behind), start = __builtin_amdgcn_readlane(s.start, l), rows = __builtin_amdgcn_readlane(s.n, l);
      const int at = r0 + done - start;
      if (lane == done && at >= 0 && at < rows) {
        b = b0 + l;
        pos = __builtin_amdgcn_readlane(s.len, l) - rows + at;
      }
    }
  }
  if (lane < n) {
    const bool in = b >= 0 && pos >= 0 && pos < paged_room(pb);
    const int id = in ? paged_page(pb, b, pos) : -1;
    to.pos[lane] = in ? pos : b >= 0 ? -2 : -1;              // -2: a sequence's row all the same, which is read as zeros
    to.id[lane] = id;
    to.row[lane] = id >= 0 ? paged_row(pb, n_kv_heads, id, 0, pos) : 0;
  }
}

// PR_ROWS rows to a block, for batches with blocks enough all the same: more loads behind each look-up.
template <int HD, bool I8> __global__ __launch_bounds__(PR_THREADS) void paged_read_rows_kernel(PagedArgs a) {
  constexpr int G = HD / 8, U = 4;
  __shared__ PagedRows all[PR_THREADS / 64];
  PagedRows &at = all[threadIdx.x >> 6];
  const int r0 = blockIdx.x * PR_ROWS, n_rows = min(PR_ROWS, a.pb.rows - r0), KV = a.n_kv_heads, total = n_rows * (int)a.pieces.d;
  paged_rows(a.pb, KV, r0, n_rows, at);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // of this wavefront, in order
  for (int i0 = threadIdx.x; i0 < total; i0 += U * PR_THREADS) {
    h8_t v[U];
    uint2 c[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = min(i0 + u * PR_THREADS, total - 1), r = a.pieces.div(i), h = (i - r * (int)a.pieces.d) / G, which = h < KV ? 0 : 1;
      // a row without a page asks for the first one's
      const size_t row = at.row[r] + (at.id[r] >= 0 ? (size_t)(h - which * KV) << a.pb.page_shift : 0);
      if constexpr (I8) {
        c[u] = *(const uint2 *)((const int8_t *)a.pages[which] + row * HD + i % G * 8);
        scale[u] = a.scales[which][row];
      } else {
        v[u] = *(const h8_t *)((const _Float16 *)a.pages[which] + row * HD + i % G * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * PR_THREADS, r = a.pieces.div(min(i, total - 1)), h = (i - r * (int)a.pieces.d) / G, which = h < KV ? 0 : 1;
      if (i >= total || at.pos[r] == -1) continue;
      h8_t o = {};
      if (at.id[r] >= 0) {
        if constexpr (I8) {
#pragma unroll
          for (int e = 0; e < 8; e++) o[e] = mul_rn16((float)(int8_t)((e < 4 ? c[u].x : c[u].y) >> (8 * (e & 3))), scale[u]);
        } else {
          o = v[u];
        }
      }
      *(h8_t *)(a.y[which] + ((size_t)(r0 + r) * KV + h - which * KV) * HD + i % G * 8) = o;
    }
  }
}

// Argument checks that the calls on a paged cache share; fills the batch.  Made before anything asks for a device.
int paged_check(const char *who, const jsgrad_hip_pages_t *pg, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, PagedBatch *pb) {
  JSG_REQUIRE(pg && row_starts && lengths, "%s: null pointer argument", who);
  JSG_REQUIRE(pg->pages_k && pg->pages_v && pg->page_table, "%s: null pointer in the pages", who);
  JSG_REQUIRE(pg->kind == JSGRAD_W_F16 || pg->kind == JSGRAD_W_I8, "%s: pages of kind %d (fp16 and int8 are built)", who, pg->kind);
  JSG_REQUIRE(pg->kind == JSGRAD_W_F16 || (pg->scales_k && pg->scales_v), "%s: int8 pages without scales", who);
  JSG_REQUIRE(pg->head_dim == 64 || pg->head_dim == 128, "%s: head_dim %d (64 and 128 are built)", who, pg->head_dim);
  JSG_REQUIRE(pg->page_size >= 16 && pg->page_size <= 256 && (pg->page_size & (pg->page_size - 1)) == 0, "%s: page_size %d (a power of two from 16 to 256)", who, pg->page_size);
  JSG_REQUIRE(pg->n_kv_heads > 0 && pg->n_kv_heads <= 1024 && pg->n_pages > 0, "%s: n_kv_heads %d, n_pages %d", who, pg->n_kv_heads, pg->n_pages);
  JSG_REQUIRE(pg->table_width > 0 && pg->table_width <= (1 << 30) / pg->page_size, "%s: table_width %d", who, pg->table_width);
  JSG_REQUIRE(n_seqs > 0 && n_seqs <= 65535 && rows > 0 && rows < PAGED_GRID, "%s: %d sequences, %d rows", who, n_seqs, rows);
  JSG_REQUIRE((uintptr_t)pg->pages_k % 16 == 0 && (uintptr_t)pg->pages_v % 16 == 0, "%s: pages must be 16-byte aligned", who);
  JSG_REQUIRE(pg->kind == JSGRAD_W_F16 || ((uintptr_t)pg->scales_k % 16 == 0 && (uintptr_t)pg->scales_v % 16 == 0), "%s: scales must be 16-byte aligned", who);
  JSG_REQUIRE((uintptr_t)row_starts % 4 == 0 && (uintptr_t)lengths % 4 == 0 && (uintptr_t)pg->page_table % 4 == 0, "%s: row_starts, lengths and page_table must be 4-byte aligned", who);
  pb->row_starts = row_starts; pb->lengths = lengths; pb->table = pg->page_table;
  pb->n_seqs = n_seqs; pb->rows = rows; pb->width = pg->table_width; pb->n_pages = pg->n_pages;
  pb->page_shift = __builtin_ctz(pg->page_size);
  return 0;
}
static bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

}  // namespace jsg

using namespace jsg;

extern "C" {

int jsgrad_hip_paged_write(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, const void *q,
                           const void *k, const void *v, const void *rope_table, int rope_rows, void *q_out, int n_heads) {
  const char *who = "jsgrad_hip_paged_write";
  PagedArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  JSG_REQUIRE(k && v, "%s: null pointer argument", who);
  JSG_REQUIRE(!q == !q_out, "%s: q and q_out go together", who);
  JSG_REQUIRE(!q || (n_heads > 0 && n_heads <= 65535), "%s: n_heads %d", who, n_heads);
  JSG_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(rope_table) && aligned16(q_out), "%s: rows and the rope table must be 16-byte aligned", who);
  JSG_REQUIRE(!rope_table || rope_rows >= paged_room(a.pb), "%s: a rope table of %d positions, the page table has %d", who, rope_rows, paged_room(a.pb));
  JSG_READY();
  a.pages[0] = host_pages->pages_k; a.pages[1] = host_pages->pages_v;
  a.scales[0] = (float *)host_pages->scales_k; a.scales[1] = (float *)host_pages->scales_v;
  a.x[0] = (const _Float16 *)k; a.x[1] = (const _Float16 *)v; a.x[2] = (const _Float16 *)q;
  a.y[2] = (_Float16 *)q_out;
  a.rope = (const _Float16 *)rope_table;
  a.n_kv_heads = host_pages->n_kv_heads; a.n_heads = q ? n_heads : 0;
  const dim3 grid(rows), block(PR_THREADS);
  const bool i8 = host_pages->kind == JSGRAD_W_I8;
  if (host_pages->head_dim == 64 && i8) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_write_kernel<64, true>), grid, block, 0, a);
  else if (host_pages->head_dim == 64) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_write_kernel<64, false>), grid, block, 0, a);
  else if (i8) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_write_kernel<128, true>), grid, block, 0, a);
  else JSG_LAUNCH(PROF_PAGED_ROWS, (paged_write_kernel<128, false>), grid, block, 0, a);
  return 0;
}

int jsgrad_hip_paged_read(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, void *k_out, void *v_out) {
  const char *who = "jsgrad_hip_paged_read";
  PagedArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  JSG_REQUIRE(k_out && v_out, "%s: null pointer argument", who);
  JSG_REQUIRE(aligned16(k_out) && aligned16(v_out), "%s: rows must be 16-byte aligned", who);
  JSG_READY();
  a.pages[0] = host_pages->pages_k; a.pages[1] = host_pages->pages_v;
  a.scales[0] = (float *)host_pages->scales_k; a.scales[1] = (float *)host_pages->scales_v;
  a.y[0] = (_Float16 *)k_out; a.y[1] = (_Float16 *)v_out;
  a.n_kv_heads = host_pages->n_kv_heads;
  a.pieces = divisor(2 * a.n_kv_heads * (host_pages->head_dim / 8));
  // us, a row to a block | eight, 8 kv heads of 128: int8 2000 rows 4.8 | 6.5, 4096 6.8 | 8.0, fp16 9000 12.9 | 13.5, 32768 47.5 | 43.5 (6.2 TB/s), int8 32768 48 | 34.5 (5.9)
  const bool i8 = host_pages->kind == JSGRAD_W_I8, several = rows > 12288;
  const dim3 grid(several ? (rows + PR_ROWS - 1) / PR_ROWS : rows), block(PR_THREADS);
#define JSG_READ(HD, I8)                                                                             \
  do {                                                                                               \
    if (several) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_read_rows_kernel<HD, I8>), grid, block, 0, a);     \
    else JSG_LAUNCH(PROF_PAGED_ROWS, (paged_read_kernel<HD, I8>), grid, block, 0, a);                  \
  } while (0)
  if (host_pages->head_dim == 64 && i8) JSG_READ(64, true);
  else if (host_pages->head_dim == 64) JSG_READ(64, false);
  else if (i8) JSG_READ(128, true);
  else JSG_READ(128, false);
#undef JSG_READ
  return 0;
}

}  // extern "C"
