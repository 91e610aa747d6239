// Attention over pages that every row chooses by a bound of what they hold: the pages' bounds (jsgrad_hip_paged_bounds), the choice (jsgrad_hip_paged_select), and the attention over what was chosen
// (jsgrad_hip_attn_selected).  No counterpart in the reference.
//
// No key of a page scores more with a query than sum_d q_d (q_d > 0 ? hi_d : lo_d), lo and hi being the least and the largest of each feature.  Both are kept as whole numbers, rounded outwards, times one power of
// two per page and head; a row's queries are rounded to whole numbers times one power of two as well.  So scores are whole numbers below 2^21 times a power of two, exact however they are summed, and
// which pages are chosen is a question of the inputs alone: with float sums two scores that are nearly the same would fall either way.
//
// Figures: us a call, 300 of them with the same inputs one after another, unless they are said to be a profiler's.
#include <type_traits>

#include "paged_device.h"

namespace jsg {

typedef int i4v __attribute__((ext_vector_type(4)));
constexpr int PS_THREADS = 256, PS_MOST = 1024, PS_WIDTH = 32768;      // pages that a row chooses, columns of the table

struct PagedSelectArgs {
  PagedBatch pb;
  const void *pages_k;
  const float *scales_k;
  const _Float16 *q;                     // [rows][H][HD]
  int8_t *bounds;                        // [n_pages][KV][lo, hi][HD]
  float *bound_scales;                   // [n_pages][KV]
  int n_kv_heads, n_rep, first, recent, top;
  int tile, heads_log, stride;           // rows of a block, columns of queries to a row as a power of two, keys of a row
  int32_t *selected;                     // [rows][KV][top]
};

// sums of a lane's value and those of the lanes below
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);    // row_shr 1, 2, 4, 8
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
  return v;
}

// The sequence of a row, and its number; n_seqs where none has it.  As paged_find and paged_seq, for a uniform r, but in one trip to memory for up to 64 sequences: it is in front of everything else.
__device__ __forceinline__ int find_row(const PagedBatch &pb, int r, PagedSeq &s) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < pb.n_seqs; b0 += 64) {
    const int b = min(b0 + lane, pb.n_seqs - 1), start = pb.row_starts[b], end = pb.row_starts[b + 1], len = pb.lengths[b];
    const uint64_t behind = __builtin_amdgcn_ballot_w64(end > r);
    if (!behind) continue;
    const int l = __builtin_ctzll(behind);
    s = paged_seq(__builtin_amdgcn_readlane(start, l), __builtin_amdgcn_readlane(end, l), __builtin_amdgcn_readlane(len, l), pb.rows);
    return b0 + l;
  }
  return pb.n_seqs;
}

// The smallest power of two, 2^-126 and more, that 127 times is `most` (finite) and more; 1 for 0.
__device__ __forceinline__ float bound_step(float most) {
  if (most == 0.0f) return 1.0f;
  const int e = __builtin_amdgcn_frexp_expf(most);           // most = f * 2^e, 1/2 <= f < 1
  const float f = __builtin_amdgcn_frexp_mantf(most);
  return __builtin_amdgcn_ldexpf(1.0f, max(e - 7 + (f > 127.0f / 128.0f), -126));
}

// The t-th page that the batch's rows are on, sequence by sequence: its sequence (n_seqs: there are not so many) and the page's first position.  A sequence to a lane.
__device__ __forceinline__ int find_touched(const PagedBatch &pb, uint32_t t, PagedSeq &s, int &first) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < pb.n_seqs; b0 += 64) {
    const int b = min(b0 + lane, pb.n_seqs - 1), start = pb.row_starts[b], end = pb.row_starts[b + 1], len = pb.lengths[b];
    const PagedSeq mine = paged_seq(start, end, len, pb.rows);
    const int p0 = max(paged_pos(mine, 0), 0) >> pb.page_shift;
    const uint32_t n = b0 + lane < pb.n_seqs && mine.n > 0 && mine.len > 0 ? (uint32_t)(((mine.len - 1) >> pb.page_shift) - p0 + 1) : 0, upto = wave_upto(n);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(upto > t);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      s = {__builtin_amdgcn_readlane(mine.start, l), __builtin_amdgcn_readlane(mine.n, l), __builtin_amdgcn_readlane(mine.len, l)};
      first = (__builtin_amdgcn_readlane(p0, l) + (int)(t - (uint32_t)__builtin_amdgcn_readlane((int)(upto - n), l))) << pb.page_shift;
      return b0 + l;
    }
    t -= (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  }
  return pb.n_seqs;
}

// Block = (page that the batch's rows are on, kv head): the whole page is looked at, so bounds do not depend on how its rows came.  Bound by memory: HD / 8 lanes a row, 16 bytes (int8: 8) each.
// One row behind 33000 positions takes 4.5 us, 16 of 16 sequences 4.5, most of it a launch; 2048 rows on 32 pages 5.1.  (A block for every row, most of which have nothing to do: 27.)
template <int HD, bool I8> __global__ __launch_bounds__(PS_THREADS) void paged_bounds_kernel(PagedSelectArgs a) {
  constexpr int G = HD / 8, RPB = PS_THREADS / G;
  __shared__ float lo_sh[PS_THREADS / 64][HD], hi_sh[PS_THREADS / 64][HD];
  __shared__ float most_sh[PS_THREADS / 64];
  const int g = blockIdx.y, KV = a.n_kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  PagedSeq s;
  int first;
  const int b = find_touched(a.pb, blockIdx.x, s, first);
  if (b >= a.pb.n_seqs) return;
  const int id = paged_page(a.pb, b, first);
  if (id < 0) return;
  const int n = min(1 << a.pb.page_shift, s.len - first);
  const size_t row0 = paged_row(a.pb, KV, id, g, first);
  const int e0 = threadIdx.x % G * 8;
  float lo[8], hi[8];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; e++) { lo[e] = INFINITY; hi[e] = -INFINITY; }
  for (int i = threadIdx.x / G; i < n; i += RPB) {
    float f[8];
    if constexpr (I8) {
      const uint2 c = *(const uint2 *)((const int8_t *)a.pages_k + (row0 + i) * HD + e0);
      const float scale = a.scales_k[row0 + i];
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = (float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3))) * scale;
    } else {
      const h8_t x = *(const h8_t *)((const _Float16 *)a.pages_k + (row0 + i) * HD + e0);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = (float)x[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      bad |= !(fabsf(f[e]) < INFINITY);
      lo[e] = fminf(lo[e], f[e]);
      hi[e] = fmaxf(hi[e], f[e]);
    }
  }
  // over the rows of a wavefront: lanes G, 2 G .. apart
#pragma unroll
  for (int d = G; d < 64; d <<= 1)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      lo[e] = fminf(lo[e], __shfl_xor(lo[e], d));
      hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], d));
    }
  if (lane < G)
#pragma unroll
    for (int e = 0; e < 8; e++) { lo_sh[wave][e0 + e] = lo[e]; hi_sh[wave][e0 + e] = hi[e]; }
  bad = __syncthreads_or(bad);
  float l = INFINITY, h = -INFINITY, most = 0.0f;
  const int d = threadIdx.x % HD;
  for (int w = 0; w < PS_THREADS / 64; w++) {
    l = fminf(l, lo_sh[w][d]);
    h = fmaxf(h, hi_sh[w][d]);
  }
  most = wave_max(fmaxf(fabsf(l), fabsf(h)));
  if (lane == 0) most_sh[wave] = most;
  __syncthreads();
  for (int w = 0; w < PS_THREADS / 64; w++) most = fmaxf(most, most_sh[w]);
  const float step = bad ? INFINITY : bound_step(most);      // of a page with a key that is not finite: no bound
  if (threadIdx.x < HD) {
    int8_t *const to = a.bounds + ((size_t)id * KV + g) * 2 * HD + d;
    // outwards also where the quotient is nothing that a float holds
    const float lower = floorf(__fdiv_rn(l, step)), upper = ceilf(__fdiv_rn(h, step));
    to[0] = bad ? 0 : (int8_t)(int)(l < 0.0f ? fminf(lower, -1.0f) : lower);
    to[HD] = bad ? 0 : (int8_t)(int)(h > 0.0f ? fmaxf(upper, 1.0f) : upper);
    if (d == 0) a.bound_scales[(size_t)id * KV + g] = step;
  }
}

// Order of scores as that of whole numbers above 0.
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

constexpr uint32_t KEY_ALWAYS = 0xffffffffu;               // of a page that is among the first or the recent ones; 0: of one that is not there

// over the lanes, for all of them: a value from the lanes below, row by row, then from row to row; the last lane has everything
template <typename Op> __device__ __forceinline__ uint32_t wave_all(uint32_t v, Op op) {
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, false));     // quad_perm [1,0,3,2], [2,3,0,1], then the halves of a row and the row mirrored
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xf, 0xf, false));
  auto row = [&](int r) { return (uint32_t)__builtin_amdgcn_readlane((int)v, r * 16); };
  return op(op(row(0), row(1)), op(row(2), row(3)));
}
// The first `top` of n keys in the order (key descending, index ascending), those above 0, written as rising indexes with -1 behind.  By one wavefront, or by a block of NW, each with a stretch of
// the keys.  What lies between the least and the largest is counted in 256 parts, then the part with the border in 256 again, until a part is wanted whole or its keys are all alike: two or
// three turns, four at most.  (Halving a threshold takes some 15: 33000 positions in pages of 64, 4.3 us of them.)
template <int NW> struct KeyChoice {
  static constexpr int TURNS = NW == 1 ? 1 : 4;              // counts that stay zero until their turn; one wavefront clears its own
  __align__(16) uint32_t hist[TURNS][256];
  uint32_t least[NW], most[NW], real[NW], always[NW], above[NW], tied[NW];

  __device__ __forceinline__ void operator()(const uint32_t *keys, int n, int top, int32_t *out, int wave) {
    const int per = NW == 1 ? n : ((n + NW - 1) / NW + 63) & ~63, lo = min(wave * per, n), hi = min(lo + per, n);
    if (per <= 4 * 64) choose<4>(keys, lo, hi, n, top, out, wave);
    else choose<0>(keys, lo, hi, n, top, out, wave);
  }
  // K: keys of a lane; 0: any number, from where they are
  template <int K> __device__ void choose(const uint32_t *keys, int lo, int hi, int n, int top, int32_t *out, int wave) {
    const int lane = threadIdx.x & 63;
    uint32_t mine[K ? K : 1];
#pragma unroll
    for (int u = 0; u < K; u++) mine[u] = lo + u * 64 + lane < hi ? keys[lo + u * 64 + lane] : 0;
    auto each = [&](auto f) {                                // f(key, its index less the lane), 64 side by side; 0 past the end
      if constexpr (K > 0) {
#pragma unroll
        for (int u = 0; u < K; u++) f(mine[u], lo + u * 64);
      } else {
        for (int i = lo; i < hi; i += 256) {
          uint32_t k[4];
#pragma unroll
          for (int u = 0; u < 4; u++) k[u] = i + u * 64 + lane < hi ? keys[i + u * 64 + lane] : 0u;
#pragma unroll
          for (int u = 0; u < 4; u++) f(k[u], i + u * 64);
        }
      }
    };
    auto join = [&](uint32_t (&of)[NW], uint32_t v, auto op) {   // over the block, behind a barrier
      if constexpr (NW == 1) return v;
      uint32_t all = of[0];
#pragma unroll
      for (int w = 1; w < NW; w++) all = op(all, of[w]);
      return all;
    };
    auto sum = [](uint32_t x, uint32_t y) { return x + y; };
    auto lower = [](uint32_t x, uint32_t y) { return min(x, y); };
    auto upper = [](uint32_t x, uint32_t y) { return max(x, y); };
    uint32_t a = ~0u, b = 0, n_real = 0, n_always = 0;       // of the keys between 0 and KEY_ALWAYS
    each([&](uint32_t k, int) {
      const bool some = k - 1 < KEY_ALWAYS - 1;
      a = min(a, some ? k : ~0u);
      b = max(b, some ? k : 0u);
      n_real += some;
      n_always += k == KEY_ALWAYS;
    });
    a = wave_all(a, lower);
    b = wave_all(b, upper);
    n_real = wave_all(n_real, sum);
    n_always = wave_all(n_always, sum);
    if constexpr (NW > 1) {
      if (lane == 0) { least[wave] = a; most[wave] = b; real[wave] = n_real; always[wave] = n_always; }
      for (int i = threadIdx.x; i < TURNS * 256; i += NW * 64) hist[0][i] = 0;
      lds_barrier();
      a = join(least, a, lower);
      b = join(most, b, upper);
      n_real = join(real, n_real, sum);
      n_always = join(always, n_always, sum);
    }
    uint32_t t = 1;                                          // what is chosen reaches it; of the keys that are t, the first `ties`
    int ties = n;
    uint32_t need = (uint32_t)top - min(n_always, (uint32_t)top);
    if (need == 0) t = KEY_ALWAYS;
    else if (n_real > need)
      for (int turn = 0;; turn++) {
        const uint32_t span = b - a;
        const int shift = span < 256 ? 0 : 24 - __builtin_clz(span);
        uint32_t *const h = hist[NW == 1 ? 0 : turn];
        if constexpr (NW == 1) *(uint4 *)&h[lane * 4] = make_uint4(0, 0, 0, 0);
        each([&](uint32_t k, int) {
          if (k - a <= span) atomicAdd(&h[(k - a) >> shift], 1u);
        });
        if constexpr (NW > 1) lds_barrier();
        const uint4 c = *(const uint4 *)&h[252 - 4 * lane];  // from the largest down
        const uint32_t four = c.x + c.y + c.z + c.w, upto = wave_upto(four);
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto >= need));
        auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
        uint32_t before = of(upto - four), bin = 255 - 4 * l, held = of(c.w);
        if (before + held < need) { before += held; held = of(c.z); bin--; }
        if (before + held < need) { before += held; held = of(c.y); bin--; }
        if (before + held < need) { before += held; held = of(c.x); bin--; }
        need -= before;
        a += bin << shift;
        t = a;
        if (held == need) break;
        if (shift == 0) { ties = (int)need; break; }
        b = min(b, a + ((1u << shift) - 1));
      }
    int at = 0, left = ties;
    if constexpr (NW > 1) {
      uint32_t over = 0, equal = 0;
      each([&](uint32_t k, int) { over += k > t; equal += k == t; });
      over = wave_all(over, sum);
      equal = wave_all(equal, sum);
      if (lane == 0) { above[wave] = over; tied[wave] = equal; }
      lds_barrier();
      for (int w = 0; w < wave; w++) {
        const int held = min(left, (int)tied[w]);
        at += (int)above[w] + held;
        left -= held;
      }
    }
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    each([&](uint32_t k, int i) {
      const uint64_t tie = __builtin_amdgcn_ballot_w64(k == t);
      const bool take = k > t || (k == t && (int)__builtin_popcountll(tie & below) < left);
      left -= min(left, (int)__builtin_popcountll(tie));
      const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
      const int place = at + (int)__builtin_popcountll(taken & below);
      if (take && place < top) out[place] = i + lane;
      at += (int)__builtin_popcountll(taken);
    });
    if (NW == 1 || wave == NW - 1)
      for (int i = at + lane; i < top; i += 64) out[i] = -1;
  }
};

// Block = some rows of a sequence, side by side, and a kv head.  Scores on the matrix cores: 16 pages' bounds against 16 columns of queries, the heads of a row next to each other, so that a lane has
// four columns' scores of its page.  Few rows are bound by what waits for what: batch, page numbers, bounds, then the turns of the choice.  Of many, the vector unit, which makes keys of scores and counts them, has half
// of the time (11.0 M instructions, 43 of 87 thousand cycles of each), and wavefronts wait for 44 % of theirs.
// us, one row of 33000 positions, pages of 64, 32 heads of 128 over 8: 8.4; 16 rows of up to 32768, pages of 32: 11; 2048 rows behind 14336, heads of 64: 26.  (A page to a thread with dot products and 32 turns
// through LDS, by the profiler: 22, 30 and 138, where these take 9, 12 and 30.)
// HT tiles of 16 columns: of more heads of the rows (HEADS), or of more rows, for which the bounds are loaded once.
template <int HD, int NW, int HT, bool HEADS> __global__ __launch_bounds__(NW * 64, 2) void paged_select_kernel(PagedSelectArgs a) {
  extern __shared__ __align__(16) uint32_t keys[];           // [rows of a block][stride]
  __shared__ union {
    KeyChoice<NW> block;
    KeyChoice<1> wave[NW];
    unsigned char box[NW][16 * (2 * HD + 16)];               // each wavefront's tile of bounds, a page to a row; sixteen bytes between them, so that 16 rows' pieces meet all banks alike
  } sm;
  constexpr int KS = 2 * HD / 64, LPP = 2 * HD / 16, ROW = 2 * HD + 16;   // steps of 64 bytes (the lower bounds, then the upper ones), lanes to a page, bytes between pages
  const int g = blockIdx.y, KV = a.n_kv_heads, n_rep = a.n_rep, lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hp = 1 << a.heads_log, shift = a.pb.page_shift;
  const int r_end = min((int)(blockIdx.x + 1) * a.tile, a.pb.rows);
  for (int r0 = blockIdx.x * a.tile; r0 < r_end;) {
    PagedSeq s;
    const int b = find_row(a.pb, r0, s);
    if (b >= a.pb.n_seqs) return;
    const int n_rows = min(s.start + s.n, r_end) - r0;
    if (r0 < s.start) { r0++; continue; }                    // no sequence has it
    const int p0 = paged_pos(s, r0 - s.start), last_page = p0 + n_rows - 1 < 0 ? -1 : (p0 + n_rows - 1) >> shift, n = min(last_page + 1, a.pb.width);
    // U tiles at a time: their page numbers in one trip to memory, asked for ahead, their bounds in the next.  The numbers without a branch: behind one, each would be waited for.
    constexpr int U = HT > 1 || NW == 8 ? 2 : 4;
    const int32_t *const table = a.pb.table + (size_t)b * a.pb.width;
    int id[U];
    auto pages_of = [&](int t0) {
#pragma unroll
      for (int u = 0; u < U; u++) id[u] = *as_global<int>(table + max(min((t0 + u * NW) * 16 + l16, n - 1), 0));
    };
    pages_of(wave);
    // column l16 of a tile: a head of a row; those past the last repeat it
    u4_t q[HT][HD / 64][2];
    float most[HT];
#pragma unroll
    for (int h = 0; h < HT; h++) {
      const int row = min((HEADS ? 0 : h * (16 >> a.heads_log)) + (l16 >> a.heads_log), n_rows - 1), head = min((HEADS ? h * 16 : 0) + (l16 & (hp - 1)), n_rep - 1);
      const _Float16 *const qp = a.q + (((size_t)(r0 + row) * KV + g) * n_rep + head) * HD + lq * 16;
      uint32_t bits = 0;                                     // of the largest |q|, in both halves
#pragma unroll
      for (int c = 0; c < HD / 64; c++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          q[h][c][u] = *as_global<u4_t>(qp + c * 64 + u * 8);
#pragma unroll
          for (int w = 0; w < 4; w++) {
            typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
            const us2_t v = __builtin_bit_cast(us2_t, q[h][c][u][w] & 0x7fff7fffu), m = __builtin_bit_cast(us2_t, bits);
            bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(v, m));
          }
        }
      bits = max(bits & 0xffff, bits >> 16);                 // halves without their sign are in the order of their bits
      most[h] = bits < 0x7c00 ? h2f(__builtin_bit_cast(_Float16, (uint16_t)bits)) : INFINITY;
      most[h] = max_xor32(max_xor16(most[h]));
      for (int off = 1; off < hp; off <<= 1) most[h] = fmaxf(most[h], __shfl_xor(most[h], off));
    }
    if (HEADS)
#pragma unroll
      for (int h = 0; h < HT; h++) most[0] = fmaxf(most[0], most[h]);
    i4v qf[HT][KS];                                          // negative parts against lower bounds, positive ones against upper
#pragma unroll
    for (int h = 0; h < HT; h++) {
      const bool says = most[HEADS ? 0 : h] < INFINITY;      // queries that are not finite say nothing
      const float per_step = says ? 1.0f / bound_step(most[HEADS ? 0 : h]) : 0.0f;   // of a power of two: exact
#pragma unroll
      for (int c = 0; c < HD / 64; c++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
          uint32_t v[4];                                     // the addition rounds to a whole number, whose last byte is the code
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const h2_t p = as_h2(q[h][c][w / 2][w % 2 * 2 + e / 2]);
            v[e] = __float_as_uint(__builtin_fmaf((float)p[e % 2], per_step, 12582912.0f));
          }
          const uint32_t code = says ? __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], 0x0c0c0400u), __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u), 0x05040100u) : 0;
          const uint32_t sign = (code >> 7) & 0x01010101u, minus = (sign << 8) - sign;
          qf[h][c][w] = (int)(code & minus);
          qf[h][HD / 64 + c][w] = (int)(code & ~minus);
        }
    }
    for (int t0 = wave; t0 * 16 < n; t0 += U * NW) {
      // As they lie, neighbouring lanes on one page, and through LDS into the operand, whose lanes of a quarter are on different pages: straight from there, L1 is asked 64 times for what it gives in 16
      // (2048 rows behind 14336, heads of 64, 30.7 us instead of 26.4, one row of 33000 9.7 instead of 8.4 together with the four more wavefronts that it has).
      i4v box[U][KS];
      float scale[U];
      bool held[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if ((t0 + u * NW) * 16 + l16 >= n || id[u] >= a.pb.n_pages) id[u] = -1;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const size_t at = (size_t)max(id[u], 0) * KV + g;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const int of = max(__shfl(id[u], k * (64 / LPP) + lane / LPP), 0);
          box[u][k] = *as_global<i4v>(a.bounds + ((size_t)of * KV + g) * 2 * HD + lane % LPP * 16);
        }
        scale[u] = *as_global<float>(a.bound_scales + at);
        held[u] = id[u] >= 0;
      }
      pages_of(t0 + U * NW);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = (t0 + u * NW) * 16 + l16;
        if (i - l16 >= n) break;
        i4v bf[KS];
#pragma unroll
        for (int k = 0; k < KS; k++) *(i4v *)(sm.box[wave] + (k * (64 / LPP) + lane / LPP) * ROW + lane % LPP * 16) = box[u][k];
#pragma unroll
        for (int k = 0; k < KS; k++) bf[k] = *(const i4v *)(sm.box[wave] + l16 * ROW + k * 64 + lq * 16);
        float v[4];
#pragma unroll
        for (int h = 0; h < HT; h++) {
          i4v acc = {0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < KS; k++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf[h][k], bf[k], acc, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] = HEADS && h ? fmaxf(v[e], (float)acc[e]) : (float)acc[e];   // column 4 lq + e, page l16
        if (HEADS && h < HT - 1) continue;
        // over a row's columns
        if (a.heads_log >= 1) { v[0] = fmaxf(v[0], v[1]); v[2] = fmaxf(v[2], v[3]); }
        if (a.heads_log >= 2) v[0] = fmaxf(v[0], v[2]);
        if (a.heads_log >= 3) v[0] = max_xor16(v[0]);
        if (a.heads_log >= 4) v[0] = max_xor32(v[0]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int at = (HEADS ? 0 : h * (16 >> a.heads_log)) + ((4 * lq + e) >> a.heads_log);
          if ((e & (hp - 1)) != 0 || at >= n_rows || i >= n) continue;
          const int last = p0 + at < 0 ? -1 : (p0 + at) >> shift;
          // in units 2^-15 as large: 2^21 times the largest, 2^122, is a float then, and a whole number of the smallest, 2^-126, still one (below the normal ones)
          uint32_t key = min(score_key(scale[u] < INFINITY ? v[e] * (scale[u] * 0x1p-15f) : INFINITY), KEY_ALWAYS - 1);
          if (i < a.first || i > last - a.recent) key = KEY_ALWAYS;
          if (!held[u] || i > last) key = 0;
          keys[at * a.stride + i] = key;
        }
        }
      }
    }
    __syncthreads();
    auto place = [&](int at) { return a.selected + ((size_t)(r0 + at) * KV + g) * a.top; };
    auto pages = [&](int at) { return p0 + at < 0 ? 0 : min(((p0 + at) >> shift) + 1, a.pb.width); };
    if (a.tile == 1) sm.block(keys, n, a.top, place(0), wave);
    else
      for (int at = wave; at < n_rows; at += NW) sm.wave[wave](keys + at * a.stride, pages(at), a.top, place(at), 0);
    r0 += n_rows;
    if (r0 < r_end) __syncthreads();
  }
}

// ---------------------------------------------------------------- attention over the chosen pages

// Block = 4 wavefronts.  Where there are few rows, one row, up to 16 of its query heads of a kv head (usually four), and a part of its chosen pages, each wavefront with steps of its own; else (SOLO) four
// rows, a wavefront to each, which neither wait for one another nor start anew every few steps.  A step is 64 keys: rows of K and V
// come through registers into the wavefront's own LDS, 32 at a time, V's for the transposing reads; the next step's rows are asked for as soon as the registers are free.  K straight to registers, as the
// matrix operand has it, would put the lanes of a quarter on different rows, and the L1 cache would be asked 64 times for what it gives in 16: 2048 rows, heads of 64, 305 us by the profiler.
//
// us, 32 heads over 8: one row, 32 pages of 64, heads of 128, 9.8, of which 4 go by until the first keys are there and 4 in the join of the parts; 16 rows, 64 int8 pages of 32, heads of 128, 21: memory, 4 TB/s and start
// and join; 2048 rows, 16 pages of 64, heads of 64, 168 (the profiler says 195): every row gathers 2 MB of its own, 4.3 GB in all, in the profile at 64 % of what L1 gives and as much of LDS's rate (each byte goes in
// once and out once), 20 TB/s of it from L2, with the vector unit at 32 %.
//
// A matrix instruction scores 16 keys for 16 columns, and a row has few heads: with four, three columns of four would score the same again, and the vector unit would make the exponentials of
// all.  So the columns are heads times groups of keys: column c of what a lane keeps has head c % HP over the keys of group c / HP of the step's four, each picked from that group's scores
// (a selection per value), and holds its own running maximum, sum and share of the output; its weights are the operand of O^T = V^T . P^T with zeros at the other groups' keys.  The columns of a
// head meet at the end, with the wavefronts.  A: accumulators that are left, 1 where a row has up to 4 heads, 2 up to 8, 4 beyond.
constexpr int PA_THREADS = 256, PA_QROWS = 16, PA_MOST = 64;           // parts of a row: a lane for each
constexpr int PA_SLOTS = 1024, PA_BLOCKS = 512;
constexpr float PA_TOP = 15.0f;                            // a column's largest weight is 2^15: halves are normal numbers down to 2^-29 of it

struct SelectedArgs {
  PagedBatch pb;
  const void *pages_k, *pages_v;
  const float *scales_k, *scales_v;
  const _Float16 *q;                     // [rows][H][HD]
  _Float16 *out;
  const int32_t *selected;               // [rows][KV][top]
  int n_heads, n_rep, heads_log, top, parts, q_tiles;
  Divisor n_kv_heads;
  float scale_log2;                      // float(1 / sqrt(HD)) * log2(e)
  int *counters;                         // zero, and zero again afterwards
  float *ws;
};

template <int HD, bool I8, int A, bool SOLO> struct SelectedRow {
  static constexpr int NW = 4, ROW_WAVES = SOLO ? 1 : NW, ROW_THREADS = ROW_WAVES * 64, KEYS = 64, ROWB = HD * 2;
  static constexpr int VROW = ROWB + 32;                     // bytes between V rows in LDS: eight banks further each, so that the reads of 16 rows by 32 bytes meet all banks alike
  static constexpr int NT = HD / 16, KS = HD / 32;           // 16-feature tiles of the output, matrix instructions per 16 keys
  static constexpr int OROW = HD + 4;                        // floats between rows of a wavefront's sums in LDS
  static constexpr int KROW = ROWB + 16;                     // and K rows in LDS: eight rows' 16 bytes meet all banks alike
  static constexpr int LPR = HD / (I8 ? 16 : 8), GV = LPR / 4;   // lanes to a row, 16-byte loads of 16 keys' rows
  static constexpr int SLOT = PA_QROWS * (HD + 4);           // floats of a part: the heads' sums, then (m, l, -, -) of each
  struct Smem {
    union {
      unsigned char v[32 * VROW];
      float o[16 * OROW];
    } wave[NW];
    float m[NW][16], l[NW][16];
    float w[SOLO ? 1 : PA_QROWS][PA_MOST], inv[PA_QROWS];
    f4_t fold[SOLO ? 1 : PA_THREADS];
    int2 list[SOLO ? 1 : PS_MOST + 4];                       // the row's pages: number, first position; SOLO: in the lanes
    int most[NW], is_last;
  };

  // Must be called by every thread of the block (it contains barriers; SOLO: of the wavefront, and none).  r, pos: the row and its position; chosen: this thread's entry of its list.
  static __device__ void run(const SelectedArgs &a, int r, int g, int qt, int part, int b, int pos, int chosen, Smem &sm) {
    const int lane = threadIdx.x & 63, tid = SOLO ? lane : threadIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, lq = lane >> 4;
    const int n_rep = a.n_rep, KV = (int)a.n_kv_heads.d, hp = 1 << a.heads_log, shift = a.pb.page_shift, q0 = qt * PA_QROWS, nr = min(PA_QROWS, n_rep - q0);
    const int cg = l16 >> a.heads_log;                       // this lane's group
    const size_t q_off = ((size_t)r * a.n_heads + g * n_rep + q0) * HD;
    h8_t qf[KS];                                             // the features that the K fragments have: 8 (4 s + lq) ..
    {
      const _Float16 *const qp = a.q + q_off + (size_t)min(l16 & (hp - 1), nr - 1) * HD;   // columns past the last head repeat it and are never stored
#pragma unroll
      for (int s = 0; s < KS; s++) qf[s] = *as_global<h8_t>(qp + 8 * (4 * s + lq));
    }
    // the list, up to the last entry that names a page
    const int32_t *const sel = a.selected + ((size_t)r * KV + g) * a.top;
    const int last = pos < 0 ? -1 : pos >> shift;
    auto held_by = [&](int page) { return page >= 0 && page <= last && page < a.pb.width ? paged_page(a.pb, b, page << shift) : -1; };
    int n = 0, my_id = -1, my_first = 0;
    if constexpr (SOLO) {
      my_id = held_by(chosen);
      my_first = my_id >= 0 ? chosen << shift : 0;
      const uint64_t held = __builtin_amdgcn_ballot_w64(my_id >= 0);
      n = held ? 64 - __builtin_clzll(held) : 0;
    } else {
      for (int i = tid; i < a.top + 4; i += PA_THREADS) {
        const int page = i < PA_THREADS ? chosen : i < a.top ? sel[i] : -1, held = held_by(page);
        sm.list[i] = make_int2(held, held >= 0 ? page << shift : 0);
        if (held >= 0) n = i + 1;
      }
      for (int d = 32; d > 0; d >>= 1) n = max(n, __shfl_xor(n, d));
      if (lane == 0) sm.most[wave] = n;
      lds_barrier();
      n = max(max(sm.most[0], sm.most[1]), max(sm.most[2], sm.most[3]));
    }
    const int steps = ((n << shift) + KEYS - 1) / KEYS, per = SOLO ? steps : (steps + a.parts - 1) / a.parts, st_lo = SOLO ? 0 : min(part * per, steps), st_end = min(st_lo + per, steps);

    struct Step {
      int id[4], key[4];                                     // of the four groups: page, first position
    };
    auto find = [&](int st, Step &to) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int at = st * KEYS + 16 * j, i = at >> shift;
        if constexpr (SOLO) {
          to.id[j] = i < 64 ? __builtin_amdgcn_readlane(my_id, i) : -1;
          to.key[j] = (i < 64 ? __builtin_amdgcn_readlane(my_first, i) : 0) + (at & ((1 << shift) - 1));
        } else {
          const int2 e = sm.list[min(i, a.top)];             // behind the last: none
          to.id[j] = st < st_end ? __builtin_amdgcn_readfirstlane(e.x) : -1;
          to.key[j] = __builtin_amdgcn_readfirstlane(e.y) + (at & ((1 << shift) - 1));
        }
      }
    };
    u4_t kr[4][GV], vr[4][GV];
    f4_t ks[A], vs[A];                                       // of the keys that this lane keeps
    auto row_of = [&](const Step &to, int j) { return paged_row(a.pb, KV, max(to.id[j], 0), g, to.key[j]); };   // a missing page: page 0, masked
    auto mine = [&](auto v0, auto v1, auto v2, auto v3, int at) {   // of the four groups' values, that of this lane's accumulator `at`
      if constexpr (A == 1) return cg == 0 ? v0 : cg == 1 ? v1 : cg == 2 ? v2 : v3;
      else if constexpr (A == 2) return at == 0 ? (cg == 0 ? v0 : v1) : (cg == 0 ? v2 : v3);
      else return at == 0 ? v0 : at == 1 ? v1 : at == 2 ? v2 : v3;
    };
    // a group's rows lie side by side: a base that all lanes share, and a lane's place from there
    constexpr int HELD = I8 ? HD : ROWB;
    const uint32_t lane_at = lane / LPR * HELD + lane % LPR * 16;
    auto load_rows = [&](const void *pages, const Step &to, int j, u4_t (&r)[GV]) {
      const JSG_GLOBAL unsigned char *const from = as_global<unsigned char>(pages) + row_of(to, j) * HELD;
#pragma unroll
      for (int c = 0; c < GV; c++) r[c] = *(const JSG_GLOBAL u4_t *)(from + (lane_at + c * (64 / LPR) * HELD));
    };
    auto store_rows = [&](const u4_t (&r)[GV], int h, int row_bytes) {   // 16 rows to LDS as halves, behind h * 16 others
#pragma unroll
      for (int c = 0; c < GV; c++) {
        unsigned char *const to = sm.wave[wave].v + (16 * h + c * (64 / LPR) + lane / LPR) * row_bytes + lane % LPR * (I8 ? 32 : 16);
        if constexpr (I8) {
#pragma unroll
          for (int x = 0; x < 2; x++) {
            uint32_t w[4];
            i8x4_to_h2x2(r[c][2 * x], w[0], w[1]);
            i8x4_to_h2x2(r[c][2 * x + 1], w[2], w[3]);
            *(u4_t *)(to + x * 16) = u4_t{w[0], w[1], w[2], w[3]};
          }
        } else {
          *(u4_t *)to = r[c];
        }
      }
    };
    auto load_k = [&](const Step &to) {
#pragma unroll
      for (int j = 0; j < 4; j++) load_rows(a.pages_k, to, j, kr[j]);
      if constexpr (I8)
#pragma unroll
        for (int s = 0; s < A; s++) ks[s] = *as_global<f4_t>(a.scales_k + mine(row_of(to, 0), row_of(to, 1), row_of(to, 2), row_of(to, 3), s) + 4 * lq);
    };
    auto load_v = [&](const Step &to, int u) {               // groups 2 u and 2 u + 1
#pragma unroll
      for (int j = 2 * u; j < 2 * u + 2; j++) load_rows(a.pages_v, to, j, vr[j]);
    };
    auto load_vs = [&](const Step &to) {
      if constexpr (I8)
#pragma unroll
        for (int s = 0; s < A; s++) vs[s] = *as_global<f4_t>(a.scales_v + mine(row_of(to, 0), row_of(to, 1), row_of(to, 2), row_of(to, 3), s) + 4 * lq);
    };

    int st;
    Step at, next;
    f4_t o[NT];
    float m_run, l_run;
    const float unit = I8 ? 1.0f : a.scale_log2;
    unsigned char *const vl = sm.wave[wave].v;

    // more: there is another step; careful: V may hold halves that are not finite
    auto step = [&](auto more, auto careful) {
      constexpr bool MORE = decltype(more)::value, CAREFUL = decltype(careful)::value;
      find(st + ROW_WAVES, next);
      f4_t d[4];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        store_rows(kr[2 * u], 0, KROW);
        store_rows(kr[2 * u + 1], 1, KROW);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < KS; c++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const h8_t *)(vl + (16 * h + l16) * KROW + (4 * c + lq) * 16), qf[c], acc, 0, 0, 0);
          d[2 * u + h] = acc;
        }
      }
      f4_t s[A];
#pragma unroll
      for (int x = 0; x < A; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[x][e] = mine(d[0][e], d[1][e], d[2][e], d[3][e], x);
      f4_t kscale[A], inv_v[A];
      if constexpr (I8)
#pragma unroll
        for (int x = 0; x < A; x++) kscale[x] = ks[x] * a.scale_log2;
      if constexpr (MORE) load_k(next);
      if constexpr (I8) {
        // scale_of_v, for which there is a reason in few steps: 16 codes of zero side by side, or a scale below PAGED_TINY
        uint32_t codes = ~0u;
        float least = INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int c = 0; c < GV; c++) codes = min(codes, vr[j][c][0] | vr[j][c][1] | vr[j][c][2] | vr[j][c][3]);
#pragma unroll
        for (int x = 0; x < A; x++)
#pragma unroll
          for (int e = 0; e < 4; e++) least = fminf(least, vs[x][e]);
        if (__builtin_amdgcn_ballot_w64(codes == 0 || least < PAGED_TINY)) {
          uint32_t zeros[4];                                 // of rows 4 lq .. of each group: which are all zero
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint64_t some[GV];                               // lanes LPR * r and on have row r of the sixteen: LPR bits of each of these four rows
#pragma unroll
            for (int c = 0; c < GV; c++) some[c] = __builtin_amdgcn_ballot_w64((vr[j][c][0] | vr[j][c][1] | vr[j][c][2] | vr[j][c][3]) != 0);
            const uint64_t held = GV == 1 || lq * GV / 4 == 0 ? some[0] : some[GV - 1];
            const uint32_t rows = (uint32_t)(held >> (lq * 4 % (64 / LPR)) * LPR);
            zeros[j] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) zeros[j] |= (uint32_t)(((rows >> e * LPR) & ((1u << LPR) - 1)) == 0) << e;
          }
#pragma unroll
          for (int x = 0; x < A; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) vs[x][e] = scale_of_v(vs[x][e], mine(zeros[0], zeros[1], zeros[2], zeros[3], x) >> e & 1);
        }
#pragma unroll
        for (int x = 0; x < A; x++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            // the scale of V in the exponent, its reciprocal finite whatever lies in a place that no row sees
            const float v = vs[x][e];
            s[x][e] = __builtin_fmaf(s[x][e], kscale[x][e], __builtin_amdgcn_logf(v));
            inv_v[x][e] = v >= PAGED_TINY && v < INFINITY ? __builtin_amdgcn_rcpf(v) : 1.0f;
          }
      }
      // value e of s[x] is key 4 lq + e of this lane's group
      const bool masked = (at.id[0] | at.id[1] | at.id[2] | at.id[3]) < 0 || max(max(at.key[0], at.key[1]), max(at.key[2], at.key[3])) + 15 > pos;
      if (masked)
#pragma unroll
        for (int x = 0; x < A; x++) {
          const int seen = pos - mine(at.key[0], at.key[1], at.key[2], at.key[3], x) - 4 * lq, id = mine(at.id[0], at.id[1], at.id[2], at.id[3], x);
#pragma unroll
          for (int e = 0; e < 4; e++) s[x][e] = id >= 0 && e <= seen ? s[x][e] : -INFINITY;
        }
      if (A == 1 && a.heads_log < 2)                         // more groups of columns than of keys
#pragma unroll
        for (int e = 0; e < 4; e++) s[0][e] = cg < 4 ? s[0][e] : -INFINITY;
      float mx = m_run;
#pragma unroll
      for (int x = 0; x < A; x++) mx = fmaxf(fmaxf(fmaxf(mx, s[x][0]), fmaxf(s[x][1], s[x][2])), s[x][3]);
      mx = max_xor32(max_xor16(mx));
      if (__builtin_amdgcn_ballot_w64(mx > m_run)) {
        const float alpha = __builtin_amdgcn_exp2f((m_run - mx) * unit);
        m_run = mx;
        l_run *= alpha;
#pragma unroll
        for (int t = 0; t < NT; t++) o[t] *= alpha;
      }
      uint32_t pk[A][2];
#pragma unroll
      for (int x = 0; x < A; x++) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          // the difference first: it is never above zero, however large the scores are
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e] - m_run, unit, PA_TOP));
          l_run = I8 ? __builtin_fmaf(p[e], inv_v[x][e], l_run) : l_run + p[e];
        }
#pragma unroll
        for (int e = 0; e < 2; e++) pk[x][e] = __builtin_bit_cast(uint32_t, h2_t{(_Float16)p[2 * e], (_Float16)p[2 * e + 1]});
      }
#pragma unroll
      for (int u = 0; u < 2; u++) {                          // 32 keys: groups 2 u and 2 u + 1
        store_rows(vr[2 * u], 0, VROW);
        store_rows(vr[2 * u + 1], 1, VROW);
        if constexpr (MORE) {
          load_v(next, u);
          if (u == 1) load_vs(next);
        }
        u4_t pw;                                             // this column's weights, zero at the other groups' keys
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int x = A == 1 ? 0 : A == 2 ? u : 2 * u + h;
          const bool own = A == 4 || cg == (A == 1 ? 2 * u + h : h);
#pragma unroll
          for (int e = 0; e < 2; e++) pw[2 * h + e] = own ? pk[x][e] : 0;
        }
        const h8_t pf = __builtin_bit_cast(h8_t, pw);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          s4_t v[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int row = 16 * h + 4 * lq + (l16 >> 2), c = t * 32 + (l16 & 3) * 8;
            v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t *)(vl + row * VROW + c));
          }
          u4_t w = __builtin_bit_cast(u4_t, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
          if constexpr (CAREFUL) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t x = ((w[e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;   // the sign bit of halves that are not finite
              w[e] &= ~(x | (x - (x >> 15)));
            }
          }
          o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, w), pf, o[t], 0, 0, 0);
        }
        if constexpr (CAREFUL) {
          // those are left out of the product, where a weight of zero would not stop them, and added once for each head that sees them
          for (int key = 0; key < 32; key++) {
            const bool upper = key >= 16;
            const int id = upper ? at.id[2 * u + 1] : at.id[2 * u], first = upper ? at.key[2 * u + 1] : at.key[2 * u];
            const bool seen = id >= 0 && first + (key & 15) <= pos && (A == 4 || cg == (A == 1 ? 2 * u : 0) + upper);
#pragma unroll
            for (int t = 0; t < NT; t++) {
              const uint2 w = *(const uint2 *)(vl + key * VROW + t * 32 + 8 * lq);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t x = (e < 2 ? w.x : w.y) >> (16 * (e & 1)) & 0xffffu;
                o[t][e] += seen && (x & 0x7c00u) == 0x7c00u ? (float)__builtin_bit_cast(_Float16, (uint16_t)x) : 0.0f;
              }
            }
          }
        }
      }
      at = next;
    };
    auto walk = [&](auto careful) {
#pragma unroll
      for (int t = 0; t < NT; t++) o[t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
      m_run = -1e30f;                                        // finite: a step may hold no key that a column sees
      l_run = 0.0f;
      st = st_lo + (SOLO ? 0 : wave);
      find(st, at);
      if (st >= st_end) return;
      load_k(at);
      load_v(at, 0);
      load_v(at, 1);
      load_vs(at);
      // the last step by itself: behind a branch around its loads every wait would be for all of them
      for (; st + ROW_WAVES < st_end; st += ROW_WAVES) step(std::true_type(), careful);
      step(std::false_type(), careful);
    };
    walk(std::false_type());
    if constexpr (!I8) {
      // Halves of V that are not finite make sums so that are not finite, also where their weight is zero.  It is seen here, and then the walk is made once more with a look at every half: that look in
      // every walk is a quarter of the vector unit's work.
      bool bad = false;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) bad |= !(fabsf(o[t][e]) < INFINITY);
      if (__builtin_amdgcn_ballot_w64(bad)) walk(std::true_type());
    }

    // the block's wavefronts and columns: value e of o[t] is feature 16 t + 4 lq + e of column l16
    l_run = add_xor32(add_xor16(l_run));
#pragma unroll
    for (int t = 0; t < NT; t++) *(f4_t *)&sm.wave[wave].o[l16 * OROW + t * 16 + 4 * lq] = o[t];
    if (lq == 0) { sm.m[wave][l16] = m_run; sm.l[wave][l16] = l_run; }
    if constexpr (SOLO) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // of this wavefront, in order
    else lds_barrier();
    constexpr int GROUPS = 4 / A;                            // columns of a head
    auto block_sum = [&](int h, int c, f4_t &sum, float &M, float &L) {   // features 4 c .. of head h
      M = -1e30f;
#pragma unroll
      for (int w = 0; w < ROW_WAVES; w++)
#pragma unroll
        for (int j = 0; j < GROUPS; j++) M = fmaxf(M, sm.m[SOLO ? wave : w][j * hp + h]);
      sum = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
      L = 0.0f;
#pragma unroll
      for (int w0 = 0; w0 < ROW_WAVES; w0++)
#pragma unroll
        for (int j = 0; j < GROUPS; j++) {
          const int col = j * hp + h, w = SOLO ? wave : w0;
          const float e = __builtin_amdgcn_exp2f((sm.m[w][col] - M) * unit);
          L = __builtin_fmaf(sm.l[w][col], e, L);
          const f4_t v = *(const f4_t *)&sm.wave[w].o[col * OROW + 4 * c];
#pragma unroll
          for (int x = 0; x < 4; x++) sum[x] = __builtin_fmaf(v[x], e, sum[x]);
        }
    };
    auto put = [&](int h, int c, f4_t sum, float inv) {
      const h2_t lo = {(_Float16)(sum[0] * inv), (_Float16)(sum[1] * inv)}, hi = {(_Float16)(sum[2] * inv), (_Float16)(sum[3] * inv)};
      *(uint2 *)(a.out + q_off + (size_t)h * HD + 4 * c) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    };
    const int pieces = nr * (HD / 4);
    if (SOLO || a.parts == 1) {
      for (int i = tid; i < pieces; i += ROW_THREADS) {
        f4_t sum;
        float M, L;
        block_sum(i / (HD / 4), i % (HD / 4), sum, M, L);
        put(i / (HD / 4), i % (HD / 4), sum, L == 0.0f ? 0.0f : 1.0f / L);   // 0: the row sees nothing
      }
      return;
    }
    if constexpr (!SOLO) join(a, r, g, qt, part, pieces, nr, unit, block_sum, put, sm);
  }

  template <typename Sum, typename Put>
  static __device__ void join(const SelectedArgs &a, int r, int g, int qt, int part, int pieces, int nr, float unit, Sum block_sum, Put put, Smem &sm) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), KV = (int)a.n_kv_heads.d;
    // Parts: sums through memory at device scope (cache policy 16), counted once they are acknowledged; the last block of the row and heads folds them in order.
    const int slot = (r * a.q_tiles + qt) * a.parts * KV + g;
    const uint32_t part_bytes = (uint32_t)KV * SLOT * 4;
    const __amdgpu_buffer_rsrc_t rw = wave_buffer(a.ws + (size_t)slot * SLOT, (uint32_t)(a.parts - 1) * part_bytes + SLOT * 4);
    for (int i = tid; i < pieces; i += PA_THREADS) {
      f4_t sum;
      float M, L;
      const int h = i / (HD / 4), c = i % (HD / 4);
      block_sum(h, c, sum, M, L);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, sum), rw, (uint32_t)part * part_bytes + i * 16, 0, 16);
      if (c == 0) {
        const f4_t ml = {M, L, 0.0f, 0.0f};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, ml), rw, (uint32_t)part * part_bytes + (PA_QROWS * HD + h * 4) * 4, 0, 16);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) sm.is_last = __hip_atomic_fetch_add(&a.counters[slot], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.parts - 1;
    __syncthreads();
    if (!sm.is_last) return;
    if (tid == 0) __hip_atomic_store(&a.counters[slot], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
    // weights of the parts: a wavefront per head, a part per lane
    for (int h = wave; h < nr; h += NW) {
      const f4_t ml = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)min(lane, a.parts - 1) * part_bytes + (PA_QROWS * HD + h * 4) * 4, 0, 16));
      const float m = lane < a.parts ? ml[0] : -1e30f, M = wave_max(m), e = lane < a.parts ? __builtin_amdgcn_exp2f((m - M) * unit) : 0.0f;
      const float L = wave_sum(lane < a.parts ? ml[1] * e : 0.0f);
      sm.w[h][lane] = e;
      if (lane == 0) sm.inv[h] = L == 0.0f ? 0.0f : 1.0f / L;
    }
    lds_barrier();
    // a thread per four features of a head; where those are fewer than threads, teams of threads share the parts
    const int teams = pieces < PA_THREADS ? PA_THREADS / pieces : 1, team = teams > 1 ? tid / pieces : 0;
    for (int i0 = teams > 1 ? tid - team * pieces : tid; i0 < pieces; i0 += PA_THREADS) {
      const int h = i0 / (HD / 4), c = i0 % (HD / 4);
      f4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
      if (team < teams)
        for (int f = team; f < a.parts; f += teams * 8) {
          f4_t v[8];
#pragma unroll
          for (int u = 0; u < 8; u++)
            v[u] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)min(f + u * teams, a.parts - 1) * part_bytes + i0 * 16, 0, 16));
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (f + u * teams < a.parts)
#pragma unroll
              for (int x = 0; x < 4; x++) sum[x] = __builtin_fmaf(v[u][x], sm.w[h][f + u * teams], sum[x]);
        }
      if (teams == 1) put(h, c, sum, sm.inv[h]);
      else sm.fold[tid] = sum;
    }
    if (teams > 1) {
      lds_barrier();
      if (tid < pieces) {
        f4_t sum = sm.fold[tid];
        for (int u = 1; u < teams; u++) sum += sm.fold[tid + u * pieces];
        put(tid / (HD / 4), tid % (HD / 4), sum, sm.inv[tid / (HD / 4)]);
      }
    }
  }
};

// Block numbers have the kv heads innermost: blocks are dealt to the eight XCDs in turn, so that with eight kv heads each XCD has one, all rows of which share its K and V in that L2.
template <int HD, bool I8, int A, bool SOLO> __global__ __launch_bounds__(PA_THREADS, HD == 64 ? (I8 || A > 1 ? 3 : 4) : 2) void attn_selected_kernel(SelectedArgs a) {
  typedef SelectedRow<HD, I8, A, SOLO> Row;
  __shared__ typename Row::Smem sm;
  const int id = blockIdx.x, KV = (int)a.n_kv_heads.d, rest = a.n_kv_heads.div(id), g = id - rest * KV;
  int part = 0, tile = rest;
  if constexpr (SOLO) {
    tile = rest * Row::NW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  } else {
    tile = rest / a.parts;
    part = rest - tile * a.parts;
  }
  const int r = tile / a.q_tiles, qt = tile - r * a.q_tiles;
  if (r >= a.pb.rows) return;
  // the row's first pages are asked for beside its sequence
  const int first = SOLO ? threadIdx.x & 63 : threadIdx.x, chosen = first < a.top ? a.selected[((size_t)r * KV + g) * a.top + first] : -1;
  PagedSeq s;
  const int b = find_row(a.pb, r, s);
  if (b >= a.pb.n_seqs || r < s.start) return;
  Row::run(a, r, g, qt, part, b, paged_pos(s, r - s.start), chosen, sm);
}

// Argument checks that the calls here share
static int bounds_check(const char *who, const void *bounds, const float *bound_scales) {
  JSG_REQUIRE(bounds && bound_scales, "%s: null pointer argument", who);
  JSG_REQUIRE((uintptr_t)bounds % 16 == 0 && (uintptr_t)bound_scales % 4 == 0, "%s: bounds must be 16-byte aligned, their scales 4-byte", who);
  return 0;
}
static int heads_check(const char *who, const jsgrad_hip_pages_t *pg, const void *q, int rows, int n_heads) {
  JSG_REQUIRE(q, "%s: null pointer argument", who);
  JSG_REQUIRE((uintptr_t)q % 16 == 0, "%s: q must be 16-byte aligned", who);
  JSG_REQUIRE(n_heads > 0 && n_heads <= 65535 && n_heads % pg->n_kv_heads == 0, "%s: n_heads %d / n_kv_heads %d", who, n_heads, pg->n_kv_heads);
  JSG_REQUIRE((size_t)rows * n_heads < (size_t)1 << 30, "%s: %d rows of %d heads", who, rows, n_heads);
  return 0;
}

}  // namespace jsg

using namespace jsg;

extern "C" {

int jsgrad_hip_paged_bounds(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, int8_t *bounds, float *bound_scales) {
  const char *who = "jsgrad_hip_paged_bounds";
  PagedSelectArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  if (int e = bounds_check(who, bounds, bound_scales)) return e;
  JSG_READY();
  a.pages_k = host_pages->pages_k;
  a.scales_k = (const float *)host_pages->scales_k;
  a.bounds = bounds; a.bound_scales = bound_scales;
  a.n_kv_heads = host_pages->n_kv_heads;
  // a sequence's rows begin and end inside pages
  const dim3 grid((unsigned)(rows / host_pages->page_size + 2 * (n_seqs < rows ? n_seqs : rows)), (unsigned)a.n_kv_heads), block(PS_THREADS);
  const bool i8 = host_pages->kind == JSGRAD_W_I8;
  if (host_pages->head_dim == 64 && i8) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_bounds_kernel<64, true>), grid, block, 0, a);
  else if (host_pages->head_dim == 64) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_bounds_kernel<64, false>), grid, block, 0, a);
  else if (i8) JSG_LAUNCH(PROF_PAGED_ROWS, (paged_bounds_kernel<128, true>), grid, block, 0, a);
  else JSG_LAUNCH(PROF_PAGED_ROWS, (paged_bounds_kernel<128, false>), grid, block, 0, a);
  return 0;
}

int jsgrad_hip_paged_select(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, const void *q, int n_heads,
                            const int8_t *bounds, const float *bound_scales, int first, int recent, int top, int32_t *selected) {
  const char *who = "jsgrad_hip_paged_select";
  PagedSelectArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  if (int e = bounds_check(who, bounds, bound_scales)) return e;
  if (int e = heads_check(who, host_pages, q, rows, n_heads)) return e;
  JSG_REQUIRE(selected && (uintptr_t)selected % 4 == 0, "%s: selected must be 4-byte aligned, and not null", who);
  JSG_REQUIRE(first >= 0 && recent >= 1 && top >= 1 && top <= PS_MOST && first <= top - recent, "%s: first %d and recent %d of %d pages (1 to %d, the row's own page among the recent ones)", who, first, recent, top, PS_MOST);
  JSG_REQUIRE(host_pages->table_width <= PS_WIDTH, "%s: table_width %d (at most %d)", who, host_pages->table_width, PS_WIDTH);
  const int HD = host_pages->head_dim, n_rep = n_heads / host_pages->n_kv_heads;
  JSG_REQUIRE(n_rep <= 64, "%s: %d query heads to a kv head (at most 64)", who, n_rep);
  JSG_READY();
  a.q = (const _Float16 *)q;
  a.bounds = (int8_t *)bounds; a.bound_scales = (float *)bound_scales;
  a.n_kv_heads = host_pages->n_kv_heads; a.n_rep = n_rep;
  a.first = first; a.recent = recent; a.top = top;
  a.selected = selected;
  while ((1 << a.heads_log) < (n_rep < 16 ? n_rep : 16)) a.heads_log++;
  a.stride = (host_pages->table_width + 15) & ~15;
  // Rows of a sequence share its bounds: the columns of a matrix instruction are theirs, and with heads of 128 four such tiles where enough blocks are left.  us, one tile | four: 2048 rows behind 14336, 16 heads of
  // 128 over 1 23 | 15, 16 over 2 20 | 17, 64 over 8 70 | 60, 32 over 8 39 | 37.5, 1024 of these behind 15360 22 | 20, 700 behind 9000 14 | 18, 256 behind 16128 8 | 16.  Heads of 64, whose bounds are half as
  // long: 2048 behind 14336 31 | 29, behind 2048 21 | 23, 4096 from the start 35 | 38 (with the bounds straight to the operand).
  const bool many = n_rep > 16;
  const int tile = 16 >> a.heads_log;
  const bool four = HD == 128 && !many && (size_t)rows >= (size_t)8 * tile * n_seqs && (size_t)rows * a.n_kv_heads >= (size_t)tile * 2048 && (size_t)tile * 4 * a.stride * 4 <= 64 * 1024;
  a.tile = rows > n_seqs && (size_t)tile * a.stride * 4 <= 64 * 1024 ? tile * (four ? 4 : 1) : 1;
  const dim3 grid((unsigned)((rows + a.tile - 1) / a.tile), (unsigned)a.n_kv_heads);
  // Eight wavefronts where a unit has no more than one block.  us, four | eight: one row behind 33000 positions, pages of 64, 9.6 | 8.4, of 16 24 | 17.5; 16 rows of up to 32768, pages of 32, 13.2 | 11.3; 128
  // rows behind 16256 (256 blocks) 7.2 | 7.1; with more blocks, 64 rows of 64 sequences of 8192 7.6 | 9.9, 512 behind 15872 14.4 | 15.
  const size_t lds = (size_t)a.tile * a.stride * 4;
  const bool wide = !many && !four && (size_t)grid.x * grid.y <= 256 && lds <= 64 * 1024;   // the tiles of eight have 34 KB of LDS
#define JSG_SELECT(HD, NW, HT, HEADS)                                                                                                                                        \
  do {                                                                                                                                                                        \
    if (lds > 48 * 1024) JSG_HIP(hipFuncSetAttribute((const void *)paged_select_kernel<HD, NW, HT, HEADS>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));              \
    JSG_LAUNCH(PROF_ATTN_PAGED, (paged_select_kernel<HD, NW, HT, HEADS>), grid, dim3(NW * 64), lds, a);                                                                          \
  } while (0)
  if (HD == 64 && many) JSG_SELECT(64, 4, 4, true);
  else if (HD == 64 && wide) JSG_SELECT(64, 8, 1, false);
  else if (HD == 64) JSG_SELECT(64, 4, 1, false);
  else if (many) JSG_SELECT(128, 4, 4, true);
  else if (wide) JSG_SELECT(128, 8, 1, false);
  else if (a.tile > tile) JSG_SELECT(128, 4, 4, false);
  else JSG_SELECT(128, 4, 1, false);
#undef JSG_SELECT
  return 0;
}

size_t jsgrad_hip_attn_selected_workspace_bytes(int n_heads, int n_kv_heads, int head_dim) {
  (void)n_heads, (void)n_kv_heads;
  return PA_SLOTS * sizeof(int) + (size_t)PA_SLOTS * PA_QROWS * (head_dim + 4) * sizeof(float);
}

int jsgrad_hip_attn_selected(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, const void *q, void *out, int n_heads,
                             const int32_t *selected, int top, void *workspace) {
  const char *who = "jsgrad_hip_attn_selected";
  SelectedArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  if (int e = heads_check(who, host_pages, q, rows, n_heads)) return e;
  JSG_REQUIRE(out && selected && workspace, "%s: null pointer argument", who);
  JSG_REQUIRE((uintptr_t)out % 16 == 0 && (uintptr_t)workspace % 16 == 0 && (uintptr_t)selected % 4 == 0, "%s: out and workspace must be 16-byte aligned, selected 4-byte", who);
  JSG_REQUIRE(q != out, "%s: out must not be q", who);
  JSG_REQUIRE(top >= 1 && top <= PS_MOST, "%s: %d pages to a row (1 to %d)", who, top, PS_MOST);
  const int KV = host_pages->n_kv_heads, HD = host_pages->head_dim, n_rep = n_heads / KV;
  a.pages_k = host_pages->pages_k; a.pages_v = host_pages->pages_v;
  a.scales_k = (const float *)host_pages->scales_k; a.scales_v = (const float *)host_pages->scales_v;
  a.q = (const _Float16 *)q; a.out = (_Float16 *)out;
  a.n_heads = n_heads; a.n_rep = n_rep;
  while ((1 << a.heads_log) < (n_rep < PA_QROWS ? n_rep : PA_QROWS)) a.heads_log++;
  a.n_kv_heads = divisor(KV);
  a.scale_log2 = (float)(1.0 / sqrt((double)HD)) * 1.4426950408889634f;
  a.counters = (int *)workspace;
  a.ws = (float *)((char *)workspace + PA_SLOTS * sizeof(int));
  a.selected = selected; a.top = top;
  a.q_tiles = (n_rep + PA_QROWS - 1) / PA_QROWS;
  const size_t items = (size_t)rows * a.q_tiles * KV;
  JSG_REQUIRE(items < (size_t)PAGED_GRID, "%s: %d rows of %d heads", who, rows, n_heads);
  // Parts of a row where there are few: two blocks to a unit, each wavefront with one step at least.  us, 256 | 512 | 1024 blocks: one row, 32 pages of 64, 9.3 | 9.5 | 9.4; 16 rows of 64 pages fp16 44 | 46 | 47, int8 31 | 31 | -;
  // with 128 these take 9.4, 44 and 48.
  const int steps = (int)(((size_t)(top < a.pb.width ? top : a.pb.width) << a.pb.page_shift) / 64);
  int parts = items * 2 <= PA_BLOCKS ? (int)(PA_BLOCKS / items) : 1;
  parts = parts < PA_MOST ? parts : PA_MOST;
  parts = parts < steps / 4 ? parts : steps / 4;
  a.parts = parts > 1 ? parts : 1;
  JSG_READY();
  // A row to a wavefront where each has one and the chip is full.  us, a row to a block | to a wavefront, 16 pages of 64 for each of n rows, 32 heads over 8: heads of 64 fp16 n = 128 18 | 24, 256 32 | 32, 512
  // 58 | 52, 1024 110 | 96, int8 256 37 | 41, 512 69 | 63; heads of 128 fp16 128 33 | 35, 256 61 | 54, 1024 228 | 193, int8 256 74 | 67, 1024 280 | 238.
  const bool solo = a.parts == 1 && top <= 64 && items * HD >= (size_t)4096 * 64;
  const dim3 grid((unsigned)(solo ? ((size_t)rows * a.q_tiles + 3) / 4 * KV : items * a.parts)), block(PA_THREADS);
  const bool i8 = host_pages->kind == JSGRAD_W_I8;
#define JSG_SELECTED_A(HD, I8, A)                                                                            \
  do {                                                                                                       \
    if (solo) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_selected_kernel<HD, I8, A, true>), grid, block, 0, a);         \
    else JSG_LAUNCH(PROF_ATTN_PAGED, (attn_selected_kernel<HD, I8, A, false>), grid, block, 0, a);             \
  } while (0)
#define JSG_SELECTED(HD, I8)                              \
  do {                                                    \
    if (a.heads_log <= 2) JSG_SELECTED_A(HD, I8, 1);        \
    else if (a.heads_log == 3) JSG_SELECTED_A(HD, I8, 2);   \
    else JSG_SELECTED_A(HD, I8, 4);                         \
  } while (0)
  if (HD == 64 && i8) JSG_SELECTED(64, true);
  else if (HD == 64) JSG_SELECTED(64, false);
  else if (i8) JSG_SELECTED(128, true);
  else JSG_SELECTED(128, false);
#undef JSG_SELECTED
#undef JSG_SELECTED_A
  return 0;
}

}  // extern "C"
