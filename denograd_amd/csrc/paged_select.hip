// Attention over pages that every row chooses by a bound of what they hold: the pages' bounds (jsgrad_hip_paged_bounds), the choice (jsgrad_hip_paged_select), and the attention over what was chosen
// (jsgrad_hip_attn_selected).  No counterpart in the reference.
//
// No key of a page scores more with a query than sum_d q_d (q_d > 0 ? hi_d : lo_d), lo and hi being the least and the largest of each feature.  Both are kept as whole numbers, rounded outwards, times one power of
// two per page and head; a row's queries are rounded to whole numbers times one power of two as well.  So scores are whole numbers below 2^21 times a power of two, exact however they are summed, and
// which pages are chosen is a question of the inputs alone: with float sums two scores that are nearly the same would fall either way.
#include "paged_few.h"

namespace jsg {

constexpr int PS_THREADS = 256, PS_MOST = 1024, PS_WIDTH = 32768;      // pages that a row chooses, columns of the table

struct PagedSelectArgs {
  PagedBatch pb;
  const void *pages_k;
  const float *scales_k;
  const _Float16 *q;                     // [rows][H][HD]
  int8_t *bounds;                        // [n_pages][KV][lo, hi][HD]
  float *bound_scales;                   // [n_pages][KV]
  int n_kv_heads, n_rep, first, recent, top;
  int32_t *selected;                     // [rows][KV][top]
};

// The smallest power of two, 2^-126 and more, that 127 times is `most` (finite) and more; 1 for 0.
__device__ __forceinline__ float bound_step(float most) {
  if (most == 0.0f) return 1.0f;
  const int e = __builtin_amdgcn_frexp_expf(most);           // most = f * 2^e, 1/2 <= f < 1
  const float f = __builtin_amdgcn_frexp_mantf(most);
  return __builtin_amdgcn_ldexpf(1.0f, max(e - 7 + (f > 127.0f / 128.0f), -126));
}

// Block = (row, kv head), at work where the row is the first of the batch on its page: the whole page is looked at, so bounds do not depend on how its rows came.
// Bound by memory: HD / 8 lanes a row, 16 bytes (int8: 8) each.
template <int HD, bool I8> __global__ __launch_bounds__(PS_THREADS) void paged_bounds_kernel(PagedSelectArgs a) {
  constexpr int G = HD / 8, RPB = PS_THREADS / G;
  __shared__ float lo_sh[PS_THREADS / 64][HD], hi_sh[PS_THREADS / 64][HD];
  __shared__ float most_sh[PS_THREADS / 64];
  const int r = blockIdx.x, g = blockIdx.y, KV = a.n_kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = paged_find(a.pb, r);
  if (b >= a.pb.n_seqs) return;
  const PagedSeq s = paged_seq(a.pb, b);
  const int pos = paged_pos(s, r - s.start), P = 1 << a.pb.page_shift;
  if (r < s.start || pos < 0 || (r > s.start && pos > 0 && (pos & (P - 1)) != 0)) return;
  const int id = paged_page(a.pb, b, pos);
  if (id < 0) return;
  const int first = pos & ~(P - 1), n = min(P, s.len - first);
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
    to[0] = bad ? 0 : (int8_t)(int)floorf(__fdiv_rn(l, step));
    to[HD] = bad ? 0 : (int8_t)(int)ceilf(__fdiv_rn(h, step));
    if (d == 0) a.bound_scales[(size_t)id * KV + g] = step;
  }
}

// Order of scores as that of whole numbers above 0.
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// Block = (row, kv head).
template <int HD> __global__ __launch_bounds__(PS_THREADS) void paged_select_kernel(PagedSelectArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int r = blockIdx.x, g = blockIdx.y, KV = a.n_kv_heads, n_rep = a.n_rep, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = paged_find(a.pb, r);
  if (b >= a.pb.n_seqs) return;
  const PagedSeq s = paged_seq(a.pb, b);
  const int pos = paged_pos(s, r - s.start);
  if (r < s.start) return;
  int32_t *const out = a.selected + ((size_t)r * KV + g) * a.top;
  const int last = pos < 0 ? -1 : pos >> a.pb.page_shift, n = min(last + 1, a.pb.width);
  // the group's queries as whole numbers: positive parts, then negative ones
  int8_t *const qc = (int8_t *)smem;                         // [n_rep][2][HD]
  uint32_t *const keys = (uint32_t *)(smem + (size_t)n_rep * 2 * HD);
  __shared__ float red[PS_THREADS / 64];
  __shared__ int count[2][PS_THREADS / 64];
  const _Float16 *const q = a.q + ((size_t)r * KV + g) * n_rep * HD;
  float most = 0.0f;
  for (int i = tid; i < n_rep * HD; i += PS_THREADS) {
    const float f = fabsf((float)q[i]);
    most = f < INFINITY ? fmaxf(most, f) : INFINITY;
    if (!(f < INFINITY)) break;
  }
  most = wave_max(most);
  if (lane == 0) red[wave] = most;
  __syncthreads();
  for (int w = 0; w < PS_THREADS / 64; w++) most = fmaxf(most, red[w]);
  const float step = most < INFINITY ? bound_step(most) : 0.0f;   // queries that are not finite say nothing
  for (int i = tid; i < n_rep * HD; i += PS_THREADS) {
    const int c = step > 0.0f ? (int)rintf(__fdiv_rn((float)q[i], step)) : 0, h = i / HD, d = i % HD;
    qc[(h * 2) * HD + d] = (int8_t)max(c, 0);
    qc[(h * 2 + 1) * HD + d] = (int8_t)min(c, 0);
  }
  __syncthreads();
  for (int i = tid; i < n; i += PS_THREADS) {
    const int id = paged_page(a.pb, b, i << a.pb.page_shift);
    uint32_t key = 0;                                        // no page
    if (id >= 0) {
      if (i < a.first || i > last - a.recent) {
        key = 0xffffffffu;
      } else {
        const int *const lo = (const int *)(a.bounds + ((size_t)id * KV + g) * 2 * HD), *const hi = lo + HD / 4;
        int best = -0x7fffffff;
        for (int h = 0; h < n_rep; h++) {
          const int *const up = (const int *)(qc + h * 2 * HD), *const down = up + HD / 4;
          int sum = 0;
          for (int d = 0; d < HD / 4; d++) sum = __builtin_amdgcn_sdot4(hi[d], up[d], __builtin_amdgcn_sdot4(lo[d], down[d], sum, false), false);
          best = max(best, sum);
        }
        const float scale = a.bound_scales[(size_t)id * KV + g];
        key = min(score_key(scale < INFINITY ? (float)best * scale : INFINITY), 0xfffffffeu);
      }
    }
    keys[i] = key;
  }
  __syncthreads();
  auto block_count = [&](int mine, int turn) {               // over the block; `turn` alternates
    const int c = (int)wave_sum((float)mine);
    if (lane == 0) count[turn][wave] = c;
    __syncthreads();
    return count[turn][0] + count[turn][1] + count[turn][2] + count[turn][3];
  };
  // the largest threshold that `top` keys reach; 1 where there are fewer
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const uint32_t up = t | 1u << bit;
    int mine = 0;
    for (int i = tid; i < n; i += PS_THREADS) mine += keys[i] >= up;
    if (block_count(mine, bit & 1) >= a.top) t = up;
  }
  int more = 0;
  for (int i = tid; i < n; i += PS_THREADS) more += keys[i] > t;
  more = block_count(more, 1);
  int ties = t ? a.top - more : 0, at = 0;                   // of the keys at the threshold, the first so many
  __syncthreads();
  // in the order of the pages, 256 at a time
  for (int i0 = 0; i0 < n; i0 += PS_THREADS) {
    const int i = i0 + tid;
    const uint32_t key = i < n ? keys[i] : 0;
    const bool tie = key == t && key;
    const uint64_t tied = __builtin_amdgcn_ballot_w64(tie), above = (uint64_t)1 << lane;
    if (lane == 0) count[0][wave] = __popcll(tied);
    __syncthreads();
    int before = __popcll(tied & (above - 1)), all = 0;
    for (int w = 0; w < PS_THREADS / 64; w++) {
      if (w < wave) before += count[0][w];
      all += count[0][w];
    }
    const bool take = key > t || (tie && before < ties);
    ties -= min(ties, all);
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    if (lane == 0) count[1][wave] = __popcll(taken);
    __syncthreads();
    int place = at + __popcll(taken & (above - 1));
    for (int w = 0; w < PS_THREADS / 64; w++) {
      if (w < wave) place += count[1][w];
      at += count[1][w];
    }
    if (take && place < a.top) out[place] = i;
  }
  for (int i = at + tid; i < a.top; i += PS_THREADS) out[i] = -1;
}

// ---------------------------------------------------------------- attention over the chosen pages

struct SelectedArgs {
  PagedAttnArgs at;
  const int32_t *selected;               // [rows][KV][top]
  int top, parts, q_tiles;
};

// The keys of chosen pages: a list of {page, first position} in LDS.
struct SelectedKeys {
  const int2 *list;
  __device__ void find(const PagedBatch &pb, int st, FewStep &s) const {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int at = st * 32 + 16 * h;
      const int2 e = list[at >> pb.page_shift];
      s.id[h] = __builtin_amdgcn_readfirstlane(e.x);
      s.key[h] = __builtin_amdgcn_readfirstlane(e.y) + (at & ((1 << pb.page_shift) - 1));
    }
  }
  __device__ bool masks(const int (&k)[2], int pos_lo, int) const { return max(k[0], k[1]) + 15 > pos_lo; }
  __device__ bool sees(int key, int pos) const { return key <= pos; }
};

// Block = 16 of a row's query heads of one kv head, and a part of the row's chosen pages: PagedFew's work on one position.
constexpr int PA_SLOTS = 1024, PA_BLOCKS = 512;
template <int HD, bool I8> __global__ __launch_bounds__(FEW_THREADS, HD == 64 ? 4 : I8 ? 3 : 2) void attn_selected_kernel(SelectedArgs sa) {
  typedef PagedFew<HD, I8> A;
  __shared__ typename A::Smem sm;
  __shared__ int2 list[PS_MOST + 1];
  const PagedAttnArgs &a = sa.at;
  const int KV = (int)a.n_kv_heads.d;
  int id = blockIdx.x;
  PagedItem it;
  it.g = id % KV;
  id /= KV;
  it.part = id % sa.parts;
  id /= sa.parts;
  it.qt = id % sa.q_tiles;
  const int r = id / sa.q_tiles, b = paged_find(a.pb, r);
  if (b >= a.pb.n_seqs) return;
  const PagedSeq s = paged_seq(a.pb, b);
  if (r < s.start) return;
  const int pos = paged_pos(s, r - s.start);
  it.b = b;
  it.s = {r, 1, pos + 1};                                    // the one row, at its position
  it.parts = sa.parts;
  it.slot = (r * sa.q_tiles + it.qt) * sa.parts * KV + it.g;
  const int32_t *const sel = sa.selected + ((size_t)r * KV + it.g) * sa.top;
  const int last = pos < 0 ? -1 : pos >> a.pb.page_shift;
  int n = 0;                                                 // behind the last entry that names a page
  for (int i = threadIdx.x; i <= sa.top; i += FEW_THREADS) {
    const int page = i < sa.top ? sel[i] : -1, held = page >= 0 && page <= last && page < a.pb.width ? paged_page(a.pb, b, page << a.pb.page_shift) : -1;
    list[i] = make_int2(held, held >= 0 ? page << a.pb.page_shift : 0);
    if (held >= 0) n = i + 1;
  }
  for (int d = 32; d > 0; d >>= 1) n = max(n, __shfl_xor(n, d));
  __shared__ int most[FEW_THREADS / 64];
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = n;
  __syncthreads();
  n = max(max(most[0], most[1]), max(most[2], most[3]));
  const int steps = ((n << a.pb.page_shift) + 31) / 32, per = (steps + sa.parts - 1) / sa.parts, lo = min(it.part * per, steps);
  A::walk(a, it, SelectedKeys{list}, lo, min(lo + per, steps), sm);
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
  const dim3 grid((unsigned)rows, (unsigned)a.n_kv_heads), block(PS_THREADS);
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
  const dim3 grid((unsigned)rows, (unsigned)a.n_kv_heads), block(PS_THREADS);
  const size_t lds = (size_t)n_rep * 2 * HD + (size_t)host_pages->table_width * 4;
  if (HD == 64) {
    if (lds > 64 * 1024) JSG_HIP(hipFuncSetAttribute((const void *)paged_select_kernel<64>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    JSG_LAUNCH(PROF_ATTN_PAGED, paged_select_kernel<64>, grid, block, lds, a);
  } else {
    if (lds > 64 * 1024) JSG_HIP(hipFuncSetAttribute((const void *)paged_select_kernel<128>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    JSG_LAUNCH(PROF_ATTN_PAGED, paged_select_kernel<128>, grid, block, lds, a);
  }
  return 0;
}

size_t jsgrad_hip_attn_selected_workspace_bytes(int n_heads, int n_kv_heads, int head_dim) {
  (void)n_heads, (void)n_kv_heads;
  return PA_SLOTS * sizeof(int) + (size_t)PA_SLOTS * FEW_QROWS * (head_dim + 4) * sizeof(float);
}

int jsgrad_hip_attn_selected(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, const void *q, void *out, int n_heads,
                             const int32_t *selected, int top, void *workspace) {
  const char *who = "jsgrad_hip_attn_selected";
  SelectedArgs sa = {};
  PagedAttnArgs &a = sa.at;
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
  a.n_heads = n_heads;
  a.n_rep = divisor(n_rep); a.n_kv_heads = divisor(KV);
  a.scale_log2 = (float)(1.0 / sqrt((double)HD)) * 1.4426950408889634f;
  a.few_counters = (int *)workspace;
  a.few_ws = (float *)((char *)workspace + PA_SLOTS * sizeof(int));
  sa.selected = selected; sa.top = top;
  sa.q_tiles = (n_rep + FEW_QROWS - 1) / FEW_QROWS;
  const size_t items = (size_t)rows * sa.q_tiles * KV;
  JSG_REQUIRE(items < (size_t)PAGED_GRID, "%s: %d rows of %d heads", who, rows, n_heads);
  const int steps = (int)(((size_t)(top < a.pb.width ? top : a.pb.width) << a.pb.page_shift) / 32) + 1;
  int parts = items * 2 <= PA_BLOCKS ? (int)(PA_BLOCKS / items) : 1;
  parts = parts < FEW_MOST ? parts : FEW_MOST;
  parts = parts < steps / 8 ? parts : steps / 8;
  sa.parts = parts > 1 ? parts : 1;
  JSG_READY();
  const dim3 grid((unsigned)(items * sa.parts)), block(FEW_THREADS);
  const bool i8 = host_pages->kind == JSGRAD_W_I8;
  if (HD == 64 && i8) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_selected_kernel<64, true>), grid, block, 0, sa);
  else if (HD == 64) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_selected_kernel<64, false>), grid, block, 0, sa);
  else if (i8) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_selected_kernel<128, true>), grid, block, 0, sa);
  else JSG_LAUNCH(PROF_ATTN_PAGED, (attn_selected_kernel<128, false>), grid, block, 0, sa);
  return 0;
}

}  // extern "C"
