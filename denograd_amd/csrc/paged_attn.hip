// Grouped-query attention of a ragged batch of new rows over a paged KV cache (jsgrad_hip_attn_paged).
//
// Row i of a sequence sits at position p and sees the keys j <= p that have a page and, with a window, are among the last `window` of them or
// among the first `sinks`: out = sum_j softmax_j(q . K_j / sqrt(HD)) V_j, zeros where it sees none.  Reference semantics of the sum:
// scaled_dot_product_attention (/root/reference/jsgrad/tensor.ts:3920-3934); windows, sinks and pages have no counterpart there.
#include "gemm.h"
#include "paged.h"

namespace jsg {

int paged_check(const char *who, const jsgrad_hip_pages_t *pg, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, PagedBatch *pb);   // paged.hip

struct PagedAttnArgs {
  PagedBatch pb;
  const void *pages_k, *pages_v;
  const float *scales_k, *scales_v;
  const _Float16 *q;                     // [rows][H][HD]
  _Float16 *out;
  int n_heads, n_kv_heads, window, sinks;
  float scale_log2;                      // float(1 / sqrt(HD)) * log2(e)
};

// One wavefront per (row, query head): 64 keys at a time, a lane's score each, then their weighted V rows with a lane's features each.
template <int HD, bool I8> __global__ __launch_bounds__(64) void attn_paged_kernel(PagedAttnArgs a) {
  constexpr int F = HD / 64;
  const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, g = h / (a.n_heads / a.n_kv_heads);
  int b = 0;
  while (b < a.pb.n_seqs && a.pb.row_starts[b + 1] <= r) b++;
  if (b >= a.pb.n_seqs) return;
  const PagedSeq s = paged_seq(a.pb, b);
  if (r < s.start) return;
  const int p = paged_pos(s, r - s.start), top = min(p, paged_room(a.pb) - 1);
  const size_t at = ((size_t)r * a.n_heads + h) * HD;
  float m = -INFINITY, l = 0.0f, o[F];
#pragma unroll
  for (int f = 0; f < F; f++) o[f] = 0.0f;
  for (int j0 = 0; j0 <= top; j0 += 64) {
    const int j = j0 + lane;
    const int id = j <= top && (a.window == 0 || j > p - a.window || j < a.sinks) ? paged_page(a.pb, b, j) : -1;
    const size_t row = id >= 0 ? paged_row(a.pb, a.n_kv_heads, id, g, j) : 0;
    float x = -INFINITY;
    if (id >= 0) {
      float sum = 0.0f;
      for (int e = 0; e < HD; e++) {
        const float kv = I8 ? (float)((const int8_t *)a.pages_k)[row * HD + e] : (float)((const _Float16 *)a.pages_k)[row * HD + e];
        sum = fmaf((float)a.q[at + e], kv, sum);
      }
      x = sum * a.scale_log2 * (I8 ? a.scales_k[row] : 1.0f);
    }
    const float mx = fmaxf(m, wave_max(x));
    if (mx == -INFINITY && __builtin_amdgcn_ballot_w64(id >= 0) == 0) continue;
    const float w = id >= 0 ? __builtin_amdgcn_exp2f(x - mx) : 0.0f, f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
    m = mx;
    l = l * f0 + wave_sum(w);
#pragma unroll
    for (int f = 0; f < F; f++) o[f] *= f0;
    for (int u = 0; u < 64; u++) {
      if (__builtin_amdgcn_readlane(id, u) < 0) continue;
      const float wu = readlane_f(w, u);
      const size_t ru = ((size_t)(uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), u) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)row, u);
#pragma unroll
      for (int f = 0; f < F; f++) {
        const size_t e = ru * HD + f * 64 + lane;
        o[f] = fmaf(wu, I8 ? (float)((const int8_t *)a.pages_v)[e] * a.scales_v[ru] : (float)((const _Float16 *)a.pages_v)[e], o[f]);
      }
    }
  }
#pragma unroll
  for (int f = 0; f < F; f++) a.out[at + f * 64 + lane] = (_Float16)(l == 0.0f ? 0.0f : o[f] / l);
}

}  // namespace jsg

using namespace jsg;

extern "C" {

size_t jsgrad_hip_attn_paged_workspace_bytes(int n_heads, int n_kv_heads, int head_dim) {
  (void)n_heads, (void)n_kv_heads, (void)head_dim;
  return 256;
}

int jsgrad_hip_attn_paged(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, const void *q, void *out,
                          int n_heads, int window, int sinks, void *workspace) {
  const char *who = "jsgrad_hip_attn_paged";
  PagedAttnArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  JSG_REQUIRE(q && out && workspace, "%s: null pointer argument", who);
  JSG_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)workspace % 16 == 0, "%s: q, out and workspace must be 16-byte aligned", who);
  JSG_REQUIRE(q != out, "%s: out must not be q", who);
  JSG_REQUIRE(n_heads > 0 && n_heads <= 65535 && n_heads % host_pages->n_kv_heads == 0, "%s: n_heads %d / n_kv_heads %d", who, n_heads, host_pages->n_kv_heads);
  JSG_REQUIRE(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", who, window, sinks);
  JSG_READY();
  a.pages_k = host_pages->pages_k; a.pages_v = host_pages->pages_v;
  a.scales_k = (const float *)host_pages->scales_k; a.scales_v = (const float *)host_pages->scales_v;
  a.q = (const _Float16 *)q; a.out = (_Float16 *)out;
  a.n_heads = n_heads; a.n_kv_heads = host_pages->n_kv_heads;
  a.window = window; a.sinks = sinks;
  a.scale_log2 = (float)(1.0 / sqrt((double)host_pages->head_dim)) * 1.4426950408889634f;
  const dim3 grid(rows, n_heads), block(64);
  const bool i8 = host_pages->kind == JSGRAD_W_I8;
  if (host_pages->head_dim == 64 && i8) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_paged_kernel<64, true>), grid, block, 0, a);
  else if (host_pages->head_dim == 64) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_paged_kernel<64, false>), grid, block, 0, a);
  else if (i8) JSG_LAUNCH(PROF_ATTN_PAGED, (attn_paged_kernel<128, true>), grid, block, 0, a);
  else JSG_LAUNCH(PROF_ATTN_PAGED, (attn_paged_kernel<128, false>), grid, block, 0, a);
  return 0;
}

}  // extern "C"
