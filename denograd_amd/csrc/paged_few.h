// What the attention kernels of the paged cache share (paged_attn.hip, paged_select.hip): their arguments, and the work of blocks on one or a few rows.
#pragma once
#include <type_traits>

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
  int n_heads, window, sinks;
  Divisor n_rep, n_kv_heads;
  int few_blocks;                        // of the few-row items: what their pairs are shared among
  bool all_few;                          // the launch has blocks enough for few-row items of all its rows
  float scale_log2;                      // float(1 / sqrt(HD)) * log2(e)
  int *counters, *few_counters;          // zero, and zero again afterwards
  float *ws, *few_ws;
};

struct PagedItem {
  PagedSeq s;
  int b, g, qt, part, parts, slot;       // slot: of part 0 in the workspace; part p's is slot + p * n_kv_heads
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

// paged_page for a position that all lanes share: through the scalar cache, sixteen entries to a line, and without a place among the vector loads, whose
// results come in order, so that a page number asked for behind a tile's loads would be there only after the tile is.
__device__ __forceinline__ int page_uniform(const PagedBatch &p, int b, int pos) {
  if (pos < 0 || pos >= paged_room(p)) return -1;
  const int id = *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(p.table + (size_t)b * p.width + (pos >> p.page_shift));
  return id >= 0 && id < p.n_pages ? id : -1;
}

// The scale of V that an int8 row's weight has in the exponent.  The halves are weights times scales relative to the largest of these, so a row whose scale says more than its codes
// would push the others out of fp16's range: one of zero codes, which is written with scale 1 and in a caller's own pages may have any.  It counts with 2^-60, and its weight 2^60 times that in the sum: it
// is the largest only where it outweighs the others by so much that nothing of them is left in an fp16 result.  A scale below 2^-60 counts with that as well: values of 2^-53 and less are
// nothing there either.  A scale that is not a number, or not finite, stays what it is.
constexpr float PAGED_TINY = 0x1p-60f;
__device__ __forceinline__ float scale_of_v(float v, bool zeros) { return v >= 0.0f && v < (zeros ? INFINITY : PAGED_TINY) ? PAGED_TINY : v; }

// ---------------------------------------------------------------- one or a few new rows
//
// Block = 4 wavefronts, 16 (position, query head) pairs of one kv head of one sequence.  Bound by memory: each wavefront walks its own steps of 32 keys, K rows to registers as
// they are the matrix operand, V rows through registers into the wavefront's own LDS, from where the transposing reads take them; the next step's K rows are asked
// for as soon as the scores are made, its V rows as soon as those are in LDS, and nothing is waited for but that.  The wavefronts meet once, at the end.
// The matrix instruction's 16 columns are the rows, so that a lane has four scores of each 16 keys of one row, and its weights are the operand of O^T = V^T . P^T as they lie.
// Parts of an item are merged by the last of its blocks to arrive.
// 3 sequences of 65000, 32 heads of 128 over 8, fp16: 117 us = 5.8 TB/s, as fast as a launch that only reads.  16 of 435 to 4352, int8 (81 MB) 21.4 us = 3.8 TB/s: 4 us of launch, some 3 each
// until the first keys are there and for the merge.
constexpr int FEW_THREADS = 256, FEW_QROWS = 16, FEW_MOST = 64;   // parts of an item: a lane for each
constexpr float FEW_TOP = 15.0f;                           // a row's largest weight is 2^15: halves are normal numbers down to 2^-29 of it

// Two groups of 16 keys: their first positions, and the pages that hold them, or -1.
struct FewStep {
  int key[2], id[2];
};
// Which keys an item walks: a range of the sequence's positions, with a window and sinks.
struct RangeKeys {
  PagedKeys keys;
  int b, window, sinks;
  __device__ void find(const PagedBatch &pb, int st, FewStep &s) const {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s.key[h] = keys.tile(st >> 1) * PAGED_KEYS + (st & 1) * 32 + 16 * h;
      s.id[h] = page_uniform(pb, b, s.key[h]);
    }
  }
  // whether some row from pos_lo to pos_hi may not see some key of a step
  __device__ bool masks(const int (&k)[2], int pos_lo, int pos_hi) const { return k[0] + 31 > pos_lo || (window && k[0] <= pos_hi - window && k[0] + 32 > sinks); }
  __device__ bool sees(int key, int pos) const { return (key <= pos) & ((key > (window ? pos - window : -1)) | (key < (window ? sinks : 0))); }
};

template <int HD, bool I8> struct PagedFew {
  static constexpr int NW = 4, KEYS = 32, ROWB = HD * 2;
  static constexpr int VROW = ROWB + 32;                     // bytes between V rows in LDS: eight banks further each, so that the reads of 16 rows by 32 bytes meet all banks alike
  static constexpr int NT = HD / 16, KS = HD / 32;           // 16-feature tiles of the output, matrix instructions per 16 keys
  static constexpr int OROW = HD + 4;                        // floats between rows of a wavefront's sums in LDS
  static constexpr int GK = KS / (I8 ? 2 : 1), LPR = HD / (I8 ? 16 : 8), GV = LPR / 4;   // 16-byte loads of 16 keys' K and V; lanes per V row
  static constexpr int SLOT = FEW_QROWS * (HD + 4);           // floats of a part: the rows' sums, then (m, l, -, -) of each
  struct Smem {
    union {
      unsigned char v[KEYS * VROW];
      float o[FEW_QROWS * OROW];
    } wave[NW];
    float m[NW][FEW_QROWS], l[NW][FEW_QROWS];
    float w[FEW_QROWS][FEW_MOST], inv[FEW_QROWS];
    f4_t fold[FEW_THREADS];
    int is_last;
  };
  // Must be called by every thread of the block (it contains barriers).
  static __device__ void item(const PagedAttnArgs &a, const PagedItem &it, Smem &sm) {
    const int n_rep = (int)a.n_rep.d, room = paged_room(a.pb), rows = it.s.n * n_rep, p0 = paged_pos(it.s, 0), q0 = it.qt * FEW_QROWS, nr = min(FEW_QROWS, rows - q0);
    const PagedKeys keys = paged_keys(p0 + a.n_rep.div(q0), p0 + a.n_rep.div(q0 + nr - 1), room, a.window, a.sinks);
    int i_lo = 0, i_hi = keys.n;
    if (it.parts > 1) {
      const int per = (keys.n + it.parts - 1) / it.parts;
      i_lo = min(it.part * per, keys.n);
      i_hi = min(i_lo + per, keys.n);
    }
    walk(a, it, RangeKeys{keys, it.b, a.window, a.sinks}, 2 * i_lo, 2 * i_hi, sm);
  }
  // The item over steps st_lo to st_end of its keys.
  template <typename Keys> static __device__ void walk(const PagedAttnArgs &a, const PagedItem &it, const Keys &keys, int st_lo, int st_end, Smem &sm) {
    const float scale_log2 = a.scale_log2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lq = lane >> 4;
    const int n_rep = (int)a.n_rep.d, KV = (int)a.n_kv_heads.d, g = it.g;
    const int rows = it.s.n * n_rep, p0 = paged_pos(it.s, 0), q0 = it.qt * FEW_QROWS, nr = min(FEW_QROWS, rows - q0);
    const int pos_lo = p0 + a.n_rep.div(q0), pos_hi = p0 + a.n_rep.div(q0 + nr - 1);
    auto out_row = [&](int r) {                              // of pair q0 + r
      const int qs = a.n_rep.div(q0 + r);
      return ((size_t)(it.s.start + qs) * a.n_heads + g * n_rep + q0 + r - qs * n_rep) * HD;
    };
    const int qpos = p0 + a.n_rep.div(q0 + min(l16, nr - 1));  // columns past the end repeat the last row and are never stored
    auto sees = [&](int key) { return keys.sees(key, qpos); };
    u4_t kr[2][GK], vr[2][GV];
    f4_t ks[2], vs[2];
    FewStep at, next;
    auto find = [&](int st, FewStep &to) {
      if (st < st_end) keys.find(a.pb, st, to);
      else to = FewStep{{0, 0}, {-1, -1}};
    };
    auto load_k = [&](const FewStep &to) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const size_t row = paged_row(a.pb, KV, max(to.id[h], 0), g, to.key[h]);   // a missing page: page 0, masked
#pragma unroll
        for (int c = 0; c < GK; c++)
          kr[h][c] = *as_global<u4_t>((const unsigned char *)a.pages_k + (row + l16) * (I8 ? HD : ROWB) + (lq + 4 * c) * 16);
        if constexpr (I8) ks[h] = *as_global<f4_t>(a.scales_k + row + 4 * lq);
      }
    };
    auto load_v = [&](const FewStep &to) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const size_t row = paged_row(a.pb, KV, max(to.id[h], 0), g, to.key[h]);
#pragma unroll
        for (int c = 0; c < GV; c++)
          vr[h][c] = *as_global<u4_t>((const unsigned char *)a.pages_v + (row + c * (64 / LPR) + lane / LPR) * (I8 ? HD : ROWB) + lane % LPR * 16);
        if constexpr (I8) vs[h] = *as_global<f4_t>(a.scales_v + row + 4 * lq);
      }
    };

    int st = st_lo + wave;
    find(st, at);
    if (st < st_end) {
      load_k(at);
      load_v(at);
    }
    h8_t qf[KS];                                             // the features that the K fragments have: fp16 8 (4 s + lq) .., int8 16 (lq + 4 c) + 8 u .., s = 2 c + u
    {
      const _Float16 *const qp = a.q + out_row(min(l16, nr - 1));
#pragma unroll
      for (int s = 0; s < KS; s++) qf[s] = *(const h8_t *)(qp + (I8 ? 16 * (lq + 4 * (s / 2)) + 8 * (s % 2) : 8 * (4 * s + lq)));
    }
    f4_t o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) o[t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -1e30f, l_run = 0.0f;                      // finite: a step may hold no key that a row sees
    const float unit = I8 ? 1.0f : scale_log2;
    unsigned char *const vl = sm.wave[wave].v;

    auto step = [&](auto more) {
      find(st + NW, next);
      f4_t s[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        s[h] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < GK; c++)
#pragma unroll
          for (int u = 0; u < KS / GK; u++) {
            u4_t k = kr[h][c];
            if constexpr (I8) {
              uint32_t w[4];
              i8x4_to_h2x2(kr[h][c][2 * u], w[0], w[1]);
              i8x4_to_h2x2(kr[h][c][2 * u + 1], w[2], w[3]);
              k = u4_t{w[0], w[1], w[2], w[3]};
            }
            s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, k), qf[c * (KS / GK) + u], s[h], 0, 0, 0);
          }
      }
      if constexpr (I8) {
#pragma unroll
        for (int h = 0; h < 2; h++) ks[h] *= scale_log2;
      }
      const f4_t kscale[2] = {ks[0], ks[1]};
      if constexpr (decltype(more)::value) load_k(next);
      f4_t inv_v[2];
      if constexpr (I8) {
        // scale_of_v, for which there is a reason in few steps: 16 codes of zero side by side, or a scale below PAGED_TINY
        uint32_t codes = ~0u;
        float least = INFINITY;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int c = 0; c < GV; c++) codes = min(codes, vr[h][c][0] | vr[h][c][1] | vr[h][c][2] | vr[h][c][3]);
#pragma unroll
          for (int e = 0; e < 4; e++) least = fminf(least, vs[h][e]);
        }
        if (__builtin_amdgcn_ballot_w64(codes == 0 || least < PAGED_TINY)) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            // lanes LPR * r and on have row r of the sixteen: LPR bits of each of these four rows
            uint64_t some[GV];
#pragma unroll
            for (int c = 0; c < GV; c++) some[c] = __builtin_amdgcn_ballot_w64((vr[h][c][0] | vr[h][c][1] | vr[h][c][2] | vr[h][c][3]) != 0);
            const uint32_t mine = (uint32_t)(some[lq * GV / 4] >> (lq * 4 % (64 / LPR)) * LPR);
#pragma unroll
            for (int e = 0; e < 4; e++) vs[h][e] = scale_of_v(vs[h][e], ((mine >> e * LPR) & ((1u << LPR) - 1)) == 0);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            // as in the chunk kernel: the scale of V in the exponent, its reciprocal finite whatever lies in a place that no row sees
            const float v = vs[h][e];
            s[h][e] = __builtin_fmaf(s[h][e], kscale[h][e], __builtin_amdgcn_logf(v));
            inv_v[h][e] = v >= PAGED_TINY && v < INFINITY ? __builtin_amdgcn_rcpf(v) : 1.0f;
          }
      }
      // value r of s[h] is key at.key[h] + 4 lq + r of row l16
      const bool masked = (at.id[0] | at.id[1]) < 0 || keys.masks(at.key, pos_lo, pos_hi);
      if (masked) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            s[h][r] = (sees(at.key[h] + 4 * lq + r) & (at.id[h] >= 0)) ? s[h][r] : -INFINITY;
      }
      float mx = m_run;
#pragma unroll
      for (int h = 0; h < 2; h++) mx = fmaxf(fmaxf(fmaxf(mx, s[h][0]), fmaxf(s[h][1], s[h][2])), s[h][3]);
      mx = max_xor32(max_xor16(mx));
      if (__builtin_amdgcn_ballot_w64(mx > m_run)) {
        const float alpha = __builtin_amdgcn_exp2f((m_run - mx) * unit);
        m_run = mx;
        l_run *= alpha;
#pragma unroll
        for (int t = 0; t < NT; t++) o[t] *= alpha;
      }
      h8_t pf;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          // the difference first: it is never above zero, however large the scores are
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][r] - m_run, unit, FEW_TOP));
          l_run = I8 ? __builtin_fmaf(p, inv_v[h][r], l_run) : l_run + p;
          pf[4 * h + r] = (_Float16)p;
        }
      uint32_t bad = 0;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int c = 0; c < GV; c++) {
          const int r = 16 * h + c * (64 / LPR) + lane / LPR, piece = lane % LPR;
          if constexpr (I8) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
              uint32_t w[4];
              i8x4_to_h2x2(vr[h][c][2 * u], w[0], w[1]);
              i8x4_to_h2x2(vr[h][c][2 * u + 1], w[2], w[3]);
              *(u4_t *)(vl + r * VROW + (2 * piece + u) * 16) = u4_t{w[0], w[1], w[2], w[3]};
            }
          } else {
            *(u4_t *)(vl + r * VROW + piece * 16) = vr[h][c];
#pragma unroll
            for (int e = 0; e < 4; e++) bad |= (vr[h][c][e] & 0x7fff7fffu) + 0x04000400u;   // bits 15 and 31: a half that is not finite
          }
        }
      if constexpr (decltype(more)::value) load_v(next);
      auto weigh = [&](auto clean) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
          s4_t v[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int r = 16 * h + 4 * lq + (l16 >> 2), c = t * 32 + (l16 & 3) * 8;
            v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t *)(vl + r * VROW + c));
          }
          u4_t w = __builtin_bit_cast(u4_t, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
          if constexpr (decltype(clean)::value) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t x = ((w[e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
              w[e] &= ~(x | (x - (x >> 15)));
            }
          }
          o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, w), pf, o[t], 0, 0, 0);
        }
      };
      if (I8 || !__builtin_amdgcn_ballot_w64((bad & 0x80008000u) != 0)) {
        weigh(std::false_type());
      } else {
        // halves that are not finite: left out of the product, where a weight of zero would not stop them, and added for the rows that see them
        weigh(std::true_type());
        for (int key = 0; key < KEYS; key++) {
          const bool seen = sees((key < 16 ? at.key[0] : at.key[1]) + (key & 15)) && (key < 16 ? at.id[0] : at.id[1]) >= 0;
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
      at = next;
    };
    // the last step by itself: behind a branch around its loads every wait would be for all of them
    if (st < st_end) {
      for (; st + NW < st_end; st += NW) step(std::true_type());
      step(std::false_type());
    }

    // the block's wavefronts: value r of o[t] is feature 16 t + 4 lq + r of row l16
    l_run = add_xor32(add_xor16(l_run));
#pragma unroll
    for (int t = 0; t < NT; t++) *(f4_t *)&sm.wave[wave].o[l16 * OROW + t * 16 + 4 * lq] = o[t];
    if (lq == 0) { sm.m[wave][l16] = m_run; sm.l[wave][l16] = l_run; }
    lds_barrier();
    auto block_sum = [&](int r, int c, f4_t &sum, float &M, float &L) {   // features 4 c .. of row r
      M = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
      sum = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
      L = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float e = __builtin_amdgcn_exp2f((sm.m[w][r] - M) * unit);
        L = __builtin_fmaf(sm.l[w][r], e, L);
        const f4_t v = *(const f4_t *)&sm.wave[w].o[r * OROW + 4 * c];
#pragma unroll
        for (int x = 0; x < 4; x++) sum[x] = __builtin_fmaf(v[x], e, sum[x]);
      }
    };
    auto put = [&](int r, int c, f4_t sum, float inv) {
      const h2_t lo = {(_Float16)(sum[0] * inv), (_Float16)(sum[1] * inv)}, hi = {(_Float16)(sum[2] * inv), (_Float16)(sum[3] * inv)};
      *(uint2 *)(a.out + out_row(r) + 4 * c) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    };
    const int pieces = nr * (HD / 4);
    if (it.parts == 1) {
      for (int i = tid; i < pieces; i += FEW_THREADS) {
        f4_t sum;
        float M, L;
        block_sum(i / (HD / 4), i % (HD / 4), sum, M, L);
        put(i / (HD / 4), i % (HD / 4), sum, L == 0.0f ? 0.0f : 1.0f / L);   // 0: the row sees nothing
      }
      return;
    }
    // Parts: sums through memory at device scope (cache policy 16), counted once they are acknowledged; the last block of the item folds them in order.
    const uint32_t part_bytes = (uint32_t)KV * SLOT * 4;
    const __amdgpu_buffer_rsrc_t rw = wave_buffer(a.few_ws + (size_t)it.slot * SLOT, (uint32_t)(it.parts - 1) * part_bytes + SLOT * 4);
    for (int i = tid; i < pieces; i += FEW_THREADS) {
      f4_t sum;
      float M, L;
      const int r = i / (HD / 4), c = i % (HD / 4);
      block_sum(r, c, sum, M, L);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, sum), rw, (uint32_t)it.part * part_bytes + i * 16, 0, 16);
      if (c == 0) {
        const f4_t ml = {M, L, 0.0f, 0.0f};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, ml), rw, (uint32_t)it.part * part_bytes + (FEW_QROWS * HD + r * 4) * 4, 0, 16);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) sm.is_last = __hip_atomic_fetch_add(&a.few_counters[it.slot], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == it.parts - 1;
    __syncthreads();
    if (!sm.is_last) return;
    if (tid == 0) __hip_atomic_store(&a.few_counters[it.slot], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
    // weights of the parts: a wavefront per row, a part per lane
    for (int r = wave; r < nr; r += NW) {
      const f4_t ml = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)min(lane, it.parts - 1) * part_bytes + (FEW_QROWS * HD + r * 4) * 4, 0, 16));
      const float m = lane < it.parts ? ml[0] : -1e30f, M = wave_max(m), e = lane < it.parts ? __builtin_amdgcn_exp2f((m - M) * unit) : 0.0f;
      const float L = wave_sum(lane < it.parts ? ml[1] * e : 0.0f);
      sm.w[r][lane] = e;
      if (lane == 0) sm.inv[r] = L == 0.0f ? 0.0f : 1.0f / L;
    }
    lds_barrier();
    // a thread per four features of a row; where those are fewer than threads, groups of threads share the parts
    const int groups = pieces < FEW_THREADS ? FEW_THREADS / pieces : 1, mine = groups > 1 ? tid / pieces : 0;
    for (int i0 = groups > 1 ? tid - mine * pieces : tid; i0 < pieces; i0 += FEW_THREADS) {
      const int r = i0 / (HD / 4), c = i0 % (HD / 4);
      f4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
      if (mine < groups)
        for (int f = mine; f < it.parts; f += groups * 8) {
          f4_t v[8];
#pragma unroll
          for (int u = 0; u < 8; u++)
            v[u] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)min(f + u * groups, it.parts - 1) * part_bytes + i0 * 16, 0, 16));
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (f + u * groups < it.parts)
#pragma unroll
              for (int x = 0; x < 4; x++) sum[x] = __builtin_fmaf(v[u][x], sm.w[r][f + u * groups], sum[x]);
        }
      if (groups == 1) put(r, c, sum, sm.inv[r]);
      else sm.fold[tid] = sum;
    }
    if (groups > 1) {
      lds_barrier();
      if (tid < pieces) {
        f4_t sum = sm.fold[tid];
        for (int u = 1; u < groups; u++) sum += sm.fold[tid + u * pieces];
        put(tid / (HD / 4), tid % (HD / 4), sum, sm.inv[tid / (HD / 4)]);
      }
    }
  }
};

}  // namespace jsg
