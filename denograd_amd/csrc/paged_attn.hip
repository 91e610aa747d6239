// Grouped-query attention of a ragged batch of new rows over a paged KV cache (jsgrad_hip_attn_paged).
//
// Row i of a sequence sits at position p and sees the keys j <= p that have a page and, with a window, are among the last `window` of them or
// among the first `sinks`: out = sum_j softmax_j(q . K_j / sqrt(HD)) V_j, zeros where it sees none.  Reference semantics of the sum:
// scaled_dot_product_attention (jsgrad/tensor.ts:3920-3934); windows, sinks and pages have no counterpart there.
#include <type_traits>

#include "paged_few.h"

namespace jsg {

// ---------------------------------------------------------------- which work a block has
//
// A launch's items are (sequence, q tile, kv head); a q tile is QROWS (position, query head) pairs of a kv head, row = position * n_rep + head.  Long
// ones are cut along the keys, so that the parts of a launch have about the same number of key tiles whatever the lengths of its sequences are
// (paged_target).  The host knows neither lengths nor row starts: every wavefront goes over them, a sequence to a lane, and finds its block's item.
// Block numbers have the kv heads innermost: blocks are dealt to the eight XCDs in turn, so that with eight kv heads each XCD has one, all q tiles of which
// share its K and V in that L2, and all XCDs have the same work.  The q tiles with the most keys come first within a sequence.
constexpr uint32_t PAGED_MOST = 1u << 29;  // more than PAGED_GRID: sums stop there instead of wrapping

__device__ __forceinline__ uint32_t scan64(uint32_t v) {     // inclusive prefix sums over the lanes, saturating
  auto add = [&](uint32_t o) { v = min(v + o, PAGED_MOST); };
  add((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true));    // row_shr
  add((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true));
  add((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true));
  add((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true));
  add((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));   // row_bcast 15
  add((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));   // row_bcast 31
  return v;
}

// 64 sequences, one to a lane; n is -1 where first rows fall.
__device__ __forceinline__ PagedSeq lane_seq(const PagedBatch &p, int b0) {
  const int b = b0 + (threadIdx.x & 63);
  if (b >= p.n_seqs) return {0, 0, 0};
  PagedSeq s = paged_seq(p, b);
  if (paged_falls(p, b)) s.n = -1;
  return s;
}

// Goes over the sequences, 64 at a time: look(first of them, this lane's) until it says true.  The next ones are asked for in front of it; sequences without new rows, as a batch that is filled up has many, are
// passed over by the 64.
template <typename Look> __device__ __forceinline__ bool paged_walk(const PagedBatch &p, const PagedSeq &first, Look look) {
  PagedSeq s = first;
  for (int b0 = 0; b0 < p.n_seqs; b0 += 64) {
    PagedSeq next = {0, 0, 0};
    if (b0 + 64 < p.n_seqs) next = lane_seq(p, b0 + 64);
    if (__builtin_amdgcn_ballot_w64(s.n != 0) && look(b0, s)) return true;
    s = next;
  }
  return false;
}

// q tiles of all heads, and pairs of these and a key tile, of some of a launch's sequences
struct PagedSum {
  float pairs, items;
  __device__ void add(const PagedShare &h) { pairs += (float)h.q_tiles * (float)h.key_tiles; items += (float)h.q_tiles; }
  __device__ void join(int KV) { pairs = wave_sum(pairs) * (float)KV; items = wave_sum(items) * (float)KV; }
};

template <int QROWS> __device__ __forceinline__ PagedShare share_of(const PagedAttnArgs &a, const PagedSeq &s) {
  return paged_share(s, (int)a.n_rep.d, [&](int x) { return a.n_rep.div(x); }, QROWS, paged_room(a.pb), a.window, a.sinks);
}

// The item of block `id` among those of the sequences with `from` to `to` (position, query head) pairs per kv head, `sum` being these and share0 the first 64's: blocks: what they are shared among, least: see
// paged_target; most(key tiles): parts of an item; last: none of other sequences come behind these.  False, and id less these items' blocks, where it is none of them.
template <int QROWS, typename Most>
__device__ __forceinline__ bool paged_item(const PagedAttnArgs &a, const PagedSeq &first, const PagedShare &share0, int &id, int from, int to, const PagedSum &sum, int blocks, int least, Most most, bool last, PagedItem &it) {
  const int n_rep = (int)a.n_rep.d, KV = (int)a.n_kv_heads.d;
  const uint32_t want = (uint32_t)a.n_kv_heads.div(id);
  it.g = id - (int)want * KV;
  const float pairs = sum.pairs, items = sum.items;
  auto share_here = [&](int b0, const PagedSeq &s) {
    const PagedShare h = b0 ? share_of<QROWS>(a, s) : share0;
    return s.n * n_rep >= from && s.n * n_rep <= to ? h : PagedShare{0, 0};
  };
  // A share of the pairs each.  An item has up to one part more than its pairs make whole, so that all come to blocks + items and less.  Few items: a larger share of the
  // pairs makes up for that.  More: the first of some larger shares with which the parts are no more than the blocks; or twice the share, where nothing else is.
  const int share = paged_target(pairs, blocks, least);
  int target = 2 * share;
  auto cut = [&](const PagedShare &h, int t) { return paged_parts(h.key_tiles, t, __builtin_amdgcn_rcpf((float)t), most(h.key_tiles)); };
  if (items * 16.0f <= (float)blocks) target = share + share / 16;
  else if (a.pb.n_seqs <= 64 && items < (float)blocks) {
    const PagedShare h = share_here(0, first);
    for (int t = share; t < 2 * share; t += (share + 3) / 4)
      if (wave_sum((float)h.q_tiles * (float)cut(h, t)) * (float)KV <= (float)blocks) {
        target = t;
        break;
      }
  }
  // a launch has blocks for the worst batch of its size, most of which are behind the last item of others
  if (last && (float)id >= paged_most_blocks(pairs, items, __builtin_amdgcn_rcpf((float)target))) return false;
  uint32_t before = 0, slots = 0;
  const bool found = paged_walk(a.pb, first, [&](int b0, const PagedSeq &s) {
    const PagedShare h = share_here(b0, s);
    const int parts = cut(h, target);
    const uint32_t mine = (uint32_t)min((uint64_t)h.q_tiles * parts, (uint64_t)PAGED_MOST);
    const uint32_t upto = scan64(mine), held = scan64(parts > 1 ? mine : 0);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(before + upto > want);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      it.b = b0 + l;
      it.s = {of(s.start), of(s.n), of(s.len)};
      it.parts = of(parts);
      const int nth = (int)(want - before) - of((int)(upto - mine));
      it.part = 0;
      it.qt = of(h.q_tiles) - 1 - nth;
      if (it.parts > 1) {
        it.qt = of(h.q_tiles) - 1 - nth / it.parts;
        it.part = nth % it.parts;
      }
      it.slot = ((int)slots + of((int)(held - (parts > 1 ? mine : 0))) + nth - it.part) * KV + it.g;
      return true;
    }
    before = min(before + (uint32_t)__builtin_amdgcn_readlane((int)upto, 63), PAGED_MOST);
    slots = min(slots + (uint32_t)__builtin_amdgcn_readlane((int)held, 63), PAGED_MOST);
    return false;
  });
  if (!found) id -= (int)before * KV;
  return found;
}

// ---------------------------------------------------------------- chunks of new rows
//
// Block = 4 wavefronts = 128 (position, query head) pairs of one kv head of one sequence, keys in tiles of 64, as attn_prefill_kernel (prefill.hip) has it:
// scores transposed, S^T = K . Q^T, so that a lane holds 32 scores of one query row per tile and its fp16 weights lie as the operand of O^T = V^T . P^T
// wants them; V^T fragments by transposing LDS reads; one barrier per tile, tile t + 1 being asked for behind the barrier of tile t.
// A page has 16 rows at least: the 16 rows of a tile that a wavefront brings lie on one page, whose number it asks for a tile ahead.
// fp16 pages come by direct global-to-LDS loads.  int8 ones come through registers and become halves on their way into LDS (exact), once for the block;
// K's scale multiplies the scores.  V's scale goes into the exponent, weight = exp2(score + log2(scale) - maximum of that), so that the largest contributions
// keep their bits whatever the scales are; the sum of the weights takes it out again, in float.
// Tiles that hold keys which some row of the wavefront does not see (the diagonal, a window's edge, a missing page) take their V through a test: halves that are not
// finite are left out of the product, where a weight of zero would not stop them, and added for the rows that see them.
//
// 16 x 2048 rows of 32 heads over 8, causal: heads of 128, fp16 735 us = 0.75 PFLOP/s, int8 808; heads of 64 407 and 498.  No unit is full: at the 1.8 GHz that the power limit leaves, the
// matrix cores are busy 35 % of the time and the vector unit 51 (an exponential per score, and four more operations), LDS 18; a wavefront waits 26 % for memory and barriers and 30 % to issue, and
// registers and LDS have room for two to a SIMD (heads of 64: three or four).
constexpr int PC_THREADS = 256, PC_QROWS = 128;
constexpr int PC_BLOCKS = 512, PC_LEAST = 4;               // two blocks to a compute unit; a tile takes 1.4 us, and a part some 5 us of its own
constexpr int PC_SLOTS = 2 * PC_BLOCKS;
// A row's weights are exp2(score - its maximum + PC_TOP): the largest is 2^15, which a half holds exactly, the others are rounded to 11 bits down to 2^-29 of it.
constexpr float PC_TOP = 15.0f;

template <int HD, bool I8> struct PagedChunk {
  static constexpr int ROWB = HD * 2, PPR = HD / 8;                 // bytes and 16-byte pieces of a row of halves
  static constexpr int TILE = PAGED_KEYS * ROWB, BUF = 2 * TILE;    // K tile, then V tile
  static constexpr int LOADS = TILE / 1024 / 4;                     // a wavefront's loads per tile of K, and of V
  static constexpr int RPL = 64 / PPR;                              // rows per load
  static constexpr int NT = HD / 32;                                // 32-feature tiles of the output
  static constexpr int CPT = HD / 64;                               // 16-byte pieces of codes per thread and tile of K, and of V
  struct Smem {
    __align__(16) unsigned char tiles[2 * BUF];
    float scl[2][3][PAGED_KEYS];                             // I8: K's scale times scale_log2, log2 and reciprocal of V's
  };

  // Must be called by every thread of the block (it contains barriers).
  static __device__ void item(const PagedAttnArgs &a, const PagedItem &it, Smem &sm) {
    const float scale_log2 = a.scale_log2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, lg = lane >> 5;
    unsigned char *const lds = sm.tiles;
    auto &scl = sm.scl;
    const int n_rep = (int)a.n_rep.d, KV = (int)a.n_kv_heads.d, room = paged_room(a.pb), g = it.g;
    const int rows = it.s.n * n_rep, p0 = paged_pos(it.s, 0), q0 = it.qt * PC_QROWS, qw0 = q0 + wave * 32;
    const PagedKeys keys = paged_keys(p0 + a.n_rep.div(q0), p0 + a.n_rep.div(min(q0 + PC_QROWS, rows) - 1), room, a.window, a.sinks);
    int i_lo = 0, i_hi = keys.n;
    if (it.parts > 1) {
      const int per = (keys.n + it.parts - 1) / it.parts;
      i_lo = min(it.part * per, keys.n);
      i_hi = min(i_lo + per, keys.n);
    }
    // this wavefront's first and last position; rows past the end repeat the last one and are never stored
    const int pos_lo = p0 + a.n_rep.div(min(qw0, rows - 1)), pos_hi = p0 + a.n_rep.div(min(qw0 + 31, rows - 1));
    const bool q_valid = qw0 + l32 < rows;
    const int qrow = min(qw0 + l32, rows - 1), qs = a.n_rep.div(qrow), qpos = p0 + qs;
    const size_t q_off = ((size_t)(it.s.start + qs) * a.n_heads + g * n_rep + qrow - qs * n_rep) * HD;
    const int sees_from = a.window ? qpos - a.window : -1, sees_to = a.window ? a.sinks : 0;   // keys <= qpos that are > sees_from or < sees_to

    // where piece p of row r of a tile is kept.  A quarter of the lanes reads a piece of sixteen rows of K, half of them 64 bytes of four rows of V, and a quarter writes (int8)
    // four pieces, of different 64 bytes, of four rows: each goes over all 64 banks.
    auto k_at = [](int r, int p) { return HD == 128 ? p ^ (r & 15) : p ^ ((r >> 1) & 7); };
    auto v_at = [](int r, int p) { return HD == 128 ? p ^ ((r & 3) * 5) : p ^ (((r >> 1) & 1) * 5); };

    // this wavefront's rows of a tile: 16 * wave and on
    auto page_of = [&](int i) { return i < i_hi ? page_uniform(a.pb, it.b, keys.tile(i) * PAGED_KEYS + wave * 16) : -1; };
    auto row_of = [&](int i, int id) { return paged_row(a.pb, KV, max(id, 0), g, keys.tile(i) * PAGED_KEYS + wave * 16); };   // a missing page: page 0, masked
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds + wave * LOADS * 1024;
    const int lrow = lane / PPR, lp = lane % PPR;
    auto issue = [&](int i, int id, int buf) {                 // fp16
      const uint32_t to = lds0 + buf * BUF;
      const size_t at = row_of(i, id) * ROWB;
      const i4_t rk = dma_rsrc((const unsigned char *)a.pages_k + at), rv = dma_rsrc((const unsigned char *)a.pages_v + at);
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        const int r = j * RPL + lrow;
        dma16(rk, (uint32_t)r * ROWB + k_at(wave * 16 + r, lp) * 16, 0, to + j * 1024);
        dma16(rv, (uint32_t)r * ROWB + v_at(wave * 16 + r, lp) * 16, 0, to + TILE + j * 1024);
      }
    };
    u4_t kc[CPT], vc[CPT];                                     // int8: this thread's codes and scale on their way
    float sc = 1.0f;
    const float *const scales_k = a.scales_k, *const scales_v = a.scales_v;
    const int crow = lane >> 2, cp = (lane & 3) * CPT;         // row and first piece of codes
    auto load = [&](int i, int id) {
      const size_t row = row_of(i, id);
#pragma unroll
      for (int c = 0; c < CPT; c++) {
        kc[c] = *as_global<u4_t>((const int8_t *)a.pages_k + (row + crow) * HD + (cp + c) * 16);
        vc[c] = *as_global<u4_t>((const int8_t *)a.pages_v + (row + crow) * HD + (cp + c) * 16);
      }
      sc = *as_global<float>((lane & 16 ? scales_v : scales_k) + row + (lane & 15));
    };
    auto store = [&](int buf) {
      unsigned char *const kt = lds + buf * BUF, *const vt = kt + TILE;
      const int r = wave * 16 + crow;
#pragma unroll
      for (int c = 0; c < CPT; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          u4_t k, v;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            uint32_t lo, hi;
            i8x4_to_h2x2(kc[c][2 * h + e], lo, hi);
            k[2 * e] = lo; k[2 * e + 1] = hi;
            i8x4_to_h2x2(vc[c][2 * h + e], lo, hi);
            v[2 * e] = lo; v[2 * e + 1] = hi;
          }
          const int p = (cp + c) * 2 + h;
          *(u4_t *)(kt + r * ROWB + k_at(r, p) * 16) = k;
          *(u4_t *)(vt + r * ROWB + v_at(r, p) * 16) = v;
        }
      uint32_t codes = 0;
#pragma unroll
      for (int c = 0; c < CPT; c++) codes |= vc[c][0] | vc[c][1] | vc[c][2] | vc[c][3];
      const uint64_t some = __builtin_amdgcn_ballot_w64(codes != 0);   // four lanes to a row
      if (lane < 16) scl[buf][0][wave * 16 + lane] = sc * scale_log2;
      else if (lane < 32) {
        // A scale that is not a number makes the weights so, for the rows that see it.  Its reciprocal meets weights of zero as well, there and where
        // nothing was ever written, and has to be finite.
        const float v = scale_of_v(sc, ((uint32_t)(some >> (lane - 16) * 4) & 15) == 0);
        scl[buf][1][wave * 16 + lane - 16] = __builtin_amdgcn_logf(v);
        scl[buf][2][wave * 16 + lane - 16] = v >= PAGED_TINY && v < INFINITY ? __builtin_amdgcn_rcpf(v) : 1.0f;
      }
    };

    int id = page_of(i_lo), id_next = page_of(i_lo + 1);
    if (i_lo < i_hi) {
      if constexpr (I8) load(i_lo, id);
      else issue(i_lo, id, 0);
    }
    // whether some page of these tiles is not there
    bool holes = false;
    for (int n = i_lo * 4 + lane; n < i_hi * 4; n += 64) holes |= paged_page(a.pb, it.b, keys.tile(n >> 2) * PAGED_KEYS + (n & 3) * 16) < 0;
    holes = __builtin_amdgcn_ballot_w64(holes) != 0;
    // query row fragments: chunk c covers features [16c, 16c+16), the lane half picks 8 of them
    h8_t qf[HD / 16];
    {
      const _Float16 *qp = a.q + q_off + lg * 8;
#pragma unroll
      for (int c = 0; c < HD / 16; c++) qf[c] = *(const h8_t *)(qp + c * 16);
    }
#pragma unroll
    for (int c = 0; c < HD / 16; c++) asm volatile("" : "+v"(qf[c]));   // waited for here, in front of the loop
    if constexpr (I8)
      if (i_lo < i_hi) store(0);

    f16_t o_acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) o_acc[t][r] = 0.0f;
    // the maximum starts finite: a part of the keys may hold none that a row sees, and -inf minus -inf is not a number
    float m_run = -1e30f, l_run = 0.0f;                      // the maximum less PC_TOP
    const float unit = I8 ? 1.0f : scale_log2;               // of scores and their maximum: int8 ones have the factor in K's scale

    // K fragment of key l32 (+ 32): chunk 2c + lg of its row; V: lane -> row (lane / 4 % 4) of its half's four keys, 8 bytes
    const unsigned char *const kp = lds + l32 * ROWB;
    const int vrow = 4 * lg + ((lane >> 2) & 3), vcol = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;   // byte column inside 64 (32 features)

    // A tile that every row of the block sees whole, or one with the tests; returns after the next tile has been asked for and this one used.
    const int blk_lo = p0 + a.n_rep.div(q0), blk_hi = p0 + a.n_rep.div(min(q0 + PC_QROWS, rows) - 1);
    int i = i_lo, buf = 0;
    auto begin = [&]() {                                       // tile i is there, everyone is done with tile i - 1; whether all of the block sees all of it
      if constexpr (!I8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();
      id = id_next;
      if (i + 1 < i_hi) {
        if constexpr (I8) load(i + 1, id);
        else issue(i + 1, id, buf ^ 1);
        id_next = page_of(i + 2);
      }
      const int k0 = keys.tile(i) * PAGED_KEYS;
      return k0 + PAGED_KEYS - 1 <= blk_lo && !holes && !(a.window && k0 <= blk_hi - a.window && k0 + PAGED_KEYS > a.sinks);
    };
    auto end = [&]() {
      if constexpr (I8)
        if (i + 1 < i_hi) store(buf ^ 1);
      i++;
      buf ^= 1;
    };
    auto tile = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      const int k0 = keys.tile(i) * PAGED_KEYS;
      auto sees = [&](int key) { return (key <= qpos) & ((key > sees_from) | (key < sees_to)); };
      const unsigned char *const kt = kp + buf * BUF, *const vt = lds + buf * BUF + TILE;
      h8_t pf[2][2];
      uint32_t bad = 0;
      int pm = 15;                                           // which of the tile's four pages of 16 rows are there
      if (!WHOLE && holes) {
        pm = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) pm |= (page_uniform(a.pb, it.b, k0 + 16 * u) >= 0) << u;
      }
      // scores of 32 keys: accumulator r is key k0 + tk*32 + 8*(r/4) + 4*lg + r%4 for query row l32
      auto score = [&](int tk) {
        f16_t s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < HD / 16; c++) {
          const h8_t kf = *(const h8_t *)(kt + tk * 32 * ROWB + k_at(l32, 2 * c + lg) * 16);
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[c], s, 0, 0, 0);
        }
        return s;
      };
      auto finish = [&](f16_t &s, int tk) {
        if constexpr (I8) {
#pragma unroll
          for (int r4 = 0; r4 < 4; r4++) {
            const int at = tk * 32 + 8 * r4 + 4 * lg;
            const f4_t ks = *(const f4_t *)&scl[buf][0][at], lv = *(const f4_t *)&scl[buf][1][at];
#pragma unroll
            for (int e = 0; e < 4; e++) s[r4 * 4 + e] = __builtin_fmaf(s[r4 * 4 + e], ks[e], lv[e]);
          }
        }
        if constexpr (!WHOLE) {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int key = k0 + tk * 32 + 8 * (r / 4) + 4 * lg + (r % 4);
            s[r] = (sees(key) & ((pm >> (tk * 2 + r / 8) & 1) != 0)) ? s[r] : -INFINITY;
          }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 15; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
        return fmaxf(mx, s[15]);
      };
      // The sums are rescaled whenever some row's maximum has moved, so that the largest weight is not rounded, as in attn_prefill_kernel.  Off from float64 by 2.1e-4 with scores of
      // deviation 3 (the result's own rounding) and 2.5e-4 with deviation 1, fp16 and int8 pages; rescaled only after growth by 2^6 it was 2.5e-4 and 2.7e-4, int8 2.9e-4, and 5 % faster.
      auto raise = [&](float mx) {
        mx = max_xor32(mx) * unit;
        mx = fabsf(mx) < 0x1p22f ? mx - PC_TOP : mx;           // floats beyond have steps that the largest half has no room for beside PC_TOP
        if (__builtin_amdgcn_ballot_w64(mx > m_run)) {
          const float m = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m);   // first visible keys: 0
          m_run = m;
          l_run *= alpha;
#pragma unroll
          for (int td = 0; td < NT; td++)
#pragma unroll
            for (int r = 0; r < 16; r++) o_acc[td][r] *= alpha;
        }
      };
      auto weights = [&](const f16_t &s, int tk) {
        float psum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
          const f4_t inv_v = I8 ? *(const f4_t *)&scl[buf][2][tk * 32 + 8 * r4 + 4 * lg] : f4_t{1.0f, 1.0f, 1.0f, 1.0f};
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; e++) p[e] = __builtin_amdgcn_exp2f(I8 ? s[r4 * 4 + e] - m_run : __builtin_fmaf(s[r4 * 4 + e], unit, -m_run));
#pragma unroll
          for (int e = 0; e < 4; e++) pf[tk][r4 / 2][r4 % 2 * 4 + e] = (_Float16)p[e];
          // fp16 pages: the sum is of the rounded weights, which multiply V.  int8: of the float ones; a weight that a small scale makes vanish as a half still counts.
          if constexpr (I8) {
#pragma unroll
            for (int e = 0; e < 4; e++) psum[e & 1] = __builtin_fmaf(p[e], inv_v[e], psum[e & 1]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; e += 2)
              psum[r4 & 1] = __builtin_amdgcn_fdot2(h2_t{(_Float16)p[e], (_Float16)p[e + 1]}, h2_t{(_Float16)1.0f, (_Float16)1.0f}, psum[r4 & 1], false);
          }
        }
        l_run += psum[0] + psum[1];
      };
      auto weigh = [&](int tk) {
#pragma unroll
        for (int hs = 0; hs < 2; hs++)
#pragma unroll
          for (int td = 0; td < NT; td++) {
            s4_t v[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int r = tk * 32 + hs * 16 + 8 * e + vrow, c = td * 64 + vcol;
              v[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t *)(vt + r * ROWB + v_at(r, c >> 4) * 16 + (c & 15)));
            }
            h8_t vf = __builtin_bit_cast(h8_t, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
            if constexpr (!I8 && !WHOLE) {
              u4_t w = __builtin_bit_cast(u4_t, vf);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t t = ((w[e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;   // the sign bit of halves that are not finite
                bad |= t;
                w[e] &= ~(t | (t - (t >> 15)));
              }
              vf = __builtin_bit_cast(h8_t, w);
            }
            o_acc[td] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[tk][hs], o_acc[td], 0, 0, 0);
          }
      };
      f16_t s0 = score(0);
      f16_t s1 = score(1);
      const float mx = finish(s0, 0);
      raise(fmaxf(mx, finish(s1, 1)));
      weights(s0, 0);
      weigh(0);
      weights(s1, 1);
      weigh(1);
      if constexpr (!I8 && !WHOLE) {
        if (__builtin_amdgcn_ballot_w64(bad != 0)) {
          for (int key = 0; key < PAGED_KEYS; key++) {
            const bool seen = sees(k0 + key) && (pm >> (key >> 4) & 1);
#pragma unroll
            for (int td = 0; td < NT; td++)
#pragma unroll
              for (int r4 = 0; r4 < 4; r4++) {
                const uint2 w = *(const uint2 *)(vt + key * ROWB + v_at(key, td * 4 + r4) * 16 + lg * 8);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  const uint32_t h = (e < 2 ? w.x : w.y) >> (16 * (e & 1)) & 0xffffu;
                  o_acc[td][r4 * 4 + e] += seen && (h & 0x7c00u) == 0x7c00u ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : 0.0f;
                }
              }
          }
        }
      }
    };
    // every key of the tile is masked for this wavefront (uniform)
    auto idle = [&]() {
      const int k0 = keys.tile(i) * PAGED_KEYS;
      return k0 > pos_hi || (a.window && k0 + PAGED_KEYS - 1 <= pos_lo - a.window && k0 >= a.sinks);
    };
    // Two loops, and each with its own copy of the accumulators' life: in one loop with both kinds of tiles they are copied twice a tile.
    bool whole = i < i_hi && begin();
    while (i < i_hi) {
      while (i < i_hi && whole) {
        tile(std::true_type());
        end();
        if (i < i_hi) whole = begin();
      }
      while (i < i_hi && !whole) {
        if (!idle()) tile(std::false_type());
        end();
        if (i < i_hi) whole = begin();
      }
    }

    if (it.parts > 1) {
      // Sums cross compute units on different XCDs: device-scope stores and loads (cache policy 16), counted once they are
      // acknowledged (the offset in the vector register, see sum_parts in gemm_tile.hip).
      constexpr int VALS = (HD / 2 + 4) * 64;                   // floats of one wavefront: O^T, then (m, l)
      const uint32_t slot = (uint32_t)VALS * 4 * 4, step = (uint32_t)KV * slot;
      const __amdgpu_buffer_rsrc_t rw = wave_buffer(a.ws + ((size_t)it.slot * 4 + wave) * VALS, (uint32_t)(it.parts - 1) * step + VALS * 4);
      const uint32_t mine = (uint32_t)it.part * step + lane * 16;
#pragma unroll
      for (int td = 0; td < NT; td++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
          const f4_t v = {o_acc[td][r4 * 4], o_acc[td][r4 * 4 + 1], o_acc[td][r4 * 4 + 2], o_acc[td][r4 * 4 + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v), rw, mine + (td * 4 + r4) * 1024, 0, 16);
        }
      const f4_t ml = {m_run, l_run, 0.0f, 0.0f};
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, ml), rw, mine + NT * 4 * 1024, 0, 16);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      int old = 0;
      if (lane == 0) old = __hip_atomic_fetch_add(&a.counters[it.slot * 4 + wave], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      old = __builtin_amdgcn_readfirstlane(old);
      if (old != it.parts - 1) return;
      if (lane == 0) __hip_atomic_store(&a.counters[it.slot * 4 + wave], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
      // two parts per round trip; past the last part the last one again, with weight zero
      m_run = -1e30f;
      l_run = 0.0f;
#pragma unroll
      for (int td = 0; td < NT; td++)
#pragma unroll
        for (int r = 0; r < 16; r++) o_acc[td][r] = 0.0f;
      for (int f = 0; f < it.parts; f += 2) {
        f4_t w[2], v[2][NT * 4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const uint32_t from = (uint32_t)min(f + u, it.parts - 1) * step + lane * 16;
          w[u] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, from + NT * 4 * 1024, 0, 16));
#pragma unroll
          for (int j = 0; j < NT * 4; j++) v[u][j] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, from + j * 1024, 0, 16));
        }
        const float m = fmaxf(m_run, fmaxf(w[0][0], w[1][0]));
        const float e = __builtin_amdgcn_exp2f(m_run - m);
        const float e0 = __builtin_amdgcn_exp2f(w[0][0] - m);   // a part without a visible key: 0
        const float e1 = f + 1 < it.parts ? __builtin_amdgcn_exp2f(w[1][0] - m) : 0.0f;
        m_run = m;
        l_run = l_run * e + (w[0][1] * e0 + w[1][1] * e1);
#pragma unroll
        for (int j = 0; j < NT * 4; j++)
#pragma unroll
          for (int x = 0; x < 4; x++) o_acc[j / 4][(j % 4) * 4 + x] = o_acc[j / 4][(j % 4) * 4 + x] * e + (v[0][j][x] * e0 + v[1][j][x] * e1);
      }
    }

    const float l = add_xor32(l_run), inv = l == 0.0f ? 0.0f : 1.0f / l;   // 0: the row sees nothing
    _Float16 *op = a.out + q_off;
#pragma unroll
    for (int td = 0; td < NT; td++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        // a lane half holds four of every eight neighbouring features; the halves exchange, so that each has all eight of every other group
        uint32_t w[2][2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const h2_t h = {(_Float16)(o_acc[td][(2 * j + u) * 4 + 2 * e] * inv), (_Float16)(o_acc[td][(2 * j + u) * 4 + 2 * e + 1] * inv)};
            w[u][e] = __builtin_bit_cast(uint32_t, h);
          }
        const auto lo = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const u4_t v = {lo[0], hi[0], lo[1], hi[1]};
        if (q_valid) *(u4_t *)(op + td * 32 + 16 * j + 8 * lg) = v;
      }
  }
};

// ---------------------------------------------------------------- one or a few new rows: PagedFew (paged_few.h)
constexpr int PF_THREADS = 256, PF_QROWS = 16;
constexpr int PF_BLOCKS = 512, PF_LEAST = 2;
constexpr int PF_SLOTS = 2 * PF_BLOCKS;
static_assert(PF_THREADS == FEW_THREADS && PF_QROWS == FEW_QROWS, "PagedFew");
// Which sequences these blocks take.  A tile of 64 keys costs a compute unit 0.6 us for 16 pairs here and 1.4 for a chunk of 128 (int8 0.55 and 1.5; heads of 64 0.37 and 0.8, 0.35 and 0.95), so
// that of up to 32 pairs their rows come cheaper: us, sequences of up to 16 pairs here | up to 32 | up to 64, heads of 128, fp16 and int8: 30 sequences of up to 2300 with 32 pairs each 56 | 55 | 56 and
// 55 | 40 | 40, behind 512 rows of another 87 | 80 | 81 and 103 | 81 | 80, four of 16000 77 | 61 | 61 and 82 | 51 | 50; with 48 pairs each 51 | 51 | 69 and 58 | 58 | 59.
constexpr int PF_PAIRS = 32;
// And a batch with little work has all of its rows here: a few keys on each of many compute units are done before a chunk's blocks have started and merged.
// us, one sequence, 32 heads of 128 over 8, chunks | these, new rows behind so many (tiles of 16 pairs and 64 keys): fp16, 64 behind 1024 (2176) 17.7 | 14.3, 128 behind 1024
// (4608) 18.6 | 15.0, 10 behind 16000 (6024) 41 | 29, 256 behind 500 (6144) 18.2 | 18.7, 64 behind 4000 (8192) 25.8 | 28.4; int8, 64 behind 4000 29.1 | 28.2, 128 behind 4000 (16640) 40 | 44; heads
// of 64, 64 behind 4000 18.0 | 17.7 and 21.5 | 20.1, 128 behind 4000 24.7 | 26.9 and 26.8 | 31.8.  Few rows behind a long context would gain beyond that: 16 behind 65000, int8 99 | 85.
template <int HD, bool I8> constexpr float PF_ALL = HD == 128 && !I8 ? 6100.0f : 12288.0f;

// Parts cost their merge: as many as the root of the tiles, some more.  (us, 64 rows behind 1936, heads of 128, least part and most parts 8 tiles, sqrt(t) | 4, sqrt(t) | 4, sqrt(2 t): 22.8 | 21.5 |
// 20.5; 57 behind 1024 18.4 | 17.1 | 17.3; one row behind 8000, heads of 64, 1 | 2 | 4 sqrt(t) / 2 .. 64 parts: 17.9 | 14.7 | 12.1, 2 sqrt(t) 10.5, 64 parts 14.1.)
__device__ __forceinline__ int chunk_parts(int tiles) { return (int)__builtin_amdgcn_sqrtf(2.0f * (float)tiles); }
__device__ __forceinline__ int few_parts(int tiles) { return min(FEW_MOST, (int)(2.0f * __builtin_amdgcn_sqrtf((float)tiles))); }

// Parts for this many blocks.  Sequences with several q tiles come from L2, and where there are few tiles in all a second block to a unit only adds merges.  us, PF_BLOCKS | half of
// them: int8, heads of 128, 128 rows behind 1024 (4608 pairs) 19.5 | 16.2, 10 behind 4000 17.5 | 15.0, 57 behind 1024 16.2 | 15.1, 64 behind 4000 (8192) 26.6 | 29.9; one row each of 16
// sequences of up to 2000 (3000) 15.8 | 17.5; heads of 64, fp16, 13.2 | 9.9, 12.3 | 10.5, 11.5 | 10.6, 17.5 | 18.7; 13.5 | 14.1.
__device__ __forceinline__ int few_blocks(const PagedAttnArgs &a, float pairs, float items) {
  return items > (float)a.pb.n_seqs * (float)a.n_kv_heads.d && pairs <= 10.0f * PF_BLOCKS ? PF_BLOCKS / 2 : a.few_blocks;
}

// Every sequence by the few-row blocks: one new row each, on the whole, or little work all in all.
template <int HD, bool I8> __global__ __launch_bounds__(PF_THREADS, HD == 64 ? 4 : I8 ? 3 : 2) void attn_paged_few_kernel(PagedAttnArgs a) {
  typedef PagedFew<HD, I8> A;
  __shared__ typename A::Smem sm;
  PagedItem it;
  const PagedSeq first = lane_seq(a.pb, 0);
  int id = blockIdx.x;
  PagedSum few = {0.0f, 0.0f};
  PagedShare share0 = {0, 0};
  bool falls = false;
  paged_walk(a.pb, first, [&](int b0, const PagedSeq &s) {
    falls |= s.n < 0;
    const PagedShare h = share_of<PF_QROWS>(a, s);
    if (!b0) share0 = h;
    few.add(h);
    return false;
  });
  if (__builtin_amdgcn_ballot_w64(falls)) return;            // no batch: there may be more parts than blocks, and what counts them would not get back to zero
  few.join((int)a.n_kv_heads.d);
  if (paged_item<PF_QROWS>(a, first, share0, id, 1, 0x7fffffff, few, few_blocks(a, few.pairs, few.items), PF_LEAST, few_parts, true, it)) A::item(a, it, sm);
}

// Chunks, and beside them the sequences that have PF_PAIRS and fewer: the ones are bound by the matrix cores and the vector unit, the others by memory.  Those come first, a
// block for every compute unit, and the chunks' blocks beside them, as many again.  us, 512 rows behind 1792 and 30 sequences of up to 2304 with one each, heads of 128, fp16 | int8: chunks
// alone 36 | 43, the others alone 41 | 26, together 57 | 60.  (On an
// earlier form of the kernels, with 57 | 64 like this: chunks first, two blocks to a unit 84 | 71; the others first 66 | 71.)
template <int HD, bool I8> __global__ __launch_bounds__(PC_THREADS, HD == 128 ? 2 : I8 ? 3 : 4) void attn_paged_chunk_kernel(PagedAttnArgs a) {
  __shared__ union {
    typename PagedChunk<HD, I8>::Smem chunk;
    typename PagedFew<HD, I8>::Smem few;
  } sm;
  PagedItem it;
  const PagedSeq first = lane_seq(a.pb, 0);
  const int n_rep = (int)a.n_rep.d;
  int id = blockIdx.x;
  // small: all of the batch by the few-row blocks; few, chunk: its sequences of up to PF_PAIRS pairs, and of more
  PagedSum small = {0.0f, 0.0f}, few = {0.0f, 0.0f}, chunk = {0.0f, 0.0f};
  PagedShare few0 = {0, 0}, chunk0 = {0, 0};
  bool falls = false;
  paged_walk(a.pb, first, [&](int b0, const PagedSeq &s) {
    falls |= s.n < 0;
    const PagedShare h = share_of<PF_QROWS>(a, s);
    const bool more = s.n * n_rep > PF_PAIRS;
    if (!b0) few0 = h;
    small.add(h);
    if (!more) few.add(h);
    if (__builtin_amdgcn_ballot_w64(more)) {
      const PagedShare c = share_of<PC_QROWS>(a, s);
      if (!b0) chunk0 = c;
      if (more) chunk.add(c);
    }
    return false;
  });
  if (__builtin_amdgcn_ballot_w64(falls)) return;            // as in attn_paged_few_kernel
  const int KV = (int)a.n_kv_heads.d;
  small.join(KV); few.join(KV); chunk.join(KV);
  // no sequence of more, or, with blocks enough for that, a batch of no more than PF_ALL pairs of a q tile and a key tile
  const bool all = chunk.items == 0.0f || (a.all_few && small.pairs <= PF_ALL<HD, I8>);
  if (all) few = small;
  if (few.items > 0.0f && paged_item<PF_QROWS>(a, first, few0, id, 1, all ? 0x7fffffff : PF_PAIRS, few, all ? few_blocks(a, few.pairs, few.items) : PF_BLOCKS / 2, PF_LEAST, few_parts, all, it))
    PagedFew<HD, I8>::item(a, it, sm.few);
  else if (!all && paged_item<PC_QROWS>(a, first, chunk0, id, PF_PAIRS + 1, 0x7fffffff, chunk, few.items > 0.0f ? PC_BLOCKS / 2 : PC_BLOCKS, PC_LEAST, chunk_parts, true, it))
    PagedChunk<HD, I8>::item(a, it, sm.chunk);
}

}  // namespace jsg

using namespace jsg;

extern "C" {

// counters of chunks (one for each of a block's wavefronts) and of few-row items, then the sums of cut items, one slot for every part
static size_t counter_bytes() { return ((size_t)PC_SLOTS * 4 + PF_SLOTS) * sizeof(int); }
static size_t chunk_sums(int head_dim) { return (size_t)PC_SLOTS * 4 * (head_dim / 2 + 4) * 64; }
static size_t few_sums(int head_dim) { return (size_t)PF_SLOTS * PF_QROWS * (head_dim + 4); }
size_t jsgrad_hip_attn_paged_workspace_bytes(int n_heads, int n_kv_heads, int head_dim) {
  (void)n_heads, (void)n_kv_heads;
  return counter_bytes() + (chunk_sums(head_dim) + few_sums(head_dim)) * sizeof(float);
}

int jsgrad_hip_attn_paged(const jsgrad_hip_pages_t *host_pages, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, const void *q, void *out,
                          int n_heads, int window, int sinks, void *workspace) {
  const char *who = "jsgrad_hip_attn_paged";
  PagedAttnArgs a = {};
  if (int e = paged_check(who, host_pages, row_starts, lengths, n_seqs, rows, &a.pb)) return e;
  const int KV = host_pages->n_kv_heads, HD = host_pages->head_dim;
  JSG_REQUIRE(q && out && workspace, "%s: null pointer argument", who);
  JSG_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)workspace % 16 == 0, "%s: q, out and workspace must be 16-byte aligned", who);
  JSG_REQUIRE(q != out, "%s: out must not be q", who);
  JSG_REQUIRE(n_heads > 0 && n_heads <= 65535 && n_heads % KV == 0, "%s: n_heads %d / n_kv_heads %d", who, n_heads, KV);
  JSG_REQUIRE(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", who, window, sinks);
  const int n_rep = n_heads / KV;
  JSG_REQUIRE((size_t)rows * n_rep < (size_t)1 << 30, "%s: %d rows of %d heads", who, rows, n_heads);
  a.pages_k = host_pages->pages_k; a.pages_v = host_pages->pages_v;
  a.scales_k = (const float *)host_pages->scales_k; a.scales_v = (const float *)host_pages->scales_v;
  a.q = (const _Float16 *)q; a.out = (_Float16 *)out;
  a.n_heads = n_heads;
  a.n_rep = divisor(n_rep); a.n_kv_heads = divisor(KV);
  a.window = window < 1 << 30 ? window : 1 << 30;             // no position is further: everything
  a.sinks = sinks < 1 << 30 ? sinks : 1 << 30;
  a.scale_log2 = (float)(1.0 / sqrt((double)HD)) * 1.4426950408889634f;
  a.counters = (int *)workspace;
  a.few_counters = a.counters + PC_SLOTS * 4;
  a.ws = (float *)((char *)workspace + counter_bytes());
  a.few_ws = a.ws + chunk_sums(HD);
  // 64 KB on their way to a compute unit are enough: one block of fp16 rows of 128, else two
  const bool i8 = host_pages->kind == JSGRAD_W_I8;
  a.few_blocks = HD == 128 && !i8 ? PF_BLOCKS / 2 : PF_BLOCKS;
  // As many blocks as there may be items and parts: every sequence fills its last q tile at worst, PF_PAIRS make several of the small ones, and what is no longer than the least
  // part is not cut.  Where that is enough for items of PF_QROWS pairs alone, the device decides whether there are others (PF_ALL, and whether any sequence has more than
  // PF_PAIRS).  The launch is of the smaller kernel where rows and the table's room say that there are none, however the rows are dealt out; us, chunk kernel | that, 10 to 64 new rows alone, fp16 7.5 | 5.1.
  // As many rows as sequences say nothing: they may be one each, or one prompt among sequences without new rows.  us, heads of 128, fp16 and int8: 16 with one row each 36 | 36 and 23 | 23, 100 73 | 73 and
  // 46 | 40 (three blocks to a unit), 256 111 | 110 and 83 | 72; 512 rows of one of 512 sequences 54 | 99 and 59 | 76, heads of 64 33 | 56 and 41 | 52.
  const int room_tiles = (paged_room(a.pb) + PAGED_KEYS - 1) / PAGED_KEYS, seqs = n_seqs < rows ? n_seqs : rows;
  const size_t few_items = KV * paged_most_tiles(rows, n_rep, seqs, PF_QROWS, PF_QROWS, 1), few_slots = room_tiles > PF_LEAST ? PF_SLOTS : 0;
  const size_t items = KV * paged_most_tiles(rows, n_rep, seqs, PC_QROWS, PF_QROWS, PF_PAIRS / PF_QROWS), slots = few_slots + (room_tiles > PC_LEAST ? PC_SLOTS : 0);
  const float all = HD == 64 ? (i8 ? PF_ALL<64, true> : PF_ALL<64, false>) : i8 ? PF_ALL<128, true> : PF_ALL<128, false>;
  const bool few = paged_few_only(rows, n_rep, PF_PAIRS, few_items, room_tiles, all);
  const size_t blocks = few ? few_items + few_slots : items + slots;
  a.all_few = few_items + few_slots <= blocks;
  JSG_REQUIRE(blocks < (size_t)PAGED_GRID, "%s: %d rows of %d heads", who, rows, n_heads);
  JSG_READY();
  const dim3 grid((unsigned)blocks);
#define JSG_PAGED(KERNEL, THREADS)                                                                    \
  do {                                                                                                \
    if (HD == 64 && i8) JSG_LAUNCH(PROF_ATTN_PAGED, (KERNEL<64, true>), grid, dim3(THREADS), 0, a);     \
    else if (HD == 64) JSG_LAUNCH(PROF_ATTN_PAGED, (KERNEL<64, false>), grid, dim3(THREADS), 0, a);     \
    else if (i8) JSG_LAUNCH(PROF_ATTN_PAGED, (KERNEL<128, true>), grid, dim3(THREADS), 0, a);           \
    else JSG_LAUNCH(PROF_ATTN_PAGED, (KERNEL<128, false>), grid, dim3(THREADS), 0, a);                  \
  } while (0)
  if (few) JSG_PAGED(attn_paged_few_kernel, PF_THREADS);
  else JSG_PAGED(attn_paged_chunk_kernel, PC_THREADS);
#undef JSG_PAGED
  return 0;
}

}  // extern "C"
