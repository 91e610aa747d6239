// Grouped-query attention of a ragged batch of new rows over a paged KV cache (jsgrad_hip_attn_paged).
//
// Row i of a sequence sits at position p and sees the keys j <= p that have a page and, with a window, are among the last `window` of them or
// among the first `sinks`: out = sum_j softmax_j(q . K_j / sqrt(HD)) V_j, zeros where it sees none.  Reference semantics of the sum:
// scaled_dot_product_attention (jsgrad/tensor.ts:3920-3934); windows, sinks and pages have no counterpart there.
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

// ---------------------------------------------------------------- which work a block has
//
// A launch's items are (sequence, q tile, kv head); a q tile is QROWS (position, query head) pairs of a kv head, row = position * n_rep + head.  Long
// ones are cut along the keys, so that the parts of a launch have about the same number of key tiles whatever the lengths of its sequences are
// (paged_target).  The host knows neither lengths nor row starts: every wavefront goes over them, a sequence to a lane, and finds its block's item.
// Block numbers have the kv heads innermost: blocks are dealt to the eight XCDs in turn, so that with eight kv heads each XCD has one, all q tiles of which
// share its K and V in that L2, and all XCDs have the same work.  The q tiles with the most keys come first within a sequence.
struct PagedItem {
  PagedSeq s;
  int b, g, qt, part, parts, slot;       // slot: of part 0 in the workspace; part p's is slot + p * n_kv_heads
};
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

// ---------------------------------------------------------------- one or a few new rows
//
// Block = 4 wavefronts, 16 (position, query head) pairs of one kv head of one sequence.  Bound by memory: each wavefront walks its own steps of 32 keys, K rows to registers as
// they are the matrix operand, V rows through registers into the wavefront's own LDS, from where the transposing reads take them; the next step's K rows are asked
// for as soon as the scores are made, its V rows as soon as those are in LDS, and nothing is waited for but that.  The wavefronts meet once, at the end.
// The matrix instruction's 16 columns are the rows, so that a lane has four scores of each 16 keys of one row, and its weights are the operand of O^T = V^T . P^T as they lie.
// Parts of an item are merged by the last of its blocks to arrive.
// 3 sequences of 65000, 32 heads of 128 over 8, fp16: 117 us = 5.8 TB/s, as fast as a launch that only reads.  16 of 435 to 4352, int8 (81 MB) 21.4 us = 3.8 TB/s: 4 us of launch, some 3 each
// until the first keys are there and for the merge.
constexpr int PF_THREADS = 256, PF_QROWS = 16;
constexpr int PF_BLOCKS = 512, PF_LEAST = 2;
constexpr int PF_SLOTS = 2 * PF_BLOCKS, PF_MOST = 64;      // parts of an item: a lane for each
constexpr float PF_TOP = 15.0f;                            // a row's largest weight is 2^15: halves are normal numbers down to 2^-29 of it
// Which sequences these blocks take.  A tile of 64 keys costs a compute unit 0.6 us for 16 pairs here and 1.4 for a chunk of 128 (int8 0.55 and 1.5; heads of 64 0.37 and 0.8, 0.35 and 0.95), so
// that of up to 32 pairs their rows come cheaper: us, sequences of up to 16 pairs here | up to 32 | up to 64, heads of 128, fp16 and int8: 30 sequences of up to 2300 with 32 pairs each 56 | 55 | 56 and
// 55 | 40 | 40, behind 512 rows of another 87 | 80 | 81 and 103 | 81 | 80, four of 16000 77 | 61 | 61 and 82 | 51 | 50; with 48 pairs each 51 | 51 | 69 and 58 | 58 | 59.
constexpr int PF_PAIRS = 32;
// And a batch with little work has all of its rows here: a few keys on each of many compute units are done before a chunk's blocks have started and merged.
// us, one sequence, 32 heads of 128 over 8, chunks | these, new rows behind so many (tiles of 16 pairs and 64 keys): fp16, 64 behind 1024 (2176) 17.7 | 14.3, 128 behind 1024
// (4608) 18.6 | 15.0, 10 behind 16000 (6024) 41 | 29, 256 behind 500 (6144) 18.2 | 18.7, 64 behind 4000 (8192) 25.8 | 28.4; int8, 64 behind 4000 29.1 | 28.2, 128 behind 4000 (16640) 40 | 44; heads
// of 64, 64 behind 4000 18.0 | 17.7 and 21.5 | 20.1, 128 behind 4000 24.7 | 26.9 and 26.8 | 31.8.  Few rows behind a long context would gain beyond that: 16 behind 65000, int8 99 | 85.
template <int HD, bool I8> constexpr float PF_ALL = HD == 128 && !I8 ? 6100.0f : 12288.0f;

template <int HD, bool I8> struct PagedFew {
  static constexpr int NW = 4, KEYS = 32, ROWB = HD * 2;
  static constexpr int VROW = ROWB + 32;                     // bytes between V rows in LDS: eight banks further each, so that the reads of 16 rows by 32 bytes meet all banks alike
  static constexpr int NT = HD / 16, KS = HD / 32;           // 16-feature tiles of the output, matrix instructions per 16 keys
  static constexpr int OROW = HD + 4;                        // floats between rows of a wavefront's sums in LDS
  static constexpr int GK = KS / (I8 ? 2 : 1), LPR = HD / (I8 ? 16 : 8), GV = LPR / 4;   // 16-byte loads of 16 keys' K and V; lanes per V row
  static constexpr int SLOT = PF_QROWS * (HD + 4);           // floats of a part: the rows' sums, then (m, l, -, -) of each
  struct Smem {
    union {
      unsigned char v[KEYS * VROW];
      float o[PF_QROWS * OROW];
    } wave[NW];
    float m[NW][PF_QROWS], l[NW][PF_QROWS];
    float w[PF_QROWS][PF_MOST], inv[PF_QROWS];
    f4_t fold[PF_THREADS];
    int is_last;
  };
  // Must be called by every thread of the block (it contains barriers).
  static __device__ void item(const PagedAttnArgs &a, const PagedItem &it, Smem &sm) {
    const float scale_log2 = a.scale_log2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lq = lane >> 4;
    const int n_rep = (int)a.n_rep.d, KV = (int)a.n_kv_heads.d, room = paged_room(a.pb), g = it.g;
    const int rows = it.s.n * n_rep, p0 = paged_pos(it.s, 0), q0 = it.qt * PF_QROWS, nr = min(PF_QROWS, rows - q0);
    const int pos_lo = p0 + a.n_rep.div(q0), pos_hi = p0 + a.n_rep.div(q0 + nr - 1);
    const PagedKeys keys = paged_keys(pos_lo, pos_hi, room, a.window, a.sinks);
    int i_lo = 0, i_hi = keys.n;
    if (it.parts > 1) {
      const int per = (keys.n + it.parts - 1) / it.parts;
      i_lo = min(it.part * per, keys.n);
      i_hi = min(i_lo + per, keys.n);
    }
    auto out_row = [&](int r) {                              // of pair q0 + r
      const int qs = a.n_rep.div(q0 + r);
      return ((size_t)(it.s.start + qs) * a.n_heads + g * n_rep + q0 + r - qs * n_rep) * HD;
    };
    const int qpos = p0 + a.n_rep.div(q0 + min(l16, nr - 1));  // columns past the end repeat the last row and are never stored
    const int sees_from = a.window ? qpos - a.window : -1, sees_to = a.window ? a.sinks : 0;
    auto sees = [&](int key) { return (key <= qpos) & ((key > sees_from) | (key < sees_to)); };

    auto key_of = [&](int st) { return keys.tile(st >> 1) * PAGED_KEYS + (st & 1) * KEYS; };
    const int st_end = 2 * i_hi;
    u4_t kr[2][GK], vr[2][GV];
    f4_t ks[2], vs[2];
    int id[2], next[2];
    auto ids = [&](int st, int *to) {
#pragma unroll
      for (int h = 0; h < 2; h++) to[h] = st < st_end ? page_uniform(a.pb, it.b, key_of(st) + 16 * h) : -1;
    };
    auto load_k = [&](int st, const int *page) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const size_t row = paged_row(a.pb, KV, max(page[h], 0), g, key_of(st) + 16 * h);   // a missing page: page 0, masked
#pragma unroll
        for (int c = 0; c < GK; c++)
          kr[h][c] = *as_global<u4_t>((const unsigned char *)a.pages_k + (row + l16) * (I8 ? HD : ROWB) + (lq + 4 * c) * 16);
        if constexpr (I8) ks[h] = *as_global<f4_t>(a.scales_k + row + 4 * lq);
      }
    };
    auto load_v = [&](int st, const int *page) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const size_t row = paged_row(a.pb, KV, max(page[h], 0), g, key_of(st) + 16 * h);
#pragma unroll
        for (int c = 0; c < GV; c++)
          vr[h][c] = *as_global<u4_t>((const unsigned char *)a.pages_v + (row + c * (64 / LPR) + lane / LPR) * (I8 ? HD : ROWB) + lane % LPR * 16);
        if constexpr (I8) vs[h] = *as_global<f4_t>(a.scales_v + row + 4 * lq);
      }
    };

    int st = 2 * i_lo + wave;
    ids(st, id);
    if (st < st_end) {
      load_k(st, id);
      load_v(st, id);
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
      ids(st + NW, next);
      const int k0 = key_of(st);
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
      if constexpr (decltype(more)::value) load_k(st + NW, next);
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
      // value r of s[h] is key k0 + 16 h + 4 lq + r of row l16
      const bool masked = k0 + KEYS - 1 > pos_lo || (id[0] | id[1]) < 0 || (a.window && k0 <= pos_hi - a.window && k0 + KEYS > a.sinks);
      if (masked) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            s[h][r] = (sees(k0 + 16 * h + 4 * lq + r) & (id[h] >= 0)) ? s[h][r] : -INFINITY;
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
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][r] - m_run, unit, PF_TOP));
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
      if constexpr (decltype(more)::value) load_v(st + NW, next);
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
          const bool seen = sees(k0 + key) && (key < 16 ? id[0] : id[1]) >= 0;
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
      id[0] = next[0];
      id[1] = next[1];
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
      for (int i = tid; i < pieces; i += PF_THREADS) {
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
    for (int i = tid; i < pieces; i += PF_THREADS) {
      f4_t sum;
      float M, L;
      const int r = i / (HD / 4), c = i % (HD / 4);
      block_sum(r, c, sum, M, L);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, sum), rw, (uint32_t)it.part * part_bytes + i * 16, 0, 16);
      if (c == 0) {
        const f4_t ml = {M, L, 0.0f, 0.0f};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, ml), rw, (uint32_t)it.part * part_bytes + (PF_QROWS * HD + r * 4) * 4, 0, 16);
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
      const f4_t ml = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)min(lane, it.parts - 1) * part_bytes + (PF_QROWS * HD + r * 4) * 4, 0, 16));
      const float m = lane < it.parts ? ml[0] : -1e30f, M = wave_max(m), e = lane < it.parts ? __builtin_amdgcn_exp2f((m - M) * unit) : 0.0f;
      const float L = wave_sum(lane < it.parts ? ml[1] * e : 0.0f);
      sm.w[r][lane] = e;
      if (lane == 0) sm.inv[r] = L == 0.0f ? 0.0f : 1.0f / L;
    }
    lds_barrier();
    // a thread per four features of a row; where those are fewer than threads, groups of threads share the parts
    const int groups = pieces < PF_THREADS ? PF_THREADS / pieces : 1, mine = groups > 1 ? tid / pieces : 0;
    for (int i0 = groups > 1 ? tid - mine * pieces : tid; i0 < pieces; i0 += PF_THREADS) {
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

// Parts cost their merge: as many as the root of the tiles, some more.  (us, 64 rows behind 1936, heads of 128, least part and most parts 8 tiles, sqrt(t) | 4, sqrt(t) | 4, sqrt(2 t): 22.8 | 21.5 |
// 20.5; 57 behind 1024 18.4 | 17.1 | 17.3; one row behind 8000, heads of 64, 1 | 2 | 4 sqrt(t) / 2 .. 64 parts: 17.9 | 14.7 | 12.1, 2 sqrt(t) 10.5, 64 parts 14.1.)
__device__ __forceinline__ int chunk_parts(int tiles) { return (int)__builtin_amdgcn_sqrtf(2.0f * (float)tiles); }
__device__ __forceinline__ int few_parts(int tiles) { return min(PF_MOST, (int)(2.0f * __builtin_amdgcn_sqrtf((float)tiles))); }

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
