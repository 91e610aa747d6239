// A token for every row of logits, by the row's own temperature, min-p, top-k and top-p and a given uniform number (jsgrad_hip_sample_rows).
//
// With M the row's maximum, w = exp((x - M) / T); the entries with w >= min_p; of these the first top_k in the order (x descending, index ascending); of these the first whose mass
// reaches top_p of them all; the token is the first, by index, at which the running sum of what is left exceeds u times its total.  Or min_p last (jsgrad_hip_sample_rows_ordered): the mass that top_p is a share of
// counts entries that min_p drops afterwards.  Where top_p is 1 the place makes no difference, as w falls along the order.
//
// Which entry a sum ends at is a question of borders: with float sums, off by 1e-7, one draw in a hundred over a flat vocabulary would fall to a neighbour.  So a weight is
// made in 64 bits and held as a whole number of 2^-42: sums of up to 2^20 of them are exact and come out alike in any order, and the borders p Z and u Z are
// multiplied out in full.  What the rounding to 2^-42 leaves is a chance of some 1e-10 to land on another side than real numbers would.
//
// Three launches, as the maximum has to be known before a weight is, and masses before a border: maxima of parts of the rows; per part the candidates of the first top_k (k up to SR_FEW), or its mass by steps
// of an eighth of an octave below the maximum; one block a row for what lies on the step with a border.  One row of 128256 halves 18 us: 3.6, 6.3 and 8.5, launches and trips that wait for each other.  Sixteen
// rows with settings of their own 38 to 42, by inputs, of which up to 32 are the last block of a row with top_k = 1000 and top_p: 8 to get the row from beyond the unit's L2 and look it over, 5 for the parts' sums, 3 for the draw
// (52 with a look for each of the two borders).  256 rows with top_p = 0.95 (66 MB) 83: 14 (4.7 TB/s), 39 (33 million weights in 64 bits; histograms in several copies change nothing) and 34.
#include <type_traits>

#include "common.h"
#include "sample_rows.h"

namespace jsg {

constexpr int SR_THREADS = 1024, SR_TILE = 1024, SR_MOST = 1 << 20;
constexpr int SR_DIGIT = 11, SR_BINS = 1 << SR_DIGIT;
constexpr int SR_BITS = 42;                                  // of a weight behind the point
// Parts of a row: SR_PART entries times 1, 2 or 4, one block each.
constexpr int SR_PART_THREADS = 256, SR_PART = 8 * SR_PART_THREADS, SR_PARTS = SR_MOST / SR_PART;
// Depths are 256ths of an octave below the maximum, steps an eighth of one; what is further down than the last has no weight.
constexpr int SR_FINE = 256, SR_STEP = 32, SR_STEPS = 345, SR_STEPS_UP = 352, SR_DEEP = SR_STEPS * SR_STEP;
constexpr int SR_FEW = 256, SR_HELD = 256;                   // a top_k that goes by candidates, and how many of these a part may have
constexpr int SR_GROUPS = 2048, SR_LIST = 2048;              // groups whose maxima say where candidates begin; candidates of a row
constexpr int SR_ROOM = 8192;                                // entries of a step that are listed
// A call's parts are as short as leaves it at most SR_BLOCKS of them: two a CU.  With 1024, whose joins are longer, 16 rows of 128256 took 29 us
// with top_k = 200, 56 with top_k = 1000 and top_p = 0.9 and 45 with top_p = 0.95 alone; with 512 they took 27, 52 and 43.
constexpr size_t SR_BLOCKS = 512;

struct SampleRowsArgs {
  const void *logits;
  size_t stride;
  int n;
  const float *temperature, *top_p, *min_p, *uniforms;
  const int32_t *top_k;
  int32_t *tokens;
  float *probs;
  int order;                                                 // JSGRAD_MIN_P_FIRST or _LAST
  int parts, part, lanes;                                    // of a row, entries of one, and threads that share a group
  struct SampleFound *found;                                 // [rows]
  struct SamplePart *ws;                                     // [rows][parts]
};

// What the blocks of a row's parts leave: its parts' largest entries with their lowest indexes, maxima of groups of entries, and the candidates, n of them (more than SR_LIST: too many), in any order.
struct SampleFound {
  int n, pad[3];
  float best[SR_PARTS];
  int at[SR_PARTS];
  float group[SR_GROUPS];
  float x[SR_LIST];
  int index[SR_LIST];
};
struct SamplePart {
  uint64_t total, mass[SR_STEPS_UP];
  uint32_t count[SR_STEPS_UP];
};

// What a row's blocks have to find out.
enum SampleWay { SAMPLE_GREEDY, SAMPLE_FEW, SAMPLE_WHOLE, SAMPLE_STEPS };

// What is asked for of one row.
struct SampleRow {
  float top;                                                 // M
  bool infinite;                                             // M is: it alone has weight
  double from, scale;                                        // M again, log2(e) / T
  uint64_t least, late;                                      // weight that min_p asks for in front of the others, and behind them
  float top_p, u;
  int top_k;                                                 // 0: all
  SampleWay way;

  __device__ __forceinline__ SampleRow(const SampleRowsArgs &a, int r, float best) {
    // an array that is not given is another one in its place: five loads at once, without branches
    const float *const ts = a.temperature ? a.temperature : a.uniforms, *const ps = a.top_p ? a.top_p : a.uniforms, *const ms = a.min_p ? a.min_p : a.uniforms;
    const int32_t *const ks = a.top_k ? a.top_k : (const int32_t *)a.uniforms;
    const float t = ts[r], p0 = ps[r], m0 = ms[r], v = a.uniforms[r];
    const int k0 = ks[r];
    const float temperature = a.temperature ? t : 1.0f, p = a.top_p ? p0 : 1.0f, m = a.min_p ? m0 : 0.0f;
    const int k = a.top_k ? k0 : 0;
    top = best;
    infinite = best == INFINITY;
    from = infinite ? 0.0 : (double)best;
    scale = 1.4426950408889634 / (double)temperature;
    const uint64_t asked = m > 0.0f ? (uint64_t)ceil((double)fminf(m, 1.0f) * (double)(1ull << SR_BITS)) : 0;
    top_p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;
    u = v > 0.0f ? fminf(v, 0x1.fffffep-1f) : 0.0f;
    top_k = k > 0 && k < a.n ? k : 0;
    way = !(best > -INFINITY) || !(temperature >= 1e-6f) ? SAMPLE_GREEDY : top_k > 0 && top_k <= SR_FEW ? SAMPLE_FEW : top_k > 0 || top_p < 1.0f ? SAMPLE_STEPS : SAMPLE_WHOLE;
    late = a.order == JSGRAD_MIN_P_LAST && way != SAMPLE_WHOLE ? asked : 0;
    least = late ? 0 : asked;
  }
  static constexpr double MAGIC = 6755399441055744.0;        // 1.5 * 2^52: what it is added to comes out rounded to a whole number
  // log2 of an entry's weight: x - M is exact in 64 bits, the product off by 2^-52 of itself.  Entries that are not numbers are minus infinity, and that has no weight.
  __device__ double log_of(float x) const { return fmax(((double)x - from) * scale, -50.0); }
  // Where infinity is the maximum, it counts as 0 and everything else as minus infinity, with `from` 0.
  __device__ float finite(float x) const { return infinite ? (x == INFINITY ? 0.0f : -INFINITY) : x; }
  // The depth of an entry, SR_DEEP and more where it has no weight, whatever its share; never less for a smaller entry.
  __device__ int depth(float x) const {
    return -(int)(uint32_t)__double_as_longlong(__builtin_fma(log_of(finite(x)), (double)SR_FINE, MAGIC));
  }
  // The smallest entry at a depth below `limit`, 1 to SR_DEEP, as its key: each of a wavefront's lanes asks in one place, six times.
  __device__ uint32_t edge(int limit) const {
    uint32_t lo = 0x007fffffu, hi = top < INFINITY ? __float_as_uint(top + 0.0f) ^ ((uint32_t)(__float_as_int(top + 0.0f) >> 31) | 0x80000000u) : 0xff800000u;   // minus infinity, the maximum
    const uint32_t lane = threadIdx.x & 63;
    while (hi - lo > 1) {
      const uint32_t d = (hi - lo - 1) / 64 + 1, k = (uint32_t)min((uint64_t)lo + (uint64_t)(lane + 1) * d, (uint64_t)hi);
      const int first = __builtin_ctzll(__builtin_amdgcn_ballot_w64(depth(__uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k)) < limit));
      hi = (uint32_t)__builtin_amdgcn_readlane((int)k, first);
      if (first) lo = (uint32_t)__builtin_amdgcn_readlane((int)k, first - 1);
    }
    return hi;
  }
  // The weight, and the depth.  z = n / 256 + r with |r| <= 2^-9: the powers of 2^(1/256), and e^(r ln 2) to its fourth power, off by 2^-54; the last operation scales and rounds to a whole number.
  __device__ uint64_t weight(float x, const double *table, int &deep) const { return weight_of(finite(x), table, deep); }
  __device__ uint64_t weight_of(float x, const double *table, int &deep) const {
    const double z = log_of(x), t = __builtin_fma(z, (double)SR_FINE, MAGIC);
    const int n = (int)(uint32_t)__double_as_longlong(t);
    const double r = __builtin_fma(t - MAGIC, -1.0 / SR_FINE, z);
    double p = 9.6181291076284770e-3;                        // ln2^4 / 24
    p = __builtin_fma(p, r, 5.5504108664821580e-2);          // ln2^3 / 6
    p = __builtin_fma(p, r, 2.4022650695910072e-1);          // ln2^2 / 2
    p = __builtin_fma(p, r, 6.9314718055994531e-1);          // ln2
    p = __builtin_fma(p, r, 1.0);
    const double unit = __longlong_as_double((int64_t)((n >> 8) + SR_BITS + 1023) << 52);
    const double v = __builtin_fma(p * table[n & (SR_FINE - 1)], unit, 4503599627370496.0);
    const uint64_t whole = (uint64_t)__double_as_longlong(v) & 0xfffffffffffffull;
    deep = -n;
    return whole < least ? 0 : whole;
  }
  __device__ uint64_t weight(float x, const double *table) const {
    int unused;
    return weight(x, table, unused);
  }
  // The step on which weights fall below `late`, 1 and more: rounded they reach it from half a unit less on.
  __device__ int late_step() const { return -(int)rint((log2((double)late - 0.5) - SR_BITS) * SR_FINE) / SR_STEP; }
};
// 2^(i / 256), filled by the first 256 threads
__device__ __forceinline__ void sample_table(double *table) {
  if (threadIdx.x < SR_FINE) table[threadIdx.x] = exp2((double)threadIdx.x / SR_FINE);
}

// Order of floats as that of whole numbers; -0 is 0, what is not a number is minus infinity.
__device__ __forceinline__ float sample_clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
__device__ __forceinline__ uint32_t sample_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sample_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// An entry is kept where its key is above `key`, or is `key` and its index no more than `last`.
struct SampleCut {
  uint32_t key;
  int last;
  __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

struct SampleList {
  uint64_t place[SR_ROOM], w[SR_LIST];
  uint64_t near[SR_LIST], near_w[SR_LIST];                   // those about a border
  uint64_t mass[SR_STEPS_UP];
  uint32_t count[SR_STEPS_UP];
  uint64_t fine_mass[SR_STEP];
  uint32_t fine_count[SR_STEP];
  uint64_t part[SR_PARTS];
  int n, n_near;
};
struct SampleShared {
  union {
    struct {
      uint64_t mass[SR_BINS];
      uint32_t count[SR_BINS];
    } hist;                                                  // SampleBlock
    SampleList list;                                         // SampleLast
  };
  uint64_t wave[SR_THREADS / 64];
  uint64_t result[2];
};

template <int CTRL, int ROWS> __device__ __forceinline__ void add_dpp(uint64_t &v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, ROWS == 0xf), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, ROWS == 0xf);
  v += ((uint64_t)hi << 32) | lo;
}
// sums of this lane's value and those of the lanes below
__device__ __forceinline__ void wave_scan(uint64_t &s) {
  add_dpp<0x111, 0xf>(s); add_dpp<0x112, 0xf>(s); add_dpp<0x114, 0xf>(s); add_dpp<0x118, 0xf>(s);   // row_shr 1, 2, 4, 8
  add_dpp<0x142, 0xa>(s); add_dpp<0x143, 0xc>(s);            // row_bcast 15, 31
}
// Sum of the values of the threads before this one, and of all; contains barriers.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t &total, SampleShared &sm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t s = v;
  wave_scan(s);
  __syncthreads();
  if (lane == 63) sm.wave[wave] = s;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SR_THREADS / 64; w++) {
    const uint64_t o = sm.wave[w];
    if (w < wave) before += o;
    all += o;
  }
  total = all;
  return before + s - v;
}
__device__ __forceinline__ uint64_t sum_xor(uint64_t v, int lanes) {
  for (int off = 1; off < lanes; off <<= 1) {
    const uint32_t lo = __shfl_xor((uint32_t)v, off), hi = __shfl_xor((uint32_t)(v >> 32), off);
    v += ((uint64_t)hi << 32) | lo;
  }
  return v;
}

template <typename AT> struct SampleBlock {
  const AT *x;
  int n;
  SampleRow row;
  SampleShared &sm;
  const double *table;
  __device__ float at(int i) const { return sample_clean((float)x[i]); }

  // The cut behind the first entries, in the row's order, that `within` keeps and whose counts (or, MASS, weights) together reach `target`, 1 and more; everything where they do not.
  template <bool MASS> __device__ __forceinline__ SampleCut cut(uint64_t target, SampleCut within) {
    uint32_t prefix = 0;
    int shift = 32;
    uint64_t above = 0;                                      // of the keys above the prefix
    uint64_t here = 0;                                       // count of the last bin
    // the float of a half has 13 bits that say nothing
    const int least = sizeof(AT) == 2 ? 13 : 0;
    while (shift > least) {
      const int bits = min(SR_DIGIT, shift - least), from = shift - bits;
      __syncthreads();
      for (int b = threadIdx.x; b < SR_BINS; b += SR_THREADS) {
        sm.hist.mass[b] = 0;
        sm.hist.count[b] = 0;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += SR_THREADS) {
        const float v = at(i);
        const uint32_t k = sample_key(v);
        if ((shift < 32 && k >> shift != prefix) || !within.keeps(k, i)) continue;
        const uint32_t b = (k >> from) & ((1u << bits) - 1);
        atomicAdd(&sm.hist.count[b], 1u);
        if (MASS) atomicAdd((unsigned long long *)&sm.hist.mass[b], (unsigned long long)row.weight(v, table));
      }
      __syncthreads();
      // two bins to a thread, the highest first
      const int b1 = SR_BINS - 1 - 2 * (int)threadIdx.x, b0 = b1 - 1;
      const uint64_t v1 = MASS ? sm.hist.mass[b1] : sm.hist.count[b1], v0 = MASS ? sm.hist.mass[b0] : sm.hist.count[b0];
      uint64_t total;
      const uint64_t before = above + block_scan(v1 + v0, total, sm);
      if (threadIdx.x == 0) sm.result[0] = ~0ull;
      __syncthreads();
      if (before < target && before + v1 + v0 >= target) {
        const bool upper = before + v1 >= target;
        sm.result[0] = upper ? b1 : b0;
        sm.result[1] = upper ? before : before + v1;
      }
      __syncthreads();
      if (sm.result[0] == ~0ull) return within;              // all together fall short
      prefix = (shift < 32 ? prefix << bits : 0) | (uint32_t)sm.result[0];
      above = sm.result[1];
      here = sm.hist.count[sm.result[0]];
      shift = from;
    }
    SampleCut c;
    c.key = prefix << shift;
    if (least) c.key |= c.key & 0x80000000u ? 0 : (1u << least) - 1;
    const float v = sample_value(c.key);
    const uint64_t each = MASS ? row.weight(v, table) : 1;
    uint64_t r = (target - above + each - 1) / each;         // of `here` equal ones: 1 to that
    c.last = n;
    if (r < here) {
      for (int i0 = 0; i0 < n; i0 += SR_THREADS) {
        const int i = i0 + threadIdx.x;
        bool tie = false;
        if (i < n) {
          const uint32_t k = sample_key(at(i));
          tie = k == c.key && within.keeps(k, i);
        }
        uint64_t total;
        const uint64_t before = block_scan(tie ? 1 : 0, total, sm);
        if (r <= total) {
          if (tie && before + 1 == r) sm.result[0] = i;
          __syncthreads();
          c.last = (int)sm.result[0];
          break;
        }
        r -= total;
      }
    } else if (c.key == within.key) {
      c.last = within.last;
    }
    return c;
  }

  __device__ __forceinline__ uint64_t mass(SampleCut c) {
    uint64_t s = 0, total;
    for (int i = threadIdx.x; i < n; i += SR_THREADS) {
      const float v = at(i);
      if (c.keeps(sample_key(v), i)) s += row.weight(v, table);
    }
    block_scan(s, total, sm);
    return total;
  }

  // The first entry at which the running sum of what c, and min_p behind it, keep exceeds u of it all.
  __device__ uint64_t kept(SampleCut c, int i) const {
    const float v = at(i);
    const uint64_t w = c.keeps(sample_key(v), i) ? row.weight(v, table) : 0;
    return w < row.late ? 0 : w;
  }
  __device__ __forceinline__ int draw(SampleCut c, float u, uint64_t &weight, uint64_t &total) {
    const int tiles = (n + SR_TILE - 1) / SR_TILE;
    __syncthreads();
    for (int t = threadIdx.x; t < SR_MOST / SR_TILE; t += SR_THREADS) sm.hist.mass[t] = 0;
    __syncthreads();
    for (int t = 0; t < tiles; t++) {
      const int i = t * SR_TILE + threadIdx.x;
      const uint64_t w = i < n ? kept(c, i) : 0;
      if (w) atomicAdd((unsigned long long *)&sm.hist.mass[t], (unsigned long long)w);
    }
    __syncthreads();
    const uint64_t mine = sm.hist.mass[threadIdx.x], before = block_scan(mine, total, sm);
    const uint64_t target = sample_share(__float_as_uint(u), total, false);
    if (before <= target && before + mine > target) {
      sm.result[0] = threadIdx.x;
      sm.result[1] = before;
    }
    __syncthreads();
    const int t = (int)sm.result[0], i = t * SR_TILE + threadIdx.x;
    const uint64_t base = sm.result[1];
    uint64_t all;
    const uint64_t w = i < n ? kept(c, i) : 0;
    const uint64_t run = base + block_scan(w, all, sm);
    if (run <= target && run + w > target) {
      sm.result[0] = i;
      sm.result[1] = w;
    }
    __syncthreads();
    weight = sm.result[1];
    return (int)sm.result[0];
  }
};

// ---------------------------------------------------------------- parts
// Eight entries of a row from i on, as they are; VEC: rows begin at, and are apart by, whole 16 bytes.
template <typename AT, bool VEC> __device__ __forceinline__ void sample_load(const AT *x, int i, int n, float *f) {
  if (VEC && i + 8 <= n) {
    if constexpr (sizeof(AT) == 2) {
      const h8_t h = *as_global<h8_t>(x + i);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = (float)h[e];
    } else {
      const f4_t l = *as_global<f4_t>(x + i), h = *as_global<f4_t>(x + i + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) { f[e] = l[e]; f[4 + e] = h[e]; }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = i + e < n ? (float)x[i + e] : -INFINITY;
  }
}

__device__ __forceinline__ void sample_better(float &v, int &i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}
// The largest of the row's parts, and its lowest index; by every wavefront for itself
__device__ __forceinline__ void sample_best(const SampleFound &f, int parts, float &v, int &i) {
  v = -INFINITY;
  i = 0x7fffffff;
  for (int p = threadIdx.x & 63; p < parts; p += 64) sample_better(v, i, f.best[p], f.at[p]);
  for (int off = 32; off > 0; off >>= 1) sample_better(v, i, __shfl_xor(v, off), __shfl_xor(i, off));
}

// The largest entry of a part, and of each group of it.
template <typename AT, bool VEC> __global__ __launch_bounds__(SR_PART_THREADS) void sample_max_kernel(SampleRowsArgs a) {
  __shared__ float v_sh[SR_PART_THREADS / 64];
  __shared__ int i_sh[SR_PART_THREADS / 64];
  const AT *const x = (const AT *)a.logits + (size_t)blockIdx.y * a.stride;
  SampleFound &to = a.found[blockIdx.y];
  float v = -INFINITY;
  int at = 0x7fffffff;
  for (int j = 0; j < a.part; j += SR_PART) {
    const int i = blockIdx.x * a.part + j + threadIdx.x * 8;
    float f[8];
    sample_load<AT, VEC>(x, i, a.n, f);
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (f[e] > v) { v = f[e]; at = i + e; }
  }
  for (int off = 1; off < 64; off <<= 1) {
    if (off == a.lanes && (threadIdx.x & (off - 1)) == 0) to.group[(blockIdx.x * SR_PART_THREADS + threadIdx.x) / off] = v;
    sample_better(v, at, __shfl_xor(v, off), __shfl_xor(at, off));
  }
  if ((threadIdx.x & 63) == 0) {
    if (a.lanes == 64) to.group[(blockIdx.x * SR_PART_THREADS + threadIdx.x) / 64] = v;
    v_sh[threadIdx.x >> 6] = v;
    i_sh[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < SR_PART_THREADS / 64; w++) sample_better(v, at, v_sh[w], i_sh[w]);
    to.best[blockIdx.x] = v;
    to.at[blockIdx.x] = at;
    if (blockIdx.x == 0) to.n = 0;
  }
}

// A part once the maximum is known: its candidates, its mass, or masses and counts by steps below the maximum.
template <typename AT, bool VEC> __global__ __launch_bounds__(SR_PART_THREADS) void sample_part_kernel(SampleRowsArgs a) {
  __shared__ double table[SR_FINE];
  __shared__ uint64_t mass[SR_STEPS_UP];
  __shared__ uint32_t count[SR_STEPS_UP];
  __shared__ int held, upto, base;
  const int tid = threadIdx.x, lane = tid & 63;
  SampleFound &found = a.found[blockIdx.y];
  SamplePart &to = a.ws[(size_t)blockIdx.y * a.parts + blockIdx.x];
  const AT *const x = (const AT *)a.logits + (size_t)blockIdx.y * a.stride;
  const int groups = a.parts * SR_PART_THREADS / a.lanes;
  // asked for in front of everything that waits
  float f0[8], g0[4];
  sample_load<AT, VEC>(x, blockIdx.x * a.part + tid * 8, a.n, f0);
#pragma unroll
  for (int u = 0; u < 4; u++) g0[u] = found.group[min(tid + u * SR_PART_THREADS, groups - 1)];
  float best;
  int unused;
  sample_best(found, a.parts, best, unused);
  const SampleRow row(a, blockIdx.y, best);
  if (row.way == SAMPLE_GREEDY) return;
  if (row.way != SAMPLE_FEW) sample_table(table);
  for (int s = tid; s < SR_STEPS_UP; s += SR_PART_THREADS) { mass[s] = 0; count[s] = 0; }
  if (tid == 0) held = 0;
  __syncthreads();
  if (row.way == SAMPLE_FEW) {
    // The step on which the top_k-th largest of the groups' maxima is: as many entries are on it or above, so no entry further down is among the first top_k.
    for (int i = tid, u = 0; i < groups; i += SR_PART_THREADS, u++) {
      const int d = row.depth(u == 0 ? g0[0] : u == 1 ? g0[1] : u == 2 ? g0[2] : u == 3 ? g0[3] : found.group[i]);
      if (d < SR_DEEP) atomicAdd(&count[(uint32_t)d / SR_STEP], 1u);
    }
    __syncthreads();
    if (tid < 64) {
      uint32_t mine = 0, c[6];
#pragma unroll
      for (int e = 0; e < 6; e++) mine += c[e] = lane * 6 + e < SR_STEPS ? count[lane * 6 + e] : 0;
      uint32_t run = mine;
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(run, d);
        if (lane >= d) run += o;
      }
      run -= mine;
      int s = SR_STEPS - 1;
#pragma unroll
      for (int e = 0; e < 6; e++) {
        if (run < (uint32_t)row.top_k && run + c[e] >= (uint32_t)row.top_k) s = min(s, lane * 6 + e);
        run += c[e];
      }
      for (int off = 32; off > 0; off >>= 1) s = min(s, __shfl_xor(s, off));
      if (lane == 0) upto = s;
    }
    __syncthreads();
    const float from = sample_value(row.edge((upto + 1) * SR_STEP));
    float *const held_x = (float *)mass;                     // SR_HELD of each fit
    int *const held_at = (int *)(held_x + SR_HELD);
    static_assert(SR_STEPS_UP * 8 >= SR_HELD * 8, "candidates of a part");
    for (int j = 0; j < a.part; j += SR_PART) {
      const int i = blockIdx.x * a.part + j + tid * 8;
      float f[8];
      if (j == 0)
        for (int e = 0; e < 8; e++) f[e] = f0[e];
      else sample_load<AT, VEC>(x, i, a.n, f);
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (f[e] >= from) {
          const int slot = atomicAdd(&held, 1);              // in any order: the row's last block goes by entry and index
          if (slot < SR_HELD) { held_x[slot] = f[e]; held_at[slot] = i + e; }
        }
    }
    __syncthreads();
    const int n = held;
    if (n == 0) return;
    if (tid == 0) base = atomicAdd(&found.n, n);
    __syncthreads();
    if (n <= SR_HELD) {
      for (int i = tid; i < n; i += SR_PART_THREADS)
        if (base + i < SR_LIST) { found.x[base + i] = held_x[i]; found.index[base + i] = held_at[i]; }
    } else if (base < SR_LIST) {                             // once more, straight to where they go
      if (tid == 0) held = 0;
      __syncthreads();
      for (int j = 0; j < a.part; j += SR_PART) {
        const int i = blockIdx.x * a.part + j + tid * 8;
        float f[8];
        sample_load<AT, VEC>(x, i, a.n, f);
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (f[e] >= from) {
            const int slot = base + atomicAdd(&held, 1);
            if (slot < SR_LIST) { found.x[slot] = f[e]; found.index[slot] = i + e; }
          }
      }
    }
    return;
  }
  uint64_t sum = 0;
  for (int j = 0; j < a.part; j += SR_PART) {
    float f[8];
    if (j == 0)
      for (int e = 0; e < 8; e++) f[e] = f0[e];
    else sample_load<AT, VEC>(x, blockIdx.x * a.part + j + tid * 8, a.n, f);
    if (row.infinite)
      for (int e = 0; e < 8; e++) f[e] = row.finite(f[e]);
    uint64_t w[8];
    int d[8];
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = row.weight_of(f[e], table, d[e]);
    if (row.way != SAMPLE_STEPS) {
#pragma unroll
      for (int e = 0; e < 8; e++) sum += w[e];
      continue;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (d[e] < SR_DEEP) atomicAdd((unsigned long long *)&mass[(uint32_t)d[e] / SR_STEP], (unsigned long long)w[e]);
    if (row.top_k)
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (d[e] < SR_DEEP) atomicAdd(&count[(uint32_t)d[e] / SR_STEP], 1u);
  }
  if (row.way == SAMPLE_STEPS) {
    __syncthreads();
    for (int s = tid; s < SR_STEPS; s += SR_PART_THREADS) {
      to.mass[s] = mass[s];
      if (row.top_k) to.count[s] = count[s];
    }
    return;
  }
  sum = sum_xor(sum, 64);
  if (lane == 0) mass[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) to.total = mass[0] + mass[1] + mass[2] + mass[3];
}

// ---------------------------------------------------------------- the row's last block
// Entries by their place in the row's order: what is larger comes first.
__device__ __forceinline__ uint64_t sample_place(float x, int at) { return ((uint64_t)sample_key(x + 0.0f) << 32) | (0xffffffffu - (uint32_t)at); }
__device__ __forceinline__ float place_value(uint64_t p) { return sample_value((uint32_t)(p >> 32)); }
__device__ __forceinline__ int place_at(uint64_t p) { return (int)(0xffffffffu - (uint32_t)p); }

// take(i, number of the c places that come before place[i], the sum of their w): for every i, by one thread each.  As many threads to an i as there are for all.
template <typename Take> __device__ __forceinline__ void sample_before(const uint64_t *place, const uint64_t *w, int c, Take take) {
  int lanes = 64;
  while (lanes > 1 && lanes * c > SR_THREADS) lanes >>= 1;
  const int sub = threadIdx.x & (lanes - 1);
  for (int i = threadIdx.x / lanes; i < c; i += SR_THREADS / lanes) {
    const uint64_t mine = place[i];
    uint64_t sum = 0;
    uint32_t n = 0;
#pragma unroll 4
    for (int j = sub; j < c; j += lanes) {
      const bool first = place[j] > mine;
      sum += first ? w[j] : 0;
      n += first;
    }
    for (int off = 1; off < lanes; off <<= 1) n += __shfl_xor(n, off);
    sum = sum_xor(sum, lanes);
    if (sub == 0) take(i, n, sum);
  }
}

template <typename AT, bool VEC> struct SampleLast {
  const SampleRowsArgs &a;
  const SampleRow &row;
  const SampleFound &found;
  const SamplePart *ws;
  const AT *x;
  SampleShared &sm;
  SampleList &l;
  const double *table;

  // The step at which counts (or masses) of the steps reach `target`, 1 and more, and what is before it; SR_STEPS where they do not.  Contains barriers.
  template <typename V> __device__ int reach(const V *v, uint64_t target, uint64_t &before) {
    uint64_t total;
    const int s = threadIdx.x;
    const uint64_t mine = s < SR_STEPS ? v[s] : 0, run = block_scan(mine, total, sm);
    if (s == 0) { sm.result[0] = SR_STEPS; sm.result[1] = total; }
    __syncthreads();
    if (run < target && run + mine >= target) { sm.result[0] = s; sm.result[1] = run; }
    __syncthreads();
    before = sm.result[1];
    const int at = (int)sm.result[0];
    __syncthreads();
    return at;
  }

  // Of the first top_k among the candidates; false where there are more than the list has room for.
  __device__ __forceinline__ bool few(int c, const float (&v)[2], const int (&index)[2], int &token, uint64_t &weight, uint64_t &total) {
    const int tid = threadIdx.x;
    if (c > SR_LIST) return false;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int i = tid + u * SR_THREADS;
      if (i < c) {
        l.place[i] = sample_place(v[u], index[u]);
        l.w[i] = row.weight(v[u], table);
      }
    }
    __syncthreads();
    // l.near_w: the weight of those that are left; by index from here on
    uint64_t z = 0;
    sample_before(l.place, l.w, c, [&](int i, uint32_t n, uint64_t before) {
      const bool in = n < (uint32_t)row.top_k;
      l.near[i] = in ? before : ~0ull;
      if (in) z += l.w[i];
    });
    block_scan(z, z, sm);
    const uint64_t target = row.top_p < 1.0f ? max(sample_share(__float_as_uint(row.top_p), z, true), (uint64_t)1) : z;
    uint64_t left = 0;
    for (int i = tid; i < c; i += SR_THREADS) {
      const uint64_t w = l.near[i] < target && l.w[i] >= row.late ? l.w[i] : 0;
      l.near_w[i] = w;
      left += w;
    }
    block_scan(left, total, sm);
    for (int i = tid; i < c; i += SR_THREADS) l.near[i] = l.place[i] & 0xffffffffu;
    __syncthreads();
    const uint64_t at = sample_share(__float_as_uint(row.u), total, false);
    sample_before(l.near, l.near_w, c, [&](int i, uint32_t, uint64_t before) {
      const uint64_t w = l.near_w[i];
      if (before <= at && before + w > at) { sm.result[0] = (uint64_t)place_at(l.place[i]); sm.result[1] = w; }
    });
    __syncthreads();
    token = (int)sm.result[0];
    weight = sm.result[1];
    return true;
  }

  int list_lo, list_hi;                                      // the steps whose entries were listed, and whether they are all in the list
  bool fits;
  __device__ float least_of(int step) const { return sample_value(row.edge((step + 1) * SR_STEP)); }
  __device__ float most_of(int step) const { return step ? sample_value(row.edge(step * SR_STEP) - 1) : row.top; }
  // f(entry, index) for all of the row that are on these steps
  template <typename F> __device__ __forceinline__ void on_steps(int lo, int hi, F f) {
    const float from = least_of(hi), to = most_of(lo);
    constexpr int U = sizeof(AT) == 2 ? 4 : 2;
    for (int i0 = threadIdx.x * 8; i0 < a.n; i0 += U * SR_THREADS * 8) {
      float v[U][8];
#pragma unroll
      for (int u = 0; u < U; u++) sample_load<AT, VEC>(x, i0 + u * SR_THREADS * 8, a.n, v[u]);
      uint32_t hits = 0;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) hits |= (uint32_t)(v[u][e] >= from && v[u][e] <= to) << (u * 8 + e);
      for (; hits; hits &= hits - 1) {                       // few: asked for again
        const int b = __builtin_ctz(hits), i = i0 + (b >> 3) * SR_THREADS * 8 + (b & 7);
        f((float)x[i] + 0.0f, i);
      }
    }
  }
  // Lists the entries of steps; between barriers.
  __device__ __forceinline__ void list(int lo, int hi) {
    on_steps(lo, hi, [&](float v, int i) {
      const int slot = atomicAdd(&l.n, 1);
      if (slot < SR_ROOM) l.place[slot] = sample_place(v, i);
    });
    __syncthreads();
    list_lo = lo;
    list_hi = hi;
    fits = l.n <= SR_ROOM;
  }
  // f(key, index, weight, depth) for all entries of a step, one of those listed
  template <typename F> __device__ __forceinline__ void entries(int step, F f) {
    auto take = [&](float v, int i) {
      int d;
      const uint64_t w = row.weight(v, table, d);
      if (d / SR_STEP == step) f(sample_key(v), i, w, d);
    };
    if (!fits) return on_steps(step, step, take);
    for (int i = threadIdx.x; i < l.n; i += SR_THREADS) {
      const uint64_t p = l.place[i];
      take(place_value(p), place_at(p));
    }
  }
  // The cut among the entries of a step that `within` keeps at which their counts (MASS: weights) reach `target`, 1 and more, and the weight up to it; false where too many are on one depth.  Where the row has to be
  // gone over for that, everything from the step `first` on is listed.
  template <bool MASS> __device__ __forceinline__ bool border(int step, int first, uint64_t target, SampleCut within, SampleCut &cut, uint64_t &mass) {
    const int tid = threadIdx.x, lane = tid & 63;
    __syncthreads();
    if (tid < SR_STEP) { l.fine_mass[tid] = 0; l.fine_count[tid] = 0; }
    const bool again = step < list_lo || step > list_hi;
    if (tid == 0) { l.n_near = 0; if (again) l.n = 0; }
    __syncthreads();
    if (again) list(first, step);
    entries(step, [&](uint32_t key, int i, uint64_t w, int d) {
      if (!within.keeps(key, i)) return;
      atomicAdd((unsigned long long *)&l.fine_mass[(uint32_t)d % SR_STEP], (unsigned long long)w);
      atomicAdd(&l.fine_count[(uint32_t)d % SR_STEP], 1u);
    });
    __syncthreads();
    // the depth on which the border is, and what comes before it
    const uint64_t m = lane < SR_STEP ? l.fine_mass[lane] : 0, n = lane < SR_STEP ? l.fine_count[lane] : 0;
    uint64_t sum = m, count = n;
    wave_scan(sum);
    wave_scan(count);
    const int on = __builtin_ctzll(__builtin_amdgcn_ballot_w64((MASS ? sum : count) >= target) | 1ull << (SR_STEP - 1));
    auto at_on = [&](uint64_t v) { return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), on) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, on); };
    sum = at_on(sum - m);
    count = at_on(count - n);
    entries(step, [&](uint32_t key, int i, uint64_t w, int d) {
      if ((int)((uint32_t)d % SR_STEP) != on || !within.keeps(key, i)) return;
      const int slot = atomicAdd(&l.n_near, 1);
      if (slot < SR_LIST) { l.near[slot] = sample_place(sample_value(key), i); l.near_w[slot] = w; }
    });
    __syncthreads();
    if (l.n_near > SR_LIST) return false;
    sample_before(l.near, l.near_w, l.n_near, [&](int i, uint32_t k, uint64_t before) {
      const uint64_t w = l.near_w[i];
      if (MASS ? sum + before < target && sum + before + w >= target : count + k + 1 == target) { sm.result[0] = l.near[i]; sm.result[1] = sum + before + w; }
    });
    __syncthreads();
    cut = {(uint32_t)(sm.result[0] >> 32), place_at(sm.result[0])};
    mass = sm.result[1];
    __syncthreads();
    return true;
  }

  // By masses and counts of the steps: those above one step are kept whole, of that one what the cut keeps.  False where a step holds too many entries.
  __device__ __forceinline__ bool steps(int &token, uint64_t &weight, uint64_t &total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    SampleCut cut = {0, 0x7fffffff};
    int step = SR_STEPS;                                     // kept whole: the steps before this one
    uint64_t z = 0, extra = 0;                               // mass that is kept, and how much of it is on `step`
    const int late = row.late ? row.late_step() : SR_STEPS;  // a last border that is further down is not looked for: nothing of its step is left
    if (row.way == SAMPLE_STEPS) {
      for (int s = tid; s < SR_STEPS_UP; s += SR_THREADS) { l.mass[s] = 0; l.count[s] = 0; }
      list_lo = 1;
      list_hi = 0;
      __syncthreads();
      constexpr int E = (SR_STEPS + 63) / 64;                // a wavefront to a part, steps to its lanes
      uint64_t m[E] = {};
      uint32_t c[E] = {};
      auto sum = [&](auto &to, auto of, auto together) {     // so many parts at once; behind the last part: that one, and not counted
        constexpr int U = decltype(together)::value;
        for (int p0 = wave; p0 < a.parts; p0 += U * (SR_THREADS / 64)) {
          std::remove_reference_t<decltype(to[0])> v[U][E];
#pragma unroll
          for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < E; e++) v[u][e] = of(ws[min(p0 + u * (SR_THREADS / 64), a.parts - 1)])[min(e * 64 + lane, SR_STEPS_UP - 1)];
#pragma unroll
          for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < E; e++) to[e] += p0 + u * (SR_THREADS / 64) < a.parts ? v[u][e] : 0;
        }
      };
      auto masses = [](const SamplePart &p) { return p.mass; };
      auto counts = [](const SamplePart &p) { return p.count; };
      if (a.parts > 2 * (SR_THREADS / 64)) {
        sum(m, masses, std::integral_constant<int, 4>());
        if (row.top_k) sum(c, counts, std::integral_constant<int, 4>());
      } else {
        sum(m, masses, std::integral_constant<int, 1>());
        if (row.top_k) sum(c, counts, std::integral_constant<int, 1>());
      }
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int s = e * 64 + lane;
        if (s >= SR_STEPS) continue;
        if (m[e]) atomicAdd((unsigned long long *)&l.mass[s], (unsigned long long)m[e]);
        if (c[e]) atomicAdd(&l.count[s], c[e]);
      }
      __syncthreads();
      if (row.top_k) {
        uint64_t before;
        const int s = reach(l.count, (uint64_t)row.top_k, before);
        if (s < SR_STEPS && before + l.count[s] > (uint64_t)row.top_k) {
          // all that the first top_k are among, where it fits: a border by top_p is there too
          if ((row.top_p < 1.0f || s <= late) &&
              !border<false>(s, row.top_p < 1.0f && before + l.count[s] <= SR_ROOM ? 0 : s, (uint64_t)row.top_k - before, cut, cut, extra))
            return false;
          step = s;
        } else if (s < SR_STEPS) {
          step = s + 1;
        }
        if (tid == 0 && step < SR_STEPS) l.mass[step] = extra;
        for (int e = tid; e < SR_STEPS; e += SR_THREADS)
          if (e > step) l.mass[e] = 0;
        __syncthreads();
      }
      if (row.top_p < 1.0f) {
        uint64_t before;
        block_scan(tid < SR_STEPS ? l.mass[tid] : 0, z, sm);
        __syncthreads();
        const uint64_t target = max(sample_share(__float_as_uint(row.top_p), z, true), (uint64_t)1);
        const int s = reach(l.mass, target, before);
        if (before + l.mass[s] > target) {
          if (s <= late && !border<true>(s, s, target - before, s == step ? cut : SampleCut{0, 0x7fffffff}, cut, extra)) return false;
          step = s;
        } else if (s != step) {                              // the whole step, which is none that a cut went through
          step = s + 1;
          cut = SampleCut{0, 0x7fffffff};
          extra = 0;
        }
      }
      if (late < step) {                                     // steps above this one are kept whole, of those below nothing is
        if (late < list_lo || late > list_hi) fits = false;    // looked for once, so not listed
        step = late;
        cut = SampleCut{0, 0x7fffffff};
        extra = 1;
      }
      // what of every part is kept: whole steps, sixteen threads to a part, then those of the step with the cut
      for (int p = tid / 16; p < a.parts; p += SR_THREADS / 16) {
        uint64_t m = 0;
#pragma unroll 8
        for (int s = tid % 16; s < min(step, SR_STEPS); s += 16) m += ws[p].mass[s];
        m = sum_xor(m, 16);
        if (tid % 16 == 0) l.part[p] = m;
      }
      __syncthreads();
      if (extra)
        entries(step, [&](uint32_t key, int i, uint64_t w, int) {
          if (cut.keeps(key, i) && w >= row.late) atomicAdd((unsigned long long *)&l.part[i / a.part], (unsigned long long)w);
        });
    } else {
      for (int p = tid; p < a.parts; p += SR_THREADS) l.part[p] = ws[p].total;
    }
    __syncthreads();
    const uint64_t mine = tid < a.parts ? l.part[tid] : 0, run = block_scan(mine, total, sm);
    const uint64_t at = sample_share(__float_as_uint(row.u), total, false);
    if (run <= at && run + mine > at) { sm.result[0] = tid; sm.result[1] = run; }
    __syncthreads();
    // that part's entries, a few side by side to a thread
    const int p = (int)sm.result[0], each = a.part / SR_THREADS, i0 = p * a.part + tid * each;
    const uint64_t base = sm.result[1];
    uint64_t w[8], sum = 0, unused;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int i = i0 + e;
      w[e] = 0;
      if (e < each && i < a.n) {
        const float v = sample_clean((float)x[i]);
        int d;
        const uint64_t m = row.weight(v, table, d);
        if (d < step * SR_STEP || (d < (step + 1) * SR_STEP && extra && cut.keeps(sample_key(v), i) && m >= row.late)) w[e] = m;
      }
      sum += w[e];
    }
    uint64_t here = base + block_scan(sum, unused, sm);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (here <= at && here + w[e] > at) { sm.result[0] = (uint64_t)(i0 + e); sm.result[1] = w[e]; }
      here += w[e];
    }
    __syncthreads();
    token = (int)sm.result[0];
    weight = sm.result[1];
    return true;
  }
};

template <typename AT, bool VEC> __global__ __launch_bounds__(SR_THREADS) void sample_last_kernel(SampleRowsArgs a) {
  __shared__ SampleShared sm;
  __shared__ double table[SR_FINE];
  const int r = blockIdx.x;
  const SampleFound &found = a.found[r];
  const SamplePart *const ws = a.ws + (size_t)r * a.parts;
  const AT *const x = (const AT *)a.logits + (size_t)r * a.stride;
  // asked for before anyone knows whether it is wanted
  const int n_found = found.n;
  const float vs[2] = {found.x[threadIdx.x], found.x[threadIdx.x + SR_THREADS]};
  const int indexes[2] = {found.index[threadIdx.x], found.index[threadIdx.x + SR_THREADS]};
  sample_table(table);
  float best;
  int token;
  sample_best(found, a.parts, best, token);
  const SampleRow row(a, r, best);
  float prob = 1.0f;
  if (!(best > -INFINITY)) {
    token = -1;
    prob = 0.0f;
  } else if (row.way != SAMPLE_GREEDY) {
    __syncthreads();
    SampleLast<AT, VEC> last = {a, row, found, ws, x, sm, sm.list, table, 1, 0, false};
    uint64_t w, total;
    if (!(row.way == SAMPLE_FEW ? last.few(n_found, vs, indexes, token, w, total) : last.steps(token, w, total))) {
      // many entries side by side in the order, where the cut is: digit by digit over the whole row
      SampleBlock<AT> b = {x, a.n, row, sm, table};
      SampleCut c = {0, 0x7fffffff};
      __syncthreads();
      if (row.top_k) c = b.template cut<false>((uint64_t)row.top_k, c);
      if (row.top_p < 1.0f) c = b.template cut<true>(max(sample_share(__float_as_uint(row.top_p), b.mass(c), true), (uint64_t)1), c);
      token = b.draw(c, row.u, w, total);
    }
    prob = (float)((double)w / (double)total);
  }
  if (threadIdx.x == 0) {
    a.tokens[r] = token;
    if (a.probs) a.probs[r] = prob;
  }
}

// Entries of a part: enough blocks for the chip where there are few rows, fewer and longer parts where there are many.
static int sample_part(int rows, int n) {
  for (int g = 1; g < 4; g *= 2)
    if ((size_t)rows * ((n + SR_PART * g - 1) / (SR_PART * g)) <= SR_BLOCKS) return SR_PART * g;
  return SR_PART * 4;
}

// jsgrad_hip_sample_rows and _sample_rows_ordered
static int sample_rows(const char *who, const void *logits, int rows, int n, size_t row_stride, int act, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                       int order, const float *uniforms, int32_t *tokens_out, float *probs_out, void *workspace) {
  JSG_REQUIRE(logits && uniforms && tokens_out && workspace, "%s: null pointer argument", who);
  JSG_REQUIRE(act == JSGRAD_F16 || act == JSGRAD_F32, "%s: unknown activation dtype %d", who, act);
  JSG_REQUIRE(rows > 0 && rows <= 65535, "%s: %d rows (1 to 65535)", who, rows);
  JSG_REQUIRE(n > 0 && n <= SR_MOST, "%s: %d logits (1 to %d)", who, n, SR_MOST);
  JSG_REQUIRE(row_stride >= (size_t)n && row_stride < (size_t)1 << 40, "%s: a stride of %zu for rows of %d", who, row_stride, n);
  JSG_REQUIRE((uintptr_t)logits % (act == JSGRAD_F16 ? 2 : 4) == 0, "%s: logits must be aligned to their type", who);
  JSG_REQUIRE(((uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)uniforms | (uintptr_t)tokens_out | (uintptr_t)probs_out) % 4 == 0,
              "%s: the rows' arrays must be 4-byte aligned", who);
  JSG_REQUIRE((uintptr_t)workspace % 16 == 0, "%s: workspace must be 16-byte aligned", who);
  JSG_REQUIRE(order == JSGRAD_MIN_P_FIRST || order == JSGRAD_MIN_P_LAST, "%s: order %d (min-p first or last)", who, order);
  JSG_READY();
  SampleRowsArgs a = {logits, row_stride, n, temperature, top_p, min_p, uniforms, top_k, tokens_out, probs_out, order};
  a.part = sample_part(rows, n);
  a.parts = (n + a.part - 1) / a.part;
  a.lanes = 1;                                               // of the groups, as many as are no more than four times SR_FEW
  while (a.lanes < 64 && a.parts * (SR_PART_THREADS / a.lanes) > 4 * SR_FEW) a.lanes *= 2;
  a.found = (SampleFound *)workspace;
  a.ws = (SamplePart *)(a.found + rows);
  const size_t size = act == JSGRAD_F16 ? 2 : 4;
  const bool vec = (uintptr_t)logits % 16 == 0 && row_stride * size % 16 == 0;
  const dim3 parts((unsigned)a.parts, (unsigned)rows), block(SR_PART_THREADS);
#define JSG_SAMPLE(AT, VEC)                                                                           \
  do {                                                                                                \
    JSG_LAUNCH(PROF_SAMPLE, (sample_max_kernel<AT, VEC>), parts, block, 0, a);                          \
    JSG_LAUNCH(PROF_SAMPLE, (sample_part_kernel<AT, VEC>), parts, block, 0, a);                         \
    JSG_LAUNCH(PROF_SAMPLE, (sample_last_kernel<AT, VEC>), dim3(rows), dim3(SR_THREADS), 0, a);         \
  } while (0)
  if (act == JSGRAD_F16 && vec) JSG_SAMPLE(_Float16, true);
  else if (act == JSGRAD_F16) JSG_SAMPLE(_Float16, false);
  else if (vec) JSG_SAMPLE(float, true);
  else JSG_SAMPLE(float, false);
#undef JSG_SAMPLE
  return 0;
}

}  // namespace jsg

using namespace jsg;

extern "C" {

size_t jsgrad_hip_sample_rows_workspace_bytes(int rows, int n) {
  if (rows <= 0 || n <= 0 || n > SR_MOST) return 0;
  // of all numbers of rows up to this: fewer rows have shorter parts, up to SR_BLOCKS of them
  const size_t longest = (size_t)rows * ((n + 4 * SR_PART - 1) / (4 * SR_PART)), shortest = (size_t)rows * ((n + SR_PART - 1) / SR_PART);
  return (size_t)rows * sizeof(SampleFound) + sizeof(SamplePart) * (shortest < SR_BLOCKS ? shortest : longest < SR_BLOCKS ? SR_BLOCKS : longest);
}

int jsgrad_hip_sample_rows(const void *logits, int rows, int n, size_t row_stride, int act, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                           const float *uniforms, int32_t *tokens_out, float *probs_out, void *workspace) {
  return sample_rows("jsgrad_hip_sample_rows", logits, rows, n, row_stride, act, temperature, top_k, top_p, min_p, JSGRAD_MIN_P_FIRST, uniforms, tokens_out, probs_out, workspace);
}

int jsgrad_hip_sample_rows_ordered(const void *logits, int rows, int n, size_t row_stride, int act, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                                   int order, const float *uniforms, int32_t *tokens_out, float *probs_out, void *workspace) {
  return sample_rows("jsgrad_hip_sample_rows_ordered", logits, rows, n, row_stride, act, temperature, top_k, top_p, min_p, order, uniforms, tokens_out, probs_out, workspace);
}

}  // extern "C"
