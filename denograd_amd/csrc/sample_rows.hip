// A token for every row of logits, by the row's own temperature, min-p, top-k and top-p and a given uniform number (jsgrad_hip_sample_rows).
//
// With M the row's maximum, w = exp((x - M) / T); the entries with w >= min_p; of these the first top_k in the order (x descending, index ascending); of these the first whose mass
// reaches top_p of them all; the token is the first, by index, at which the running sum of what is left exceeds u times its total.
//
// Which entry a sum ends at is a question of borders: with float sums, off by 1e-7, one draw in a hundred over a flat vocabulary would fall to a neighbour.  So a weight is
// made in 64 bits and held as a whole number of 2^-42: sums of up to 2^20 of them are exact and come out alike in any order, and the borders p Z and u Z are
// multiplied out in full.  What the rounding to 2^-42 leaves is a chance of some 1e-10 to land on another side than real numbers would.
#include "common.h"
#include "sample_rows.h"

namespace jsg {

constexpr int SR_THREADS = 1024, SR_TILE = 1024, SR_MOST = 1 << 20;
constexpr int SR_DIGIT = 11, SR_BINS = 1 << SR_DIGIT;
constexpr int SR_BITS = 42;                                  // of a weight behind the point

struct SampleRowsArgs {
  const void *logits;
  size_t stride;
  int n;
  const float *temperature, *top_p, *min_p, *uniforms;
  const int32_t *top_k;
  int32_t *tokens;
  float *probs;
};

// What is asked for of one row.
struct SampleRow {
  float top;                                                 // M
  double scale;                                              // log2(e) / T
  double min_p;
  // x - M is exact in 64 bits, the product off by 2^-52 of itself
  __device__ uint64_t weight(float x) const {
    if (x == top) return 1ull << SR_BITS;
    if (!(x > -INFINITY) || top == INFINITY) return 0;
    const double w = exp2(((double)x - (double)top) * scale);
    return w < min_p ? 0 : (uint64_t)rint(ldexp(w, SR_BITS));
  }
};

// Order of floats as that of whole numbers; -0 is 0, what is not a number is minus infinity.
__device__ __forceinline__ float sample_clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
__device__ __forceinline__ uint32_t sample_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// An entry is kept where its key is above `key`, or is `key` and its index no more than `last`.
struct SampleCut {
  uint32_t key;
  int last;
  __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

struct SampleShared {
  union {
    struct {
      uint64_t mass[SR_BINS];
      uint32_t count[SR_BINS];
    } hist;
    uint64_t tile[SR_MOST / SR_TILE];
  };
  uint64_t wave[SR_THREADS / 64];
  uint64_t result[2];
  float best[SR_THREADS / 64];
  int at[SR_THREADS / 64];
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
  return ((uint64_t)hi << 32) | lo;
}
// Sum of the values of the threads before this one, and of all; contains barriers.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t &total, SampleShared &sm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t s = v;
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = shfl_up64(s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 63) sm.wave[wave] = s;
  __syncthreads();
  uint64_t before = 0, all = 0;
  for (int w = 0; w < SR_THREADS / 64; w++) {
    if (w < wave) before += sm.wave[w];
    all += sm.wave[w];
  }
  total = all;
  return before + s - v;
}

template <typename AT> struct SampleBlock {
  const AT *x;
  int n;
  SampleRow row;
  SampleShared &sm;
  __device__ float at(int i) const { return sample_clean((float)x[i]); }

  // The cut behind the first entries, in the row's order, that `within` keeps and whose counts (or, MASS, weights) together reach `target`, 1 and more; everything where they do not.
  template <bool MASS> __device__ SampleCut cut(uint64_t target, SampleCut within) {
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
        if (MASS) atomicAdd((unsigned long long *)&sm.hist.mass[b], (unsigned long long)row.weight(v));
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
    const float v = __uint_as_float(c.key & 0x80000000u ? c.key ^ 0x80000000u : ~c.key);
    const uint64_t each = MASS ? row.weight(v) : 1;
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

  __device__ uint64_t mass(SampleCut c) {
    uint64_t s = 0, total;
    for (int i = threadIdx.x; i < n; i += SR_THREADS) {
      const float v = at(i);
      if (c.keeps(sample_key(v), i)) s += row.weight(v);
    }
    block_scan(s, total, sm);
    return total;
  }

  // The first entry at which the running sum of what c keeps exceeds u of it all.
  __device__ int draw(SampleCut c, float u, uint64_t &weight, uint64_t &total) {
    const int tiles = (n + SR_TILE - 1) / SR_TILE;
    __syncthreads();
    for (int t = threadIdx.x; t < SR_MOST / SR_TILE; t += SR_THREADS) sm.tile[t] = 0;
    __syncthreads();
    for (int t = 0; t < tiles; t++) {
      const int i = t * SR_TILE + threadIdx.x;
      uint64_t w = 0;
      if (i < n) {
        const float v = at(i);
        if (c.keeps(sample_key(v), i)) w = row.weight(v);
      }
      if (w) atomicAdd((unsigned long long *)&sm.tile[t], (unsigned long long)w);
    }
    __syncthreads();
    const uint64_t mine = sm.tile[threadIdx.x], before = block_scan(mine, total, sm);
    const uint64_t target = sample_share(__float_as_uint(u), total, false);
    if (before <= target && before + mine > target) {
      sm.result[0] = threadIdx.x;
      sm.result[1] = before;
    }
    __syncthreads();
    const int t = (int)sm.result[0], i = t * SR_TILE + threadIdx.x;
    const uint64_t base = sm.result[1];
    uint64_t w = 0, all;
    if (i < n) {
      const float v = at(i);
      if (c.keeps(sample_key(v), i)) w = row.weight(v);
    }
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

// One block per row.
template <typename AT> __global__ __launch_bounds__(SR_THREADS) void sample_rows_kernel(SampleRowsArgs a) {
  __shared__ SampleShared sm;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const AT *const x = (const AT *)a.logits + (size_t)r * a.stride;
  float best = -INFINITY;
  int bi = 0x7fffffff;
  for (int i = threadIdx.x; i < a.n; i += SR_THREADS) {
    const float v = sample_clean((float)x[i]);
    if (v > best) { best = v; bi = i; }
  }
  for (int off = 32; off > 0; off >>= 1) {
    const float ov = __shfl_xor(best, off);
    const int oi = __shfl_xor(bi, off);
    if (ov > best || (ov == best && oi < bi)) { best = ov; bi = oi; }
  }
  if (lane == 0) { sm.best[wave] = best; sm.at[wave] = bi; }
  __syncthreads();
  best = sm.best[0];
  bi = sm.at[0];
  for (int w = 1; w < SR_THREADS / 64; w++)
    if (sm.best[w] > best || (sm.best[w] == best && sm.at[w] < bi)) { best = sm.best[w]; bi = sm.at[w]; }
  const float temperature = a.temperature ? a.temperature[r] : 1.0f;
  int token = best == -INFINITY ? -1 : bi;
  float prob = best == -INFINITY ? 0.0f : 1.0f;
  if (best > -INFINITY && temperature >= 1e-6f) {
    const float p = a.top_p ? a.top_p[r] : 1.0f, m = a.min_p ? a.min_p[r] : 0.0f;
    const int k = a.top_k ? a.top_k[r] : 0;
    float u = a.uniforms[r];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    SampleBlock<AT> b = {x, a.n, {best, 1.4426950408889634 / (double)temperature, m > 0.0f ? (double)fminf(m, 1.0f) : 0.0}, sm};
    SampleCut c = {0, 0x7fffffff};
    if (k > 0 && k < a.n) c = b.template cut<false>((uint64_t)k, c);
    if (p < 1.0f) {
      const uint64_t target = p > 0.0f ? sample_share(__float_as_uint(p), b.mass(c), true) : 1;
      c = b.template cut<true>(target > 1 ? target : 1, c);
    }
    uint64_t w, total;
    token = b.draw(c, u, w, total);
    prob = (float)((double)w / (double)total);
  }
  if (threadIdx.x == 0) {
    a.tokens[r] = token;
    if (a.probs) a.probs[r] = prob;
  }
}

}  // namespace jsg

using namespace jsg;

extern "C" {

size_t jsgrad_hip_sample_rows_workspace_bytes(int rows, int n) {
  if (rows <= 0 || n <= 0) return 0;
  return 256;
}

int jsgrad_hip_sample_rows(const void *logits, int rows, int n, size_t row_stride, int act, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                           const float *uniforms, int32_t *tokens_out, float *probs_out, void *workspace) {
  const char *who = "jsgrad_hip_sample_rows";
  JSG_REQUIRE(logits && uniforms && tokens_out && workspace, "%s: null pointer argument", who);
  JSG_REQUIRE(act == JSGRAD_F16 || act == JSGRAD_F32, "%s: unknown activation dtype %d", who, act);
  JSG_REQUIRE(rows > 0 && rows <= 65535, "%s: %d rows (1 to 65535)", who, rows);
  JSG_REQUIRE(n > 0 && n <= SR_MOST, "%s: %d logits (1 to %d)", who, n, SR_MOST);
  JSG_REQUIRE(row_stride >= (size_t)n && row_stride < (size_t)1 << 40, "%s: a stride of %zu for rows of %d", who, row_stride, n);
  JSG_REQUIRE((uintptr_t)logits % (act == JSGRAD_F16 ? 2 : 4) == 0, "%s: logits must be aligned to their type", who);
  JSG_REQUIRE(((uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)uniforms | (uintptr_t)tokens_out | (uintptr_t)probs_out) % 4 == 0,
              "%s: the rows' arrays must be 4-byte aligned", who);
  JSG_REQUIRE((uintptr_t)workspace % 16 == 0, "%s: workspace must be 16-byte aligned", who);
  JSG_READY();
  SampleRowsArgs a = {logits, row_stride, n, temperature, top_p, min_p, uniforms, top_k, tokens_out, probs_out};
  if (act == JSGRAD_F16) JSG_LAUNCH(PROF_SAMPLE, sample_rows_kernel<_Float16>, dim3(rows), dim3(SR_THREADS), 0, a);
  else JSG_LAUNCH(PROF_SAMPLE, sample_rows_kernel<float>, dim3(rows), dim3(SR_THREADS), 0, a);
  return 0;
}

}  // extern "C"
