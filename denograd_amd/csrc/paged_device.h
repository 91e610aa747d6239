// What the kernels of the paged cache share on the device (paged.hip, paged_attn.hip, paged_select.hip).
#pragma once
#include "gemm.h"
#include "paged.h"

namespace jsg {

int paged_check(const char *who, const jsgrad_hip_pages_t *pg, const int32_t *row_starts, const int32_t *lengths, int n_seqs, int rows, PagedBatch *pb);   // paged.hip

// Sequence of row r: the first one that ends behind it.  Called by whole wavefronts with a uniform r: 64 first rows at a time.
__device__ __forceinline__ int paged_find(const PagedBatch &pb, int r) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0;; b0 += 64) {
    const int b = b0 + lane;
    const uint64_t behind = __builtin_amdgcn_ballot_w64(b >= pb.n_seqs || pb.row_starts[b + 1] > r);
    if (behind) return b0 + __builtin_ctzll(behind);         // n_seqs: no sequence has the row
  }
}

// The scale of V that an int8 row's weight has in the exponent.  The halves are weights times scales relative to the largest of these, so a row whose scale says more than its codes
// would push the others out of fp16's range: one of zero codes, which is written with scale 1 and in a caller's own pages may have any.  It counts with 2^-60, and its weight 2^60 times that in the sum: it
// is the largest only where it outweighs the others by so much that nothing of them is left in an fp16 result.  A scale below 2^-60 counts with that as well: values of 2^-53 and less are
// nothing there either.  A scale that is not a number, or not finite, stays what it is.
constexpr float PAGED_TINY = 0x1p-60f;
__device__ __forceinline__ float scale_of_v(float v, bool zeros) { return v >= 0.0f && v < (zeros ? INFINITY : PAGED_TINY) ? PAGED_TINY : v; }

}  // namespace jsg
