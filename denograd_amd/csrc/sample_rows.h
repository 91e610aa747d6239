// The borders that sampling of rows goes by (sample_rows.hip), in plain C++ so that a host compiler takes it too (tests/test_sample_rows.py).
#pragma once
#include <stdint.h>

#ifndef JSG_BOTH
#ifdef __HIPCC__
#define JSG_BOTH __host__ __device__ __forceinline__
#else
#define JSG_BOTH inline
#endif
#endif

namespace jsg {

// floor (or, up, ceiling) of f * z, without a rounding; bits: of a float f from 0 to below 1
JSG_BOTH uint64_t sample_share(uint32_t bits, uint64_t z, bool up) {
  const uint32_t e = bits >> 23;
  const uint64_t mant = e ? (bits & 0x7fffffu) | 0x800000u : bits & 0x7fffffu;
  const int shift = 150 - (int)(e ? e : 1);                  // f = mant * 2^-shift, 24 and more
  const unsigned __int128 product = (unsigned __int128)mant * z;
  if (shift >= 96) return up && product != 0;                // below one
  const uint64_t q = (uint64_t)(product >> shift);
  return q + (up && product != (unsigned __int128)q << shift);
}

}  // namespace jsg
