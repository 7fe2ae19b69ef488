// Addressing and number format of a key/value cache in 8 bits (kv8.hip, kv8_attn.hip).
//
// The 16 positions of a group (a unit of the kernels) of one head share a power of two, keys and values apart: a code c
// under exponent byte e stands for c 2^(e - 127).  As e4m3 codes have exponents of their own, a power of two more or less
// costs no precision but at the far end of small values: a group that grows is rounded again without loss up to there, and
// bf16 holds every value of the cache as it is (under exponent bytes of 3 and more).
#pragma once

#include "e4m3.h"
#include "kv8_pages.h"

namespace mx {

constexpr int kUnit = 16;

// the unit (codes: x 16 D, exponents: x 1) of the pool that holds positions 16 u .. of head hk of a slot; -1: the table
// names no page of the pool
__device__ __forceinline__ int64_t kv8_unit(const Kv8Pages& pg, int slot, int u, int hk) {
  const uint32_t per = (uint32_t)pg.block / kUnit;
  const int page = pg.table[(int64_t)slot * pg.maxp + (uint32_t)u / per];
  if ((unsigned)page >= (unsigned)pg.pages) return -1;
  return ((int64_t)page * pg.Hkv + hk) * per + (uint32_t)u % per;
}

// The least exponent byte of 1 .. 254 under which amax (>= 0, finite) is at most 448 = 1.75 * 2^8
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  return max(1, (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// four values (times 2^s) -> four codes, and back; rounded to nearest even, what is no number as NaN
__device__ __forceinline__ uint32_t kv8_code4(float a, float b, float c, float d, int s) {
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(a, s), __builtin_ldexpf(b, s), w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(c, s), __builtin_ldexpf(d, s), w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ void kv8_value4(uint32_t w, int s, float* x) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = __builtin_ldexpf(lo[0], s), x[1] = __builtin_ldexpf(lo[1], s);
  x[2] = __builtin_ldexpf(hi[0], s), x[3] = __builtin_ldexpf(hi[1], s);
}

}  // namespace mx
