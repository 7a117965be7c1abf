// The 8-bit cache's numbers: e4m3 codes (OCP, no infinities) with one scale 2^k
// for the K or V of a block of tokens and KV head.
//
// A power of two makes every step but the one rounding to a code exact: x * 2^-k
// and code * 2^k only move the exponent, a block whose scale grows keeps its
// significands (only codes that fall below 2^-6 are rounded again), and every
// value that the cache holds is a number of the pool's dtype, so reading it back
// and feeding it to the matrix cores rounds nothing. A floating-point code loses
// no relative precision by the up to one bit that the scale is too wide.
#pragma once

#include "common.hpp"

namespace ir {

// Bounds of k for a pool of dtype DT, and the largest magnitude it holds. fp16: at
// 2^-15 the smallest code is fp16's smallest number; at 2^8 the codes end at 240, the
// last whose value fp16 has. bf16 and fp32: 448 * 2^119 is the last within their
// range, and 2^-100 keeps values and scales clear of subnormal numbers.
template <int DT>
struct ScaleBounds {
  static constexpr int lo = DT == IR_DTYPE_F16 ? -15 : -100;
  static constexpr int hi = DT == IR_DTYPE_F16 ? 8 : 119;
  static constexpr float max = DT == IR_DTYPE_F16 ? 61440.f : 0x1.cp+127f;
};

// 2^k for k in [-126, 127].
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

__device__ __forceinline__ int exponent_of(float scale) { return (int)((__float_as_uint(scale) >> 23) & 0xffu) - 127; }

// The least k within the bounds with amax <= 448 * 2^k, 448 = 1.75 * 2^8.
template <int DT>
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int k = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(ScaleBounds<DT>::lo, min(ScaleBounds<DT>::hi, k));
}

// The two codes in the low (HI: high) half of w, times scale (a power of two): two
// 16-bit elements of dtype DT in one dword, exact.
template <int DT, bool HI>
__device__ __forceinline__ uint32_t decode2(uint32_t w, float scale) {
  if constexpr (DT == IR_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}

template <bool HI>
__device__ __forceinline__ f32x2 decode2_f32(uint32_t w, float scale) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, HI));
}

// The power of two that brings a row's largest magnitude to [2^14, 2^15), where fp16 has
// the most room below it (k in [-113, 126], so that 2^k and 2^-k are normal numbers).
__device__ __forceinline__ int row_shift(float most) { return max(-113, min(126, 14 - exponent_of(most))); }

}  // namespace ir
