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

// D += A . B of 128 e4m3 codes a row and column (16 rows, 16 columns): 32 codes of A and
// of B per lane, of scales 2^(ea - 127) and 2^(eb - 127). The k-slots of lane group g
// are [16 g, +16) in the first four registers and [64 + 16 g, +16) in the last four, and
// the scale of k-slots [32 b, +32) is the one that lane group b gives (both measured).
// The instruction sums eight products at a time aligned to the largest of them, some 17
// bits below which are lost (measured: 1 next to 448^2), and these sums in fp32.
typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma_codes_k128(i32x8 a, int ea, i32x8 b, int eb, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, ea, 0, eb);
}

}  // namespace ir
