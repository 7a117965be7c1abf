// The 4-bit cache's numbers and where they lie: e2m1 codes (OCP: 0, 0.5, 1, 1.5, 2, 3, 4,
// 6 and their negatives) with one scale 2^k for 32 consecutive channels of a token's
// head, K or V. A scale is a byte, k + 127; 255 makes the group's values NaN, which e2m1
// has no code for.
//
// The scale belongs to one token, so a token is written without reading what is beside
// it, and a power of two makes every step but the one rounding to a code exact: every value
// that the cache holds is a number of the pool's dtype, and the conversion instructions
// take the scale with them.
//
// A tile is 16 tokens of one head: 8 D bytes of K, as many of V, and D bytes of scales.
// Its order is that of the attention's registers (attn_tile.hpp), so that one 16-byte
// load a lane (8 at head_dim 64) reads a whole tile's K or V, contiguous over the
// wavefront, without LDS. Lane 16 g + c then holds
//   K: channels [D/4 g, +D/4) of token 4 (c % 4) + c / 4, the row c of its score product;
//   V: channels [D/16 c, +D/16) of tokens 4 r + g, r = 0..3, whose scores it holds.
// Bytes hold two channels of one token, the lower one in the low half.
#pragma once

#include "e4m3.hpp"

namespace ir {

// Bounds of k for a pool of dtype DT. fp16: at 2^-23 the smallest code is its smallest
// number, at 2^13 the largest is 49152. bf16 and fp32: 6 * 2^125 is the last within
// their range, and 2^-100 keeps values clear of subnormal numbers.
template <int DT>
struct Scale4Bounds {
  static constexpr int lo = DT == IR_DTYPE_F16 ? -23 : -100;
  static constexpr int hi = DT == IR_DTYPE_F16 ? 13 : 125;
};

// Byte offsets within a tile.
template <int D>
struct Tile4 {
  static constexpr int CODES = 8 * D;      // bytes of K, and of V
  static constexpr int SCALES = D;         // bytes of K's scales, then V's
  static constexpr int LB = D / 8;         // bytes of a lane
  static constexpr int NG = D / 32;        // groups of a token
  // the dword of K that holds channels [8 ch8, +8) of token t
  __device__ __forceinline__ static int k(int t, int ch8) {
    const int c = 4 * (t & 3) + (t >> 2);
    return (16 * (ch8 / (LB / 4)) + c) * LB + 4 * (ch8 % (LB / 4));
  }
  // the LB / 4 bytes of V that hold channels [D/16 c, +D/16) of token t
  __device__ __forceinline__ static int v(int t, int c) { return (16 * (t & 3) + c) * LB + (LB / 4) * (t >> 2); }
  __device__ __forceinline__ static int k_scale(int t, int grp) { return 16 * grp + 4 * (t & 3) + (t >> 2); }
  __device__ __forceinline__ static int v_scale(int t, int grp) {
    return D / 2 + 4 * (NG * (t & 3) + grp) + (t >> 2);
  }
};

// A line of a tile holds 8 tokens' K or all of its V's channels, some lanes of each, and workgroup i
// runs on XCD i % 8: the order of workgroups in which four that follow one another (of a few tokens
// each) meet in one XCD's L2, of a grid rounded up to whole runs of 32. (Reading 65,536 tokens of 4 heads
// of 128, bf16: 40.7 -> 26.1 us; 8,192: 4.8 -> 4.4; a write of 1,024: 4.1 -> 3.9. Slots in no order: the
// same either way.)
__device__ __forceinline__ uint32_t near_block(uint32_t i) { return (i & ~31u) | (i & 7) << 2 | (i >> 3 & 3); }
inline int64_t near_blocks(int64_t blocks) { return (blocks + 31) & ~(int64_t)31; }

// Scale byte B of w as the conversions take it: they read the exponent field alone (255
// there is NaN to them), so the neighbouring bytes that come along need not be cleared
// (measured for every exponent and code).
template <int B = 0>
__device__ __forceinline__ float scale_of_byte(uint32_t w) {
  return __uint_as_float(B == 0 ? w << 23 : B == 1 ? w << 15 : B == 2 ? w << 7 : w >> 1);
}

// Codes of byte B of w, times scale: two 16-bit elements of dtype DT in one dword, exact.
template <int DT, int B>
__device__ __forceinline__ uint32_t decode2_e2m1(uint32_t w, float scale) {
  if constexpr (DT == IR_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B));
}

template <int B>
__device__ __forceinline__ f32x2 decode2_e2m1_f32(uint32_t w, float scale) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, B));
}

// The eight codes of a dword as a row's dwords of dtype DT (4, or 8 of fp32).
template <int DT>
__device__ __forceinline__ void decode8_e2m1(uint32_t w, float scale, uint32_t (&to)[DT == IR_DTYPE_F32 ? 8 : 4]) {
  if constexpr (DT == IR_DTYPE_F32) {
    const f32x2 a = decode2_e2m1_f32<0>(w, scale), b = decode2_e2m1_f32<1>(w, scale);
    const f32x2 c = decode2_e2m1_f32<2>(w, scale), d = decode2_e2m1_f32<3>(w, scale);
    const float x[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = __float_as_uint(x[i]);
  } else {
    to[0] = decode2_e2m1<DT, 0>(w, scale);
    to[1] = decode2_e2m1<DT, 1>(w, scale);
    to[2] = decode2_e2m1<DT, 2>(w, scale);
    to[3] = decode2_e2m1<DT, 3>(w, scale);
  }
}

// Eight numbers to codes, x / scale to nearest even, past 6 saturated.
__device__ __forceinline__ uint32_t encode8_e2m1(const float* x, float scale) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// Maximum over the quad of lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppXor1, 0xf, 0xf, true));
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppXor2, 0xf, 0xf, true));
}

// Writes lane `ci`'s part (norm_rope.hpp's: elements [8 ci, +8) of either half) of a row
// of token t's head to its tile. A group of 32 channels is a quad of lanes, all here.
// The group's scale is the least 2^k within the bounds with amax <= 7 * 2^k, 7 = 1.75 * 2^2:
// up to there the largest magnitude rounds to 6, and every value is off by half a
// step of its code at most. (Magnitudes are compared as bits, where NaN and infinities
// are the largest.)
template <int DT, int D>
__device__ __forceinline__ void store_row_e2m1(const float (&x)[16], uint8_t* codes, uint8_t* scales, int t, int ci,
                                               bool is_v) {
  typedef Tile4<D> T;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float* y = x + 8 * half;
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
    m = quad_max(m);
    const int k = max(Scale4Bounds<DT>::lo, min(Scale4Bounds<DT>::hi, (int)(m >> 23) - 129 +
                                                                          ((m & 0x7fffffu) > 0x600000u ? 1 : 0)));
    const uint32_t w = encode8_e2m1(y, pow2(k));
    const int ch8 = ci + half * (D / 16);
    if (!is_v) {
      *(uint32_t*)(codes + T::k(t, ch8)) = w;
    } else if constexpr (D == 128) {
      *(uint32_t*)(codes + T::v(t, ch8)) = w;
    } else {
      *(uint16_t*)(codes + T::v(t, 2 * ch8)) = (uint16_t)w;
      *(uint16_t*)(codes + T::v(t, 2 * ch8 + 1)) = (uint16_t)(w >> 16);
    }
    if ((ci & 3) == 0) {
      const int grp = ch8 >> 2;
      scales[is_v ? T::v_scale(t, grp) : T::k_scale(t, grp)] = (uint8_t)(m >= 0x7f800000u ? 255 : k + 127);
    }
  }
}

}  // namespace ir
