// Rows of queries and keys normed per head and rotated, in one pass over them.
//
//   y = x * rsqrt(mean(x^2) + eps) * w,  out = y * cos + rotate_half(y) * sin,
//   rotate_half(y) = (-y2, y1) over the halves of head_dim,
// in fp32 throughout and rounded once, where it is stored. Without norms
// (ROTATE) the rotation is ir_rope_kv_scatter's, which rounds the tables, each
// product and the sum to the dtype as the reference's tensor operations do. kRowsTurn is
// the rotation in fp32, as with norms, of rows that have none.
//
// head_dim / 16 lanes share a row: each holds 8 elements of its first half and
// the 8 of the second half that the rotation pairs them with, so only the sum of
// squares crosses lanes.
#pragma once

#include "chunk8.hpp"

namespace ir {

enum { kRowsPlain = 0, kRowsRotate = 1, kRowsNorm = 2, kRowsTurn = 3 };

struct RowArgs {
  const uint8_t* q;
  int64_t q_tok, q_head;  // bytes, as every stride here
  uint8_t* qo;
  int qo_wide;  // the rotated queries are stored as fp32, whatever the dtype
  int64_t qo_tok, qo_head;
  const uint8_t* k;
  int64_t k_tok, k_head;
  const uint8_t* v;
  int64_t v_tok, v_head;
  const float* cos;
  const float* sin;
  int64_t cs_tok;  // elements
  const uint8_t* q_weight;
  const uint8_t* k_weight;
  float eps;
  const int64_t* slots;
  int64_t n_tokens;
  int num_q_heads, num_kv_heads;
};

// Checks a C call's row arguments (strides in elements of eb bytes, q_out's of qo_eb; the norm
// weights both given or both null) and fills r; an IR_E* code on refusal. fill_rows: those
// but the tables and slots (k and v null where there are none).
int fill_rows(const char* name, RowArgs& r, const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok,
              int64_t qo_head, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
              int64_t v_head, const void* q_weight, const void* k_weight, float eps, int64_t n_tokens,
              int num_q_heads, int num_kv_heads, int eb, int qo_eb);
int fill_row_args(const char* name, RowArgs& r, const void* q, int64_t q_tok, int64_t q_head, void* q_out,
                  int64_t qo_tok, int64_t qo_head, const void* k, int64_t k_tok, int64_t k_head, const void* v,
                  int64_t v_tok, int64_t v_head, const void* q_weight, const void* k_weight, float eps,
                  const float* cos, const float* sin, int64_t cs_tok, const int64_t* slots, int64_t n_tokens,
                  int num_q_heads, int num_kv_heads, int eb, int qo_eb);

// Lane `ci` of a row: its 16 elements of the row at `p`, [8 ci, +8) of either half.
template <int DT, int D>
struct RowPair {
  typedef Chunk8<DT> C;
  static constexpr int LPR = D / 16;           // lanes per row
  static constexpr int HALF = D / 2 * C::EB;  // bytes
  typename C::Raw a, b;
  __device__ __forceinline__ void load(const uint8_t* p, int ci) {
    C::raw_load(p + ci * 8 * C::EB, a);
    C::raw_load(p + ci * 8 * C::EB + HALF, b);
  }
  __device__ __forceinline__ void store_raw(uint8_t* p, int ci) const {
    C::raw_store_nt(p + ci * 8 * C::EB, a);
    C::raw_store_nt(p + ci * 8 * C::EB + HALF, b);
  }
  __device__ __forceinline__ void unpack(float (&x)[16]) const {
    float lo[8], hi[8];
    C::unpack(a, lo);
    C::unpack(b, hi);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = lo[e];
      x[8 + e] = hi[e];
    }
  }
  __device__ __forceinline__ static void store(uint8_t* p, int ci, const float (&x)[16]) {
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = x[e];
      hi[e] = x[8 + e];
    }
    C::store_nt(p + ci * 8 * C::EB, lo);
    C::store_nt(p + ci * 8 * C::EB + HALF, hi);
  }
};

// The lane's part of a token's tables, rounded to the dtype for ROTATE.
template <int DT, int D, int MODE>
struct Angles {
  float c[16], s[16];
  __device__ __forceinline__ void load(const float* cos, const float* sin, int ci) {
    half(cos + 8 * ci, c, 0);
    half(cos + 8 * ci + D / 2, c, 8);
    half(sin + 8 * ci, s, 0);
    half(sin + 8 * ci + D / 2, s, 8);
  }
  __device__ __forceinline__ static void half(const float* p, float (&to)[16], int at) {
    float t[8];
    Chunk8<IR_DTYPE_F32>::load((const uint8_t*)p, t);
    if constexpr (MODE == kRowsRotate) Chunk8<DT>::round8(t);
#pragma unroll
    for (int e = 0; e < 8; ++e) to[at + e] = t[e];
  }
};

// x (the lane's 16 elements of its row) to the row's result. Every lane of the
// row must be here.
template <int DT, int D, int MODE>
__device__ __forceinline__ void transform_row(float (&x)[16], const float (&w)[16], float eps,
                                              const Angles<DT, D, MODE>& t) {
#pragma clang fp contract(off)
  if constexpr (MODE == kRowsNorm || MODE == kRowsTurn) {
    if constexpr (MODE == kRowsNorm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
      const float r = rsqrtf(row_sum<D / 16>(ss) * (1.f / D) + eps);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = x[e] * r * w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[e], b = x[8 + e];
      x[e] = __builtin_fmaf(a, t.c[e], -b * t.s[e]);
      x[8 + e] = __builtin_fmaf(b, t.c[8 + e], a * t.s[8 + e]);
    }
  } else {
    typedef Chunk8<DT> C;
    float a1[8], b1[8], a2[8], b2[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a1[e] = x[e] * t.c[e];
      b1[e] = -x[8 + e] * t.s[e];
      a2[e] = x[8 + e] * t.c[8 + e];
      b2[e] = x[e] * t.s[8 + e];
    }
    C::round8(a1);
    C::round8(b1);
    C::round8(a2);
    C::round8(b2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a1[e] += b1[e];
      a2[e] += b2[e];
    }
    C::round8(a1);
    C::round8(a2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = a1[e];
      x[8 + e] = a2[e];
    }
  }
}

}  // namespace ir
