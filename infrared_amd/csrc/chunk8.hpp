// Eight consecutive elements of a row in fp32, with their raw 16-byte storage:
// what a lane of the row-wise kernels (rotation, norms, quantisation) holds.
#pragma once

#include "common.hpp"

namespace ir {

template <int DT>
struct Chunk8 {
  // 8 elements in fp32 plus their raw storage
  static constexpr int EB = DT == IR_DTYPE_F32 ? 4 : 2;
  __device__ __forceinline__ static void load(const uint8_t* p, float (&x)[8]) {
    if constexpr (DT == IR_DTYPE_F32) {
      const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
      }
    } else {
      using E = Elem<DT>;
      const u32x4 w = *(const u32x4*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = E::lo(w[i]);
        x[2 * i + 1] = E::hi(w[i]);
      }
    }
  }
  __device__ __forceinline__ static void store(uint8_t* p, const float (&x)[8]) {
    if constexpr (DT == IR_DTYPE_F32) {
      *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
      *(f32x4*)(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      using E = Elem<DT>;
      *(u32x4*)p = u32x4{E::pack2(x[0], x[1]), E::pack2(x[2], x[3]), E::pack2(x[4], x[5]), E::pack2(x[6], x[7])};
    }
  }
  // non-temporal: for rows that the next kernel reads, on any XCD, and so not from the
  // L2 that they would stay in
  __device__ __forceinline__ static void store_nt(uint8_t* p, const float (&x)[8]) {
    if constexpr (DT == IR_DTYPE_F32) {
      __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, (f32x4*)p);
      __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, (f32x4*)(p + 16));
    } else {
      using E = Elem<DT>;
      __builtin_nontemporal_store(
          u32x4{E::pack2(x[0], x[1]), E::pack2(x[2], x[3]), E::pack2(x[4], x[5]), E::pack2(x[6], x[7])}, (u32x4*)p);
    }
  }
  struct Raw {
    u32x4 w[EB / 2];
  };
  __device__ __forceinline__ static void raw_load(const uint8_t* p, Raw& r) {
#pragma unroll
    for (int i = 0; i < EB / 2; ++i) r.w[i] = *(const u32x4*)(p + 16 * i);
  }
  __device__ __forceinline__ static void raw_store(uint8_t* p, const Raw& r) {
#pragma unroll
    for (int i = 0; i < EB / 2; ++i) *(u32x4*)(p + 16 * i) = r.w[i];
  }
  __device__ __forceinline__ static void raw_store_nt(uint8_t* p, const Raw& r) {
#pragma unroll
    for (int i = 0; i < EB / 2; ++i) __builtin_nontemporal_store(r.w[i], (u32x4*)(p + 16 * i));
  }
  __device__ __forceinline__ static void unpack(const Raw& r, float (&x)[8]) {
    if constexpr (DT == IR_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __uint_as_float(r.w[0][i]);
        x[4 + i] = __uint_as_float(r.w[1][i]);
      }
    } else {
      using E = Elem<DT>;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = E::lo(r.w[0][i]);
        x[2 * i + 1] = E::hi(r.w[0][i]);
      }
    }
  }
  // each value rounded to the dtype, to nearest even, two per conversion
  // instruction (identity for fp32)
  __device__ __forceinline__ static void round8(float (&x)[8]) {
    if constexpr (DT != IR_DTYPE_F32) {
      using E = Elem<DT>;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = E::pack2(x[2 * i], x[2 * i + 1]);
        x[2 * i] = E::lo(w);
        x[2 * i + 1] = E::hi(w);
      }
    }
  }
};

}  // namespace ir
