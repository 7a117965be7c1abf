// The 8-bit K/V pool for gfx950: new rows quantised as they are written
// (optionally normed and rotated on the way), and read back. Codes and scales are
// e4m3.hpp's; a layer is dense, [H_kv][num_blocks][block_size][D] codes for K and
// for V and [H_kv][num_blocks][2] scales.
//
// The write. A block's scale covers all its tokens, so the tokens of a call that
// share a block have to be handled together, whatever their order in the call. The
// workgroup of token i drops out if the token before it is in the same block
// (which ends most of a prompt's), else it reads every slot of the call once and
// drops out if an earlier one is in the block; the one that is left owns the block,
// knows which row each of its tokens takes (the last given), and no other workgroup
// touches it. That is one launch without a workspace and with a result that does not
// depend on the order of execution. The slots are 8 bytes a token against about
// 3 KB of rows at 4 heads of 128, and come from L2, but n / block_size workgroups
// read them all: 4 us of L2 traffic at 16,384 tokens, growing with the square.
//
// A wavefront then takes K or V of one head: its rows' largest magnitude gives the
// scale, the rows become codes. A block that is not new keeps its tokens; only when
// its scale grows are they read, rounded to the wider scale and written back.
#include "e4m3.hpp"
#include "norm_rope.hpp"
#include "status.hpp"

namespace ir {
namespace {

constexpr int kMaxBlockSize = 1024;
constexpr int kWriteWaves = 4;

struct QuantArgs {
  RowArgs r;
  uint8_t* kc;
  uint8_t* vc;
  float* scales;
  int64_t num_blocks;
  int bs;
  int kv_groups;   // workgroups per token for its 2 * H_kv (head, K / V) parts
  int64_t n_kv;    // workgroups of the write; those after them take query rows
  int32_t* err;
};

// Magnitude that counts for a block's scale: none for NaN and infinities.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= __FLT_MAX__ ? a : 0.f;
}

// x * inv (inv = 2^-k) as the conversion to codes takes it: past the pool's range
// saturated, not a finite number: NaN.
template <int DT>
__device__ __forceinline__ float to_code_range(float x, float inv) {
  const float y = fminf(fmaxf(x, -ScaleBounds<DT>::max), ScaleBounds<DT>::max) * inv;
  return fabsf(x) <= __FLT_MAX__ ? y : __builtin_nanf("");
}

// Four numbers within +-448 to codes, to nearest even.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

// The query rows of wavefront `wave` (MODE not plain).
template <int DT, int D, int MODE>
__device__ __forceinline__ void query_rows(const RowArgs& r, int64_t wave) {
  typedef RowPair<DT, D> P;
  constexpr int G = 64 / P::LPR;
  const int lane = threadIdx.x & 63, ci = lane % P::LPR, grp = lane / P::LPR;
  const int runs = (r.num_q_heads + G - 1) / G;
  const int64_t tok = wave / runs;
  const int h = (int)(wave - tok * runs) * G + grp;
  if (tok >= r.n_tokens || h >= r.num_q_heads) return;  // (a row's lanes go together)
  P p, pw;
  p.load(r.q + tok * r.q_tok + h * r.q_head, ci);
  Angles<DT, D, MODE> t;
  t.load(r.cos + tok * r.cs_tok, r.sin + tok * r.cs_tok, ci);
  float x[16], w[16];
  if constexpr (MODE == kRowsNorm) {
    pw.load(r.q_weight, ci);
    pw.unpack(w);
  }
  p.unpack(x);
  transform_row<DT, D, MODE>(x, w, r.eps, t);
  P::store(r.qo + tok * r.qo_tok + h * r.qo_head, ci, x);
}

template <int DT, int D, int MODE>
__global__ __launch_bounds__(kWriteWaves * 64) void kv_write_q8_kernel(QuantArgs a) {
  typedef RowPair<DT, D> P;
  constexpr int NT = kWriteWaves * 64;
  constexpr int RPP = 64 / P::LPR;  // rows of a wavefront at a time
  __shared__ int s_row[kMaxBlockSize];  // row + 1 that each token of the block takes, 0: none
  __shared__ int s_earlier;
  if constexpr (MODE != kRowsPlain) {
    if (blockIdx.x >= a.n_kv) {
      query_rows<DT, D, MODE>(a.r, (blockIdx.x - a.n_kv) * kWriteWaves + (threadIdx.x >> 6));
      return;
    }
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t i = blockIdx.x / a.kv_groups;
  const int part0 = (int)(blockIdx.x - i * a.kv_groups) * kWriteWaves;
  const int64_t slot = a.r.slots[i];
  if (slot < 0) return;  // padding sentinel
  if (slot >= a.num_blocks * a.bs) {
    if (tid == 0 && part0 == 0) flag_error(a.err, IR_ERR_SLOT_RANGE);
    return;
  }
  const int blk = (int)((uint32_t)slot / (uint32_t)a.bs);  // (the pool's slots fit 31 bits)
  const int64_t base = (int64_t)blk * a.bs;
  auto inside = [&](int64_t s) { return (uint64_t)s - (uint64_t)base < (uint64_t)a.bs; };
  if (i > 0 && inside(a.r.slots[i - 1])) return;

  // ---- the block's tokens in this call
  for (int t = tid; t < a.bs; t += NT) s_row[t] = 0;
  if (tid == 0) s_earlier = 0;
  __syncthreads();
  for (int64_t j = tid; j < a.r.n_tokens; j += NT) {
    const int64_t s = a.r.slots[j];
    if (inside(s)) {
      atomicMax(&s_row[(int)(s - base)], (int)j + 1);
      if (j < i) s_earlier = 1;
    }
  }
  __syncthreads();
  if (s_earlier) return;  // uniform
  const bool fresh = s_row[0] != 0;

  // ---- this wavefront's head, K or V
  const int part = part0 + (tid >> 6);
  if (part >= 2 * a.r.num_kv_heads) return;
  const int h = part >> 1, is_v = part & 1;
  const int64_t hb = (int64_t)h * a.num_blocks + blk;
  float* sp = a.scales + 2 * hb + is_v;
  const float old = *sp;
  uint8_t* codes = (is_v ? a.vc : a.kc) + hb * a.bs * D;
  const uint8_t* src = is_v ? a.r.v + h * a.r.v_head : a.r.k + h * a.r.k_head;
  const int64_t tok_stride = is_v ? a.r.v_tok : a.r.k_tok;
  const int ci = lane % P::LPR, grp = lane / P::LPR;
  float w[16];
  if constexpr (MODE == kRowsNorm) {
    P pw;
    pw.load(a.r.k_weight, ci);
    pw.unpack(w);
  }
  // the new row of token t of the block into x; false: none
  auto row = [&](int t, float (&x)[16]) -> bool {
    const int64_t j = (int64_t)s_row[t] - 1;
    if (j < 0) return false;  // (a row's lanes go together)
    P p;
    p.load(src + j * tok_stride, ci);
    p.unpack(x);
    if constexpr (MODE != kRowsPlain) {
      if (!is_v) {
        Angles<DT, D, MODE> t;
        t.load(a.r.cos + j * a.r.cs_tok, a.r.sin + j * a.r.cs_tok, ci);
        transform_row<DT, D, MODE>(x, w, a.r.eps, t);
      }
    }
    return true;
  };
  // the first passes' rows stay in registers, those of larger blocks are read again
  constexpr int KEEP = 16 / RPP;
  float x[KEEP][16];
  bool has[KEEP];
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < KEEP; ++p) {
    has[p] = row(p * RPP + grp, x[p]);
    if (has[p])
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, finite_abs(x[p][e]));
  }
  for (int t = 16 + grp; t < a.bs; t += RPP) {
    float y[16];
    if (row(t, y))
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, finite_abs(y[e]));
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));

  const int need = scale_exponent<DT>(amax);
  const int held = max(ScaleBounds<DT>::lo, min(ScaleBounds<DT>::hi, exponent_of(old)));
  const int k = fresh ? need : max(held, need);
  const bool grow = !fresh && k > held;
  const float inv = pow2(-k);
  // an old code's place under the wider scale: below 2^-100 every code is zero
  const float shrink = pow2(max(held - k, -100));
  auto put = [&](int t, bool has_row, const float (&y)[16]) {
    u32x2* p0 = (u32x2*)(codes + (int64_t)t * D + 8 * ci);
    u32x2* p1 = (u32x2*)(codes + (int64_t)t * D + 8 * ci + D / 2);
    u32x2 c0 = {0u, 0u}, c1 = {0u, 0u};
    if (has_row) {
      float z[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) z[e] = to_code_range<DT>(y[e], inv);
      c0 = u32x2{encode4(z[0], z[1], z[2], z[3]), encode4(z[4], z[5], z[6], z[7])};
      c1 = u32x2{encode4(z[8], z[9], z[10], z[11]), encode4(z[12], z[13], z[14], z[15])};
    } else if (grow) {
      c0 = *p0;
      c1 = *p1;
      auto again = [&](uint32_t c) {
        const f32x2 lo = decode2_f32<false>(c, shrink), hi = decode2_f32<true>(c, shrink);
        return encode4(lo[0], lo[1], hi[0], hi[1]);
      };
      c0 = u32x2{again(c0[0]), again(c0[1])};
      c1 = u32x2{again(c1[0]), again(c1[1])};
    } else if (!fresh) {
      return;
    }
    *p0 = c0;
    *p1 = c1;
  };
#pragma unroll
  for (int p = 0; p < KEEP; ++p) put(p * RPP + grp, has[p], x[p]);
  for (int t = 16 + grp; t < a.bs; t += RPP) {
    float y[16];
    const bool has_row = row(t, y);
    put(t, has_row, y);
  }
  if (lane == 0) *sp = pow2(k);
}

struct ReadArgs {
  const uint8_t* kc;
  const uint8_t* vc;
  const float* scales;
  int64_t num_blocks;
  int bs, num_kv_heads;
  const int64_t* slots;  // one per output row, or null: through the block tables
  const int32_t* bt;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* ctx;
  int max_ctx;
  int64_t n;  // output rows
  uint8_t* ok;
  uint8_t* ov;
  int32_t* err;
};

// One lane per 8 codes of an output row's head, K and V. Bound by memory: a row is
// read at a byte and written at the dtype's size an element.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_read_q8_kernel(ReadArgs a) {
  typedef Chunk8<DT> C;
  constexpr int PIECES = D / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rh = idx / PIECES;
  const int piece = (int)(idx - rh * PIECES);
  const int64_t row = rh / a.num_kv_heads;
  const int h = (int)(rh - row * a.num_kv_heads);
  if (row >= a.n) return;
  int64_t slot = -1;
  if (a.slots) {
    slot = a.slots[row];
    if (slot < 0 || slot >= a.num_blocks * a.bs) {
      if (piece == 0 && h == 0) flag_error(a.err, IR_ERR_GATHER_RANGE);
      slot = -1;
    }
  } else {
    const int64_t b = row / a.max_ctx;
    const int t = (int)(row - b * a.max_ctx);
    const int cap = a.max_blocks * a.bs;
    int ctx = a.ctx[b];
    if (ctx < 0 || ctx > cap) {
      flag_error(a.err, IR_ERR_CONTEXT_RANGE);
      ctx = ctx < 0 ? 0 : cap;
    }
    if (t < ctx) slot = token_slot(a.bt + b * a.bt_stride, t, a.bs, a.num_blocks, a.err);
  }
  float k8[8] = {}, v8[8] = {};
  if (slot >= 0) {
    const int64_t blk = (uint32_t)slot / (uint32_t)a.bs;
    const f32x2 sc = *(const f32x2*)(a.scales + 2 * ((int64_t)h * a.num_blocks + blk));
    const int64_t at = ((int64_t)h * a.num_blocks * a.bs + slot) * D + 8 * piece;
    const u32x2 kx = *(const u32x2*)(a.kc + at), vx = *(const u32x2*)(a.vc + at);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 k0 = decode2_f32<false>(kx[i], sc[0]), k1 = decode2_f32<true>(kx[i], sc[0]);
      const f32x2 v0 = decode2_f32<false>(vx[i], sc[1]), v1 = decode2_f32<true>(vx[i], sc[1]);
      k8[4 * i] = k0[0], k8[4 * i + 1] = k0[1], k8[4 * i + 2] = k1[0], k8[4 * i + 3] = k1[1];
      v8[4 * i] = v0[0], v8[4 * i + 1] = v0[1], v8[4 * i + 2] = v1[0], v8[4 * i + 3] = v1[1];
    }
  }
  C::store(a.ok + idx * 8 * C::EB, k8);
  C::store(a.ov + idx * 8 * C::EB, v8);
}

// What every call on the pool checks.
int check_pool(const char* name, const void* kc, const void* vc, const float* scales, int64_t num_blocks,
               int block_size, int num_kv_heads, int head_dim) {
  IR_REQUIRE(num_kv_heads > 0 && num_blocks >= 0, "%s: bad sizes", name);
  IR_REQUIRE(block_size > 0 && block_size % 16 == 0 && block_size <= kMaxBlockSize,
             "%s: block size %d must be a multiple of 16, at most %d", name, block_size, kMaxBlockSize);
  if (head_dim != 64 && head_dim != 128)
    return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported (64, 128)", name, head_dim);
  IR_REQUIRE(num_blocks * block_size < ((int64_t)1 << 31), "%s: %lld blocks of %d tokens exceed 2^31 slots", name,
             (long long)num_blocks, block_size);
  IR_REQUIRE(kc && vc && scales, "%s: null pointer", name);
  IR_REQUIRE(aligned16(kc) && aligned16(vc) && ((uintptr_t)scales & 7u) == 0,
             "%s: caches must be 16-byte aligned, scales 8-byte aligned", name);
  return IR_OK;
}

template <int DT, int D>
int launch_write(const char* name, const QuantArgs& a0, int mode, hipStream_t s) {
  QuantArgs a = a0;
  constexpr int G = 64 / (D / 16);
  a.kv_groups = (2 * a.r.num_kv_heads + kWriteWaves - 1) / kWriteWaves;
  a.n_kv = a.r.n_tokens * a.kv_groups;
  const int64_t runs = (a.r.num_q_heads + G - 1) / G;
  const int64_t n_q = mode == kRowsPlain ? 0 : (a.r.n_tokens * runs + kWriteWaves - 1) / kWriteWaves;
  IR_REQUIRE(a.r.n_tokens < 0x7fffffff && a.n_kv + n_q <= 0x7fffffff, "%s: too many tokens", name);
  const dim3 grid((unsigned)(a.n_kv + n_q)), block(kWriteWaves * 64);
  if (mode == kRowsPlain)
    hipLaunchKernelGGL((kv_write_q8_kernel<DT, D, kRowsPlain>), grid, block, 0, s, a);
  else if (mode == kRowsNorm)
    hipLaunchKernelGGL((kv_write_q8_kernel<DT, D, kRowsNorm>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((kv_write_q8_kernel<DT, D, kRowsRotate>), grid, block, 0, s, a);
  return check_launch(name);
}

int dispatch_write(const char* name, const QuantArgs& a, int mode, int head_dim, int dtype, hipStream_t s) {
  switch (dtype) {
    case IR_DTYPE_BF16:
      return head_dim == 128 ? launch_write<IR_DTYPE_BF16, 128>(name, a, mode, s)
                             : launch_write<IR_DTYPE_BF16, 64>(name, a, mode, s);
    case IR_DTYPE_F16:
      return head_dim == 128 ? launch_write<IR_DTYPE_F16, 128>(name, a, mode, s)
                             : launch_write<IR_DTYPE_F16, 64>(name, a, mode, s);
    default:
      return head_dim == 128 ? launch_write<IR_DTYPE_F32, 128>(name, a, mode, s)
                             : launch_write<IR_DTYPE_F32, 64>(name, a, mode, s);
  }
}

int launch_read(const char* name, const ReadArgs& a, int head_dim, int dtype, hipStream_t s) {
  const int64_t lanes = a.n * a.num_kv_heads * (head_dim / 8);
  const int64_t grid = (lanes + 255) / 256;
  IR_REQUIRE(grid <= 0x7fffffff, "%s: too many rows", name);
  const dim3 g((unsigned)grid), b(256);
#define IR_READ(DT)                                                          \
  do {                                                                       \
    if (head_dim == 128)                                                     \
      hipLaunchKernelGGL((kv_read_q8_kernel<DT, 128>), g, b, 0, s, a);       \
    else                                                                     \
      hipLaunchKernelGGL((kv_read_q8_kernel<DT, 64>), g, b, 0, s, a);        \
  } while (0)
  if (dtype == IR_DTYPE_BF16) IR_READ(IR_DTYPE_BF16);
  else if (dtype == IR_DTYPE_F16) IR_READ(IR_DTYPE_F16);
  else IR_READ(IR_DTYPE_F32);
#undef IR_READ
  return check_launch(name);
}

}  // namespace
}  // namespace ir

using namespace ir;

extern "C" int ir_kv_scatter_q8(const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
                                int64_t v_tok_stride, int64_t v_head_stride, void* k_cache, void* v_cache,
                                float* scales, int64_t num_blocks, int block_size, const int64_t* slot_mapping,
                                int64_t n_tokens, int num_kv_heads, int head_dim, int dtype, int32_t* err_flags,
                                ir_stream_t stream) {
  const char* name = "ir_kv_scatter_q8";
  const int eb = dtype_bytes(dtype);
  IR_REQUIRE(eb > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(n_tokens >= 0, "%s: bad sizes", name);
  if (n_tokens == 0) return ok();
  int rc = check_pool(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(k && v && slot_mapping, "%s: null pointer", name);
  IR_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", name);
  for (int64_t st : {k_tok_stride, k_head_stride, v_tok_stride, v_head_stride})
    IR_REQUIRE((st * eb) % 16 == 0, "%s: strides must be multiples of 16 bytes", name);
  QuantArgs a = {};
  a.r.k = (const uint8_t*)k;
  a.r.k_tok = k_tok_stride * eb;
  a.r.k_head = k_head_stride * eb;
  a.r.v = (const uint8_t*)v;
  a.r.v_tok = v_tok_stride * eb;
  a.r.v_head = v_head_stride * eb;
  a.r.slots = slot_mapping;
  a.r.n_tokens = n_tokens;
  a.r.num_kv_heads = num_kv_heads;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.scales = scales;
  a.num_blocks = num_blocks;
  a.bs = block_size;
  a.err = err_flags;
  return dispatch_write(name, a, kRowsPlain, head_dim, dtype, (hipStream_t)stream);
}

extern "C" int ir_rope_kv_scatter_q8(const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out,
                                     int64_t qo_tok_stride, int64_t qo_head_stride, const void* k,
                                     int64_t k_tok_stride, int64_t k_head_stride, const void* v, int64_t v_tok_stride,
                                     int64_t v_head_stride, const void* q_weight, const void* k_weight, float eps,
                                     const float* cos, const float* sin, int64_t cs_tok_stride, void* k_cache,
                                     void* v_cache, float* scales, int64_t num_blocks, int block_size,
                                     const int64_t* slot_mapping, int64_t n_tokens, int num_q_heads, int num_kv_heads,
                                     int head_dim, int dtype, int32_t* err_flags, ir_stream_t stream) {
  const char* name = "ir_rope_kv_scatter_q8";
  const int eb = dtype_bytes(dtype);
  IR_REQUIRE(eb > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0, "%s: bad sizes", name);
  if (n_tokens == 0) return ok();
  int rc = check_pool(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  QuantArgs a = {};
  rc = fill_row_args(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k, k_tok_stride,
                     k_head_stride, v, v_tok_stride, v_head_stride, q_weight, k_weight, eps, cos, sin, cs_tok_stride,
                     slot_mapping, n_tokens, num_q_heads, num_kv_heads, eb);
  if (rc != IR_OK) return rc;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.scales = scales;
  a.num_blocks = num_blocks;
  a.bs = block_size;
  a.err = err_flags;
  return dispatch_write(name, a, q_weight ? kRowsNorm : kRowsRotate, head_dim, dtype, (hipStream_t)stream);
}

extern "C" int ir_gather_slots_q8(const void* k_cache, const void* v_cache, const float* scales, int64_t num_blocks,
                                  int block_size, const int64_t* slots, int64_t n, int num_kv_heads, int head_dim,
                                  int dtype, void* out_k, void* out_v, int32_t* err_flags, ir_stream_t stream) {
  const char* name = "ir_gather_slots_q8";
  IR_REQUIRE(dtype_bytes(dtype) > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(n >= 0, "%s: bad sizes", name);
  if (n == 0) return ok();
  const int rc = check_pool(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(slots && out_k && out_v, "%s: null pointer", name);
  IR_REQUIRE(aligned16(out_k) && aligned16(out_v), "%s: outputs must be 16-byte aligned", name);
  ReadArgs a = {};
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.scales = scales;
  a.num_blocks = num_blocks;
  a.bs = block_size;
  a.num_kv_heads = num_kv_heads;
  a.slots = slots;
  a.n = n;
  a.ok = (uint8_t*)out_k;
  a.ov = (uint8_t*)out_v;
  a.err = err_flags;
  return launch_read(name, a, head_dim, dtype, (hipStream_t)stream);
}

extern "C" int ir_paged_gather_q8(const void* k_cache, const void* v_cache, const float* scales, int64_t num_blocks,
                                  int block_size, const int32_t* block_tables, int64_t bt_stride,
                                  int max_blocks_per_seq, const int32_t* context_lens, int num_seqs, int max_ctx,
                                  int num_kv_heads, int head_dim, int dtype, void* out_k, void* out_v,
                                  int32_t* err_flags, ir_stream_t stream) {
  const char* name = "ir_paged_gather_q8";
  IR_REQUIRE(dtype_bytes(dtype) > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(num_seqs >= 0 && max_ctx >= 0 && max_blocks_per_seq >= 0, "%s: bad sizes", name);
  if (num_seqs == 0 || max_ctx == 0) return ok();
  const int rc = check_pool(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE((int64_t)max_blocks_per_seq * block_size <= (int64_t)1 << 30,
             "%s: block tables of %d x %d tokens exceed 2^30 keys", name, max_blocks_per_seq, block_size);
  IR_REQUIRE(block_tables && context_lens && out_k && out_v, "%s: null pointer", name);
  IR_REQUIRE(aligned16(out_k) && aligned16(out_v), "%s: outputs must be 16-byte aligned", name);
  ReadArgs a = {};
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.scales = scales;
  a.num_blocks = num_blocks;
  a.bs = block_size;
  a.num_kv_heads = num_kv_heads;
  a.bt = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks_per_seq;
  a.ctx = context_lens;
  a.max_ctx = max_ctx;
  a.n = (int64_t)num_seqs * max_ctx;
  a.ok = (uint8_t*)out_k;
  a.ov = (uint8_t*)out_v;
  a.err = err_flags;
  return launch_read(name, a, head_dim, dtype, (hipStream_t)stream);
}
