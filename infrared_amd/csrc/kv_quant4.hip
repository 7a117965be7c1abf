// The 4-bit K/V pool for gfx950: new rows quantised as they are written (optionally normed
// and rotated on the way, turn_rows.hpp), and read back. Codes, scales and the order of a
// tile are e2m1.hpp's; a layer is dense, [H_kv][tiles][8 D] bytes of codes for K and for V
// and [H_kv][tiles][D] of scales.
//
// A token's scales are its own, so the write is one pass over the rows without a workspace,
// an order among the tokens, or reading what the pool holds.
#include "status.hpp"
#include "turn_rows.hpp"

namespace ir {

// What every call on the pool checks.
int check_pool4(const char* name, const void* kc, const void* vc, const void* scales, int64_t num_blocks,
                int block_size, int num_kv_heads, int head_dim) {
  IR_REQUIRE(num_kv_heads > 0 && num_blocks >= 0, "%s: bad sizes", name);
  IR_REQUIRE(block_size > 0 && block_size % 16 == 0 && block_size <= 1024,
             "%s: block size %d must be a multiple of 16, at most 1024", name, block_size);
  if (head_dim != 64 && head_dim != 128)
    return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported (64, 128)", name, head_dim);
  IR_REQUIRE(num_blocks < ((int64_t)1 << 31) && num_blocks * block_size < ((int64_t)1 << 31),
             "%s: %lld blocks of %d tokens exceed 2^31 slots", name, (long long)num_blocks, block_size);
  IR_REQUIRE(kc && vc && scales, "%s: null pointer", name);
  IR_REQUIRE(aligned16(kc) && aligned16(vc) && aligned16(scales), "%s: caches and scales must be 16-byte aligned",
             name);
  return IR_OK;
}

namespace {

struct ReadArgs {
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* scales;
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

// One lane per 8 codes of an output row's head, K and V. Bound by memory, the rows it
// writes above all (65,536 rows of 4 heads of 128 in bf16: 26.1 us, 6.5 TB/s).
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_read_q4_kernel(ReadArgs a) {
  typedef Chunk8<DT> C;
  typedef Tile4<D> T;
  constexpr int PIECES = D / 8;
  const int64_t idx = (int64_t)near_block(blockIdx.x) * 256 + threadIdx.x;
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
  uint32_t k8[2 * C::EB] = {}, v8[2 * C::EB] = {};
  if (slot >= 0) {
    const int64_t tile = (int64_t)h * (a.num_blocks * a.bs >> 4) + (slot >> 4);
    const int t = (int)(slot & 15), grp = piece >> 2;
    const uint8_t* vt = a.vc + tile * T::CODES;
    const uint8_t* sc = a.scales + tile * T::SCALES;
    const uint32_t kw = *(const uint32_t*)(a.kc + tile * T::CODES + T::k(t, piece));
    uint32_t vw;
    if constexpr (D == 128)
      vw = *(const uint32_t*)(vt + T::v(t, piece));
    else
      vw = *(const uint16_t*)(vt + T::v(t, 2 * piece)) | (uint32_t)*(const uint16_t*)(vt + T::v(t, 2 * piece + 1)) << 16;
    decode8_e2m1<DT>(kw, scale_of_byte(sc[T::k_scale(t, grp)]), k8);
    decode8_e2m1<DT>(vw, scale_of_byte(sc[T::v_scale(t, grp)]), v8);
  }
#pragma unroll
  for (int i = 0; i < C::EB / 2; ++i) {
    __builtin_nontemporal_store(u32x4{k8[4 * i], k8[4 * i + 1], k8[4 * i + 2], k8[4 * i + 3]},
                                (u32x4*)(a.ok + idx * 8 * C::EB + 16 * i));
    __builtin_nontemporal_store(u32x4{v8[4 * i], v8[4 * i + 1], v8[4 * i + 2], v8[4 * i + 3]},
                                (u32x4*)(a.ov + idx * 8 * C::EB + 16 * i));
  }
}

template <int DT, int D>
int launch_write(const char* name, const TurnArgs& a, int mode, hipStream_t s) {
  if (mode == kRowsPlain) return launch_turn<DT, D, kRowsPlain, kAnglesNone, kToCodes4>(name, a, s);
  if (mode == kRowsNorm) return launch_turn<DT, D, kRowsNorm, kAnglesTables, kToCodes4>(name, a, s);
  return launch_turn<DT, D, kRowsRotate, kAnglesTables, kToCodes4>(name, a, s);
}

int dispatch_write(const char* name, const TurnArgs& a, int mode, int head_dim, int dtype, hipStream_t s) {
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
  const int64_t grid = near_blocks((lanes + 255) / 256);
  IR_REQUIRE(grid <= 0x7fffffff, "%s: too many rows", name);
  const dim3 g((unsigned)grid), b(256);
#define IR_READ(DT)                                                          \
  do {                                                                       \
    if (head_dim == 128)                                                     \
      hipLaunchKernelGGL((kv_read_q4_kernel<DT, 128>), g, b, 0, s, a);       \
    else                                                                     \
      hipLaunchKernelGGL((kv_read_q4_kernel<DT, 64>), g, b, 0, s, a);        \
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

extern "C" int ir_kv_scatter_q4(const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
                                int64_t v_tok_stride, int64_t v_head_stride, void* k_cache, void* v_cache,
                                uint8_t* scales, int64_t num_blocks, int block_size, const int64_t* slot_mapping,
                                int64_t n_tokens, int num_kv_heads, int head_dim, int dtype, int32_t* err_flags,
                                ir_stream_t stream) {
  const char* name = "ir_kv_scatter_q4";
  const int eb = dtype_bytes(dtype);
  IR_REQUIRE(eb > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(n_tokens >= 0, "%s: bad sizes", name);
  if (n_tokens == 0) return ok();
  int rc = check_pool4(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(k && v && slot_mapping, "%s: null pointer", name);
  TurnArgs a = {};
  rc = fill_rows(name, a.r, nullptr, 0, 0, nullptr, 0, 0, k, k_tok_stride, k_head_stride, v, v_tok_stride,
                 v_head_stride, nullptr, nullptr, 0.f, n_tokens, 0, num_kv_heads, eb, eb);
  if (rc != IR_OK) return rc;
  a.r.slots = slot_mapping;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.scales = scales;
  a.num_slots = num_blocks * block_size;
  a.err = err_flags;
  return dispatch_write(name, a, kRowsPlain, head_dim, dtype, (hipStream_t)stream);
}

extern "C" int ir_rope_kv_scatter_q4(const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out,
                                     int64_t qo_tok_stride, int64_t qo_head_stride, const void* k,
                                     int64_t k_tok_stride, int64_t k_head_stride, const void* v, int64_t v_tok_stride,
                                     int64_t v_head_stride, const void* q_weight, const void* k_weight, float eps,
                                     const float* cos, const float* sin, int64_t cs_tok_stride, void* k_cache,
                                     void* v_cache, uint8_t* scales, int64_t num_blocks, int block_size,
                                     const int64_t* slot_mapping, int64_t n_tokens, int num_q_heads, int num_kv_heads,
                                     int head_dim, int dtype, int q_out_dtype, int32_t* err_flags,
                                     ir_stream_t stream) {
  const char* name = "ir_rope_kv_scatter_q4";
  const int eb = dtype_bytes(dtype);
  IR_REQUIRE(eb > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(q_out_dtype == dtype || q_out_dtype == IR_DTYPE_F32, "%s: unknown q_out_dtype %d for dtype %d", name,
             q_out_dtype, dtype);
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0, "%s: bad sizes", name);
  if (n_tokens == 0) return ok();
  int rc = check_pool4(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  TurnArgs a = {};
  rc = fill_row_args(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k, k_tok_stride,
                     k_head_stride, v, v_tok_stride, v_head_stride, q_weight, k_weight, eps, cos, sin, cs_tok_stride,
                     slot_mapping, n_tokens, num_q_heads, num_kv_heads, eb, dtype_bytes(q_out_dtype));
  if (rc != IR_OK) return rc;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.scales = scales;
  a.num_slots = num_blocks * block_size;
  a.err = err_flags;
  return dispatch_write(name, a, q_weight ? kRowsNorm : kRowsRotate, head_dim, dtype, (hipStream_t)stream);
}

extern "C" int ir_gather_slots_q4(const void* k_cache, const void* v_cache, const uint8_t* scales, int64_t num_blocks,
                                  int block_size, const int64_t* slots, int64_t n, int num_kv_heads, int head_dim,
                                  int dtype, void* out_k, void* out_v, int32_t* err_flags, ir_stream_t stream) {
  const char* name = "ir_gather_slots_q4";
  IR_REQUIRE(dtype_bytes(dtype) > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(n >= 0, "%s: bad sizes", name);
  if (n == 0) return ok();
  const int rc = check_pool4(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
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

extern "C" int ir_paged_gather_q4(const void* k_cache, const void* v_cache, const uint8_t* scales, int64_t num_blocks,
                                  int block_size, const int32_t* block_tables, int64_t bt_stride,
                                  int max_blocks_per_seq, const int32_t* context_lens, int num_seqs, int max_ctx,
                                  int num_kv_heads, int head_dim, int dtype, void* out_k, void* out_v,
                                  int32_t* err_flags, ir_stream_t stream) {
  const char* name = "ir_paged_gather_q4";
  IR_REQUIRE(dtype_bytes(dtype) > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(num_seqs >= 0 && max_ctx >= 0 && max_blocks_per_seq >= 0, "%s: bad sizes", name);
  if (num_seqs == 0 || max_ctx == 0) return ok();
  const int rc = check_pool4(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
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
