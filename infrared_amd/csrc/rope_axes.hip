// Rotary embedding by positions with several axes, optionally with the per-head norms
// before it and the write to a pool behind it, for gfx950: the C calls (the kernel is
// turn_rows.hpp's).
#include "status.hpp"
#include "turn_rows.hpp"

namespace ir {

int check_pool4(const char* name, const void* kc, const void* vc, const void* scales, int64_t num_blocks,
                int block_size, int num_kv_heads, int head_dim);  // kv_quant4.hip

namespace {

// What every call checks, and the arguments they share.
int fill_turn(const char* name, TurnArgs& a, const int64_t* positions, int64_t pos_axis_stride, int num_axes,
              const ir_rotary_pair* pairs, float scaling, int head_dim) {
  IR_REQUIRE(positions && pairs, "%s: null pointer", name);
  IR_REQUIRE(((uintptr_t)positions & 7u) == 0 && aligned16(pairs),
             "%s: positions must be 8-byte aligned, pairs 16-byte aligned", name);
  IR_REQUIRE(num_axes >= 1 && num_axes <= IR_ROTARY_MAX_AXES, "%s: %d axes, 1 to %d expected", name, num_axes,
             IR_ROTARY_MAX_AXES);
  IR_REQUIRE(scaling - scaling == 0.f, "%s: scaling must be finite", name);
  a.pos = positions;
  a.pos_axis = pos_axis_stride;
  a.num_axes = num_axes;
  a.pairs = pairs;
  a.scaling = scaling;
  a.head_dim = head_dim;
  return IR_OK;
}

int check_dtypes(const char* name, int dtype, int q_out_dtype) {
  IR_REQUIRE(dtype_bytes(dtype) > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(q_out_dtype == dtype || q_out_dtype == IR_DTYPE_F32, "%s: unknown q_out_dtype %d for dtype %d", name,
             q_out_dtype, dtype);
  return IR_OK;
}

template <int DT, int DST>
int launch_dst(const char* name, const TurnArgs& a, hipStream_t s) {
  if (a.r.q_weight)
    return a.head_dim == 128 ? launch_turn<DT, 128, kRowsNorm, kAnglesPositions, DST>(name, a, s)
                             : launch_turn<DT, 64, kRowsNorm, kAnglesPositions, DST>(name, a, s);
  if (a.head_dim == 128) return launch_turn<DT, 128, kRowsTurn, kAnglesPositions, DST>(name, a, s);
  if (a.head_dim == 64) return launch_turn<DT, 64, kRowsTurn, kAnglesPositions, DST>(name, a, s);
  if constexpr (DST == kToRows) return launch_turn<DT, 0, kRowsTurn, kAnglesPositions, DST>(name, a, s);
  return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported (64, 128)", name, a.head_dim);
}

template <int DST>
int dispatch(const char* name, const TurnArgs& a, int dtype, hipStream_t s) {
  switch (dtype) {
    case IR_DTYPE_BF16: return launch_dst<IR_DTYPE_BF16, DST>(name, a, s);
    case IR_DTYPE_F16: return launch_dst<IR_DTYPE_F16, DST>(name, a, s);
    default: return launch_dst<IR_DTYPE_F32, DST>(name, a, s);
  }
}

}  // namespace
}  // namespace ir

using namespace ir;

extern "C" int ir_rope_axes(const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out,
                            int64_t qo_tok_stride, int64_t qo_head_stride, const void* k, int64_t k_tok_stride,
                            int64_t k_head_stride, void* k_out, int64_t ko_tok_stride, int64_t ko_head_stride,
                            const void* q_weight, const void* k_weight, float eps, const int64_t* positions,
                            int64_t pos_axis_stride, int num_axes, const ir_rotary_pair* pairs, float scaling,
                            int64_t n_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                            int q_out_dtype, ir_stream_t stream) {
  const char* name = "ir_rope_axes";
  int rc = check_dtypes(name, dtype, q_out_dtype);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0 && num_kv_heads >= 0, "%s: bad sizes", name);
  if (head_dim <= 0 || head_dim % 16 || head_dim > 2 * kMaxPairs)
    return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported (a multiple of 16, at most %d)", name, head_dim,
                2 * kMaxPairs);
  if (q_weight && head_dim != 64 && head_dim != 128)
    return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported with norms (64, 128)", name, head_dim);
  if (n_tokens == 0 || (num_q_heads == 0 && num_kv_heads == 0)) return ok();
  const int eb = dtype_bytes(dtype);
  TurnArgs a = {};
  rc = fill_turn(name, a, positions, pos_axis_stride, num_axes, pairs, scaling, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(num_kv_heads == 0 || (k && k_out), "%s: null pointer", name);
  rc = fill_rows(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k, k_tok_stride,
                 k_head_stride, nullptr, 0, 0, q_weight, k_weight, eps, n_tokens, num_q_heads, num_kv_heads, eb,
                 dtype_bytes(q_out_dtype));
  if (rc != IR_OK) return rc;
  IR_REQUIRE(aligned16(k_out) && (ko_tok_stride * eb) % 16 == 0 && (ko_head_stride * eb) % 16 == 0,
             "%s: k_out must be 16-byte aligned with strides of multiples of 16 bytes", name);
  a.ko = (uint8_t*)k_out;
  a.ko_tok = ko_tok_stride * eb;
  a.ko_head = ko_head_stride * eb;
  return dispatch<kToRows>(name, a, dtype, (hipStream_t)stream);
}

extern "C" int ir_rope_axes_kv_scatter(
    const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out, int64_t qo_tok_stride,
    int64_t qo_head_stride, const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
    int64_t v_tok_stride, int64_t v_head_stride, const void* q_weight, const void* k_weight, float eps,
    const int64_t* positions, int64_t pos_axis_stride, int num_axes, const ir_rotary_pair* pairs, float scaling,
    void* k_cache, void* v_cache, int64_t cache_slot_stride, int64_t cache_head_stride, int64_t num_slots,
    const int64_t* slot_mapping, int64_t n_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
    int q_out_dtype, int32_t* err_flags, ir_stream_t stream) {
  const char* name = "ir_rope_axes_kv_scatter";
  int rc = check_dtypes(name, dtype, q_out_dtype);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0 && num_kv_heads > 0 && num_slots >= 0, "%s: bad sizes", name);
  if (head_dim != 64 && head_dim != 128)
    return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported (64, 128)", name, head_dim);
  if (n_tokens == 0) return ok();
  const int eb = dtype_bytes(dtype);
  TurnArgs a = {};
  rc = fill_turn(name, a, positions, pos_axis_stride, num_axes, pairs, scaling, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(k && v && slot_mapping && k_cache && v_cache, "%s: null pointer", name);
  rc = fill_rows(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k, k_tok_stride,
                 k_head_stride, v, v_tok_stride, v_head_stride, q_weight, k_weight, eps, n_tokens, num_q_heads,
                 num_kv_heads, eb, dtype_bytes(q_out_dtype));
  if (rc != IR_OK) return rc;
  IR_REQUIRE(aligned16(k_cache) && aligned16(v_cache) && (cache_slot_stride * eb) % 16 == 0 &&
                 (cache_head_stride * eb) % 16 == 0,
             "%s: caches must be 16-byte aligned with strides of multiples of 16 bytes", name);
  a.r.slots = slot_mapping;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.c_slot = cache_slot_stride * eb;
  a.c_head = cache_head_stride * eb;
  a.num_slots = num_slots;
  a.err = err_flags;
  return dispatch<kToCache>(name, a, dtype, (hipStream_t)stream);
}

extern "C" int ir_rope_axes_kv_scatter_q4(
    const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out, int64_t qo_tok_stride,
    int64_t qo_head_stride, const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
    int64_t v_tok_stride, int64_t v_head_stride, const void* q_weight, const void* k_weight, float eps,
    const int64_t* positions, int64_t pos_axis_stride, int num_axes, const ir_rotary_pair* pairs, float scaling,
    void* k_cache, void* v_cache, uint8_t* scales, int64_t num_blocks, int block_size, const int64_t* slot_mapping,
    int64_t n_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype, int q_out_dtype, int32_t* err_flags,
    ir_stream_t stream) {
  const char* name = "ir_rope_axes_kv_scatter_q4";
  int rc = check_dtypes(name, dtype, q_out_dtype);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0, "%s: bad sizes", name);
  if (n_tokens == 0) return ok();
  rc = check_pool4(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  const int eb = dtype_bytes(dtype);
  TurnArgs a = {};
  rc = fill_turn(name, a, positions, pos_axis_stride, num_axes, pairs, scaling, head_dim);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(k && v && slot_mapping, "%s: null pointer", name);
  rc = fill_rows(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k, k_tok_stride,
                 k_head_stride, v, v_tok_stride, v_head_stride, q_weight, k_weight, eps, n_tokens, num_q_heads,
                 num_kv_heads, eb, dtype_bytes(q_out_dtype));
  if (rc != IR_OK) return rc;
  a.r.slots = slot_mapping;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.scales = scales;
  a.num_slots = num_blocks * block_size;
  a.err = err_flags;
  return dispatch<kToCodes4>(name, a, dtype, (hipStream_t)stream);
}
