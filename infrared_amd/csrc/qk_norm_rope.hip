// Norms of queries and keys for each head, position rotation and KV-slot scatter
// in one launch for gfx950: the row mathematics is norm_rope.hpp's.
//
// Bound by memory: every row is read once and written once, beside the token's
// cos and sin rows. A wavefront takes one token and 64 / (head_dim / 16) of its rows
// (q, then k, then v) at a time, its lanes holding their part of the token's tables
// in registers for all of them. 4,096 tokens of 28 / 4 heads of 128 in bf16 (79.7 MB):
// 14.9 us a call, 5.3 TB/s, where a copy of 2 GiB runs at 4.9 (with stores that stay in
// L2 17.4 us); 64 tokens 3.2 us, the launch and two trips to memory.
#include <algorithm>

#include "norm_rope.hpp"
#include "status.hpp"

namespace ir {
namespace {

struct NormRopeArgs {
  RowArgs r;
  uint8_t* kc;
  uint8_t* vc;
  int64_t c_slot, c_head;  // bytes
  int64_t num_slots;
  int chunks, chunk_rows;  // wavefronts per token, rows of each
  int32_t* err;
};

template <int DT, int D>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeArgs a) {
  typedef RowPair<DT, D> P;
  constexpr int G = 64 / P::LPR;  // rows of a wavefront at a time
  const int lane = threadIdx.x & 63, ci = lane % P::LPR, grp = lane / P::LPR;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t tok = wave / a.chunks;
  if (tok >= a.r.n_tokens) return;
  const int nq = a.r.num_q_heads, nkv = a.r.num_kv_heads, rows = nq + 2 * nkv;
  const int row0 = (int)(wave - tok * a.chunks) * a.chunk_rows;
  const int row_end = min(rows, row0 + a.chunk_rows);
  const int64_t slot = a.r.slots[tok];
  const bool kv_ok = slot >= 0 && slot < a.num_slots;
  if (slot >= a.num_slots && lane == 0 && row0 == 0) flag_error(a.err, IR_ERR_SLOT_RANGE);
  Angles<DT, D, kRowsNorm> t;
  t.load(a.r.cos + tok * a.r.cs_tok, a.r.sin + tok * a.r.cs_tok, ci);
  P wq, wk;
  wq.load(a.r.q_weight, ci);
  wk.load(a.r.k_weight, ci);
  for (int row = row0 + grp; row < row_end; row += G) {
    const bool is_q = row < nq, is_v = row >= nq + nkv;
    const int h = is_q ? row : is_v ? row - nq - nkv : row - nq;
    const uint8_t* src = is_q   ? a.r.q + tok * a.r.q_tok + h * a.r.q_head
                         : is_v ? a.r.v + tok * a.r.v_tok + h * a.r.v_head
                                : a.r.k + tok * a.r.k_tok + h * a.r.k_head;
    P p;
    p.load(src, ci);
    if (!is_q && !kv_ok) continue;  // (a row's lanes go together)
    uint8_t* dst = is_q ? a.r.qo + tok * a.r.qo_tok + h * a.r.qo_head
                        : (is_v ? a.vc : a.kc) + slot * a.c_slot + h * a.c_head;
    if (is_v) {
      p.store_raw(dst, ci);
      continue;
    }
    float x[16], w[16];
    p.unpack(x);
    (is_q ? wq : wk).unpack(w);
    transform_row<DT, D, kRowsNorm>(x, w, a.r.eps, t);
    P::store(dst, ci, x);
  }
}

// Wavefronts of a token: one for all its rows once the tokens alone fill the
// device, which then loads the tables once a token (4,096 tokens: 14.9 us, one for
// each run of rows 17.4); below that one for each run of rows, so that a decode step's
// few tokens are a single pass.
constexpr int64_t kTokensForDevice = 2048;

template <int DT, int D>
int launch_norm_rope(NormRopeArgs& a, hipStream_t s) {
  const int rows = a.r.num_q_heads + 2 * a.r.num_kv_heads, g = 64 / (D / 16);
  const int runs = (rows + g - 1) / g;
  a.chunks = a.r.n_tokens >= kTokensForDevice ? 1 : runs;
  a.chunk_rows = a.chunks == 1 ? rows : g;
  const int64_t grid = (a.r.n_tokens * a.chunks + 3) / 4;
  IR_REQUIRE(grid <= 0x7fffffff, "ir_qk_norm_rope_kv_scatter: too many tokens");
  hipLaunchKernelGGL((qk_norm_rope_kernel<DT, D>), dim3((unsigned)grid), dim3(256), 0, s, a);
  return check_launch("ir_qk_norm_rope_kv_scatter");
}

}  // namespace

int fill_rows(const char* name, RowArgs& r, const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok,
              int64_t qo_head, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
              int64_t v_head, const void* q_weight, const void* k_weight, float eps, int64_t n_tokens,
              int num_q_heads, int num_kv_heads, int eb, int qo_eb) {
  IR_REQUIRE(num_q_heads == 0 || (q && q_out), "%s: null pointer", name);
  IR_REQUIRE(aligned16(k) && aligned16(v) && (num_q_heads == 0 || (aligned16(q) && aligned16(q_out))),
             "%s: tensors must be 16-byte aligned", name);
  IR_REQUIRE(!q_weight == !k_weight, "%s: one norm weight without the other", name);
  IR_REQUIRE(aligned16(q_weight) && aligned16(k_weight), "%s: norm weights must be 16-byte aligned", name);
  IR_REQUIRE(!q_weight || eps >= 0.f, "%s: eps must not be negative", name);
  for (int64_t st : {qo_tok, qo_head})
    IR_REQUIRE((st * qo_eb) % 16 == 0, "%s: strides must be multiples of 16 bytes", name);
  for (int64_t st : {q_tok, q_head, k_tok, k_head, v_tok, v_head})
    IR_REQUIRE((st * eb) % 16 == 0, "%s: strides must be multiples of 16 bytes", name);
  r.q = (const uint8_t*)q;
  r.q_tok = q_tok * eb;
  r.q_head = q_head * eb;
  r.qo = (uint8_t*)q_out;
  r.qo_wide = qo_eb != eb;
  r.qo_tok = qo_tok * qo_eb;
  r.qo_head = qo_head * qo_eb;
  r.k = (const uint8_t*)k;
  r.k_tok = k_tok * eb;
  r.k_head = k_head * eb;
  r.v = (const uint8_t*)v;
  r.v_tok = v_tok * eb;
  r.v_head = v_head * eb;
  r.q_weight = (const uint8_t*)q_weight;
  r.k_weight = (const uint8_t*)k_weight;
  r.eps = eps;
  r.n_tokens = n_tokens;
  r.num_q_heads = num_q_heads;
  r.num_kv_heads = num_kv_heads;
  return IR_OK;
}

int fill_row_args(const char* name, RowArgs& r, const void* q, int64_t q_tok, int64_t q_head, void* q_out,
                  int64_t qo_tok, int64_t qo_head, const void* k, int64_t k_tok, int64_t k_head, const void* v,
                  int64_t v_tok, int64_t v_head, const void* q_weight, const void* k_weight, float eps,
                  const float* cos, const float* sin, int64_t cs_tok, const int64_t* slots, int64_t n_tokens,
                  int num_q_heads, int num_kv_heads, int eb, int qo_eb) {
  IR_REQUIRE(k && v && cos && sin && slots && (num_q_heads == 0 || (q && q_out)), "%s: null pointer", name);
  IR_REQUIRE(aligned16(cos) && aligned16(sin), "%s: tensors must be 16-byte aligned", name);
  IR_REQUIRE(cs_tok % 4 == 0, "%s: cos/sin row stride must be a multiple of 4 elements", name);
  const int rc = fill_rows(name, r, q, q_tok, q_head, q_out, qo_tok, qo_head, k, k_tok, k_head, v, v_tok, v_head,
                           q_weight, k_weight, eps, n_tokens, num_q_heads, num_kv_heads, eb, qo_eb);
  if (rc != IR_OK) return rc;
  r.cos = cos;
  r.sin = sin;
  r.cs_tok = cs_tok;
  r.slots = slots;
  return IR_OK;
}

}  // namespace ir

using namespace ir;

extern "C" int ir_qk_norm_rope_kv_scatter(
    const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out, int64_t qo_tok_stride,
    int64_t qo_head_stride, const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
    int64_t v_tok_stride, int64_t v_head_stride, const void* q_weight, const void* k_weight, float eps,
    const float* cos, const float* sin, int64_t cs_tok_stride, void* k_cache, void* v_cache,
    int64_t cache_slot_stride, int64_t cache_head_stride, int64_t num_slots, const int64_t* slot_mapping,
    int64_t n_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype, int32_t* err_flags,
    ir_stream_t stream) {
  const char* name = "ir_qk_norm_rope_kv_scatter";
  const int eb = dtype_bytes(dtype);
  IR_REQUIRE(eb > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0 && num_kv_heads > 0 && num_slots >= 0, "%s: bad sizes", name);
  if (head_dim != 64 && head_dim != 128)
    return fail(IR_EUNSUPPORTED, "%s: head_dim %d not supported (64, 128)", name, head_dim);
  if (n_tokens == 0) return ok();
  NormRopeArgs a;
  const int rc = fill_row_args(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k,
                               k_tok_stride, k_head_stride, v, v_tok_stride, v_head_stride, q_weight, k_weight, eps,
                               cos, sin, cs_tok_stride, slot_mapping, n_tokens, num_q_heads, num_kv_heads, eb, eb);
  if (rc != IR_OK) return rc;
  IR_REQUIRE(q_weight && k_cache && v_cache, "%s: null pointer", name);
  IR_REQUIRE(aligned16(k_cache) && aligned16(v_cache) && (cache_slot_stride * eb) % 16 == 0 &&
                 (cache_head_stride * eb) % 16 == 0,
             "%s: caches must be 16-byte aligned with strides of multiples of 16 bytes", name);
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.c_slot = cache_slot_stride * eb;
  a.c_head = cache_head_stride * eb;
  a.num_slots = num_slots;
  a.err = err_flags;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case IR_DTYPE_BF16:
      return head_dim == 128 ? launch_norm_rope<IR_DTYPE_BF16, 128>(a, s) : launch_norm_rope<IR_DTYPE_BF16, 64>(a, s);
    case IR_DTYPE_F16:
      return head_dim == 128 ? launch_norm_rope<IR_DTYPE_F16, 128>(a, s) : launch_norm_rope<IR_DTYPE_F16, 64>(a, s);
    default:
      return head_dim == 128 ? launch_norm_rope<IR_DTYPE_F32, 128>(a, s) : launch_norm_rope<IR_DTYPE_F32, 64>(a, s);
  }
}
