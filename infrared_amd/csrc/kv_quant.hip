// The 8-bit K/V pool for gfx950: new rows quantised as they are written
// (optionally normed and rotated on the way), and read back. Codes and scales are
// e4m3.hpp's; a layer is dense, [H_kv][num_blocks][block_size][D] codes for K and
// for V and [H_kv][num_blocks][2] scales.
//
// The write. A block's scale covers all its tokens, so the tokens of a call that
// share a block have to be handled together, whatever their order in the call. A
// workgroup looks after one token or a few; a token drops out if the one before it
// is in the same block (which ends most of a prompt's), else the workgroup reads
// every slot of the call once and the token drops out if an earlier one is in the
// block. The one that is left owns the block, its workgroup knows which row each of
// the block's tokens takes (the last given), and no other workgroup touches it. That is
// one launch without a workspace, and its result does not depend on the order of
// execution. The slots are 8 bytes a token against 4 KB of rows at 4 heads of 128, and
// come from L2, but every workgroup with a block to own reads them all. So those of a long
// call look after up to 256 tokens and read them once for 16 blocks (write_blocks):
// 131,072 tokens of 4 heads of 128 in order 216 us (944 with one reading a block), shuffled
// 2.6 ms (14.3); 16,384 in order 28 us (30), shuffled 89 (295). Below that a reading a block is
// as fast or faster (written and read back, 64 single tokens 7.0 us against 7.5 and 4,096
// in order 14.5 against 15.3).
//
// What bounds a call of usual size is latency: the slots, the scan, the rows and the codes follow each
// other (64 tokens 4.3 us a call, 4,096 tokens 9.8 us for 12.6 MB, 28 / 4 heads of 128,
// of which 2.7 us are the launch of workgroups that find nothing to do).
//
// A wavefront then takes K or V of one head: its rows' largest magnitude gives the
// scale, the rows become codes. A block that is not new keeps its tokens; only when
// its scale grows are they read, rounded to the wider scale and written back.
#include <algorithm>
#include <type_traits>

#include "e4m3.hpp"
#include "norm_rope.hpp"
#include "status.hpp"

namespace ir {
namespace {

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kMaxBlockSize = 1024;
constexpr int kWriteWaves = 4;
constexpr int kMaxWindow = 256;
constexpr int kWanted = 16;        // blocks found in one reading of the slots
constexpr int kWantedRows = 4096;  // their tokens
constexpr int kKeys = 256;
// Workgroups up to which each looks after one token only: four a CU (2,048 measured
// 11.8 against 10.3 us on a mixed step of 1,248 tokens, 10.1 against 9.8 on 4,096).
constexpr int64_t kWriteGroups = 1024;

struct QuantArgs {
  RowArgs r;
  uint8_t* kc;
  uint8_t* vc;
  float* scales;
  int64_t num_blocks;
  int bs;
  int window;      // tokens of the call that a workgroup looks after, at most kMaxWindow
  int kv_groups;   // workgroups per window for the 2 * H_kv (head, K / V) parts
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
  uint8_t* to = r.qo + tok * r.qo_tok + h * r.qo_head;
  if (r.qo_wide) RowPair<IR_DTYPE_F32, D>::store(to, ci, x);
  else P::store(to, ci, x);
}

// A lane's part of a new row as it is loaded, with the token's tables for a key that
// is rotated.
template <int DT, int D, int MODE>
struct NewRow {
  RowPair<DT, D> p;
  Angles<DT, D, MODE> t;
  __device__ __forceinline__ void load(const RowArgs& r, int h, int is_v, int64_t j, int ci) {
    p.load((is_v ? r.v + h * r.v_head + j * r.v_tok : r.k + h * r.k_head + j * r.k_tok), ci);
    if constexpr (MODE != kRowsPlain) t.load(r.cos + j * r.cs_tok, r.sin + j * r.cs_tok, ci);
  }
};

// What the pool holds of a lane's 16 elements before the rounding to codes: rows that
// are stored as they are stay packed in the 16-bit dtypes, where two elements take one
// instruction each for the maximum and for the codes (3 a pair instead of some 20).
template <int DT, int D, int MODE, bool PACKED>
struct RowValues {
  float x[16];
  float most;  // the largest magnitude, infinite if one is no number
  __device__ __forceinline__ void take(const NewRow<DT, D, MODE>& r, const float (&w)[16], float eps) {
    r.p.unpack(x);
    if constexpr (MODE != kRowsPlain) transform_row<DT, D, MODE>(x, w, eps, r.t);
    most = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(x[e]));  // (passes over NaN, whose code is NaN anyway)
  }
  __device__ __forceinline__ float finite_most() const {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, finite_abs(x[e]));
    return m;
  }
  __device__ __forceinline__ void careful(uint32_t (&c)[4], float inv) const {
    float z[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = to_code_range<DT>(x[e], inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = encode4(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
  }
  __device__ __forceinline__ void quick(uint32_t (&c)[4], float scale) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      i16x2 o = {0, 0};
      o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, x[4 * i], x[4 * i + 1], scale, false);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, x[4 * i + 2], x[4 * i + 3], scale, true);
      c[i] = __builtin_bit_cast(uint32_t, o);
    }
  }
};
template <int DT, int D, int MODE>
struct RowValues<DT, D, MODE, true> {
  uint32_t x[8];
  float most;
  __device__ __forceinline__ void take(const NewRow<DT, D, MODE>& r, const float (&)[16], float) {
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = i < 4 ? r.p.a.w[0][i] : r.p.b.w[0][i - 4];
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu));
    }
    constexpr uint32_t inf = DT == IR_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t u = max((uint32_t)m[0], (uint32_t)m[1]);
    most = Elem<DT>::to_f32((typename Elem<DT>::storage)min(u, inf));
  }
  __device__ __forceinline__ float at(int e) const {
    return e & 1 ? Elem<DT>::hi(x[e / 2]) : Elem<DT>::lo(x[e / 2]);
  }
  __device__ __forceinline__ float finite_most() const {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, finite_abs(at(e)));
    return m;
  }
  __device__ __forceinline__ void careful(uint32_t (&c)[4], float inv) const {
    float z[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = to_code_range<DT>(at(e), inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = encode4(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
  }
  __device__ __forceinline__ void quick(uint32_t (&c)[4], float scale) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      i16x2 o = {0, 0};
      if constexpr (DT == IR_DTYPE_BF16) {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2, x[2 * i]), scale, false);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2, x[2 * i + 1]), scale, true);
      } else {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(f16x2, x[2 * i]), scale, false);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(f16x2, x[2 * i + 1]), scale, true);
      }
      c[i] = __builtin_bit_cast(uint32_t, o);
    }
  }
};

// Writes K or V of head `h` of a block (block and head `hb`) by this wavefront: s_row
// gives the row + 1 that each of its tokens takes from the call, `old` its scale.
template <int DT, int D, int MODE>
__device__ __forceinline__ void write_part(const QuantArgs& a, int64_t i, int64_t hb, int h, int is_v, float old,
                                           const int* s_row) {
  typedef RowPair<DT, D> P;
  typedef NewRow<DT, D, MODE> Row;
  typedef RowValues<DT, D, MODE, MODE == kRowsPlain && DT != IR_DTYPE_F32> Values;
  constexpr int RPP = 64 / P::LPR;  // rows of a wavefront at a time
  const int lane = threadIdx.x & 63, ci = lane % P::LPR, grp = lane / P::LPR;
  const bool fresh = s_row[0] != 0;
  uint8_t* codes = (is_v ? a.vc : a.kc) + hb * a.bs * D;
  float w[16];
  if constexpr (MODE == kRowsNorm) {
    P pw;
    pw.load(a.r.k_weight, ci);
    pw.unpack(w);
  }
  // the rows of the block's first 16 tokens stay in registers (all their loads in
  // flight together; a token without a row loads row i, which is there), those of a
  // larger block are read once for the scale and once for the codes
  constexpr int KEEP = 16 / RPP;
  Row row[KEEP];
  Values x[KEEP];
  bool has[KEEP];
#pragma unroll
  for (int p = 0; p < KEEP; ++p) {
    const int64_t j = (int64_t)s_row[p * RPP + grp] - 1;  // (a row's lanes go together)
    has[p] = j >= 0;
    row[p].load(a.r, h, is_v, has[p] ? j : i, ci);
  }
  auto later = [&](int t, Values& y) -> bool {
    const int64_t j = (int64_t)s_row[t] - 1;
    if (j < 0) return false;
    Row r;
    r.load(a.r, h, is_v, j, ci);
    y.take(r, w, a.r.eps);
    return true;
  };
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < KEEP; ++p) {
    x[p].take(row[p], w, a.r.eps);
    amax = has[p] ? fmaxf(amax, x[p].most) : amax;
  }
  for (int t = 16 + grp; t < a.bs; t += RPP) {
    Values y;
    if (later(t, y)) amax = fmaxf(amax, y.most);
  }
  amax = wave_max(amax);
  bool careful = false;
  if (amax > __FLT_MAX__) {  // uniform: there are infinities, or NaN, which do not count
    careful = true;
    amax = 0.f;
#pragma unroll
    for (int p = 0; p < KEEP; ++p) amax = has[p] ? fmaxf(amax, x[p].finite_most()) : amax;
    for (int t = 16 + grp; t < a.bs; t += RPP) {
      Values y;
      if (later(t, y)) amax = fmaxf(amax, y.finite_most());
    }
    amax = wave_max(amax);
  }

  const int need = scale_exponent<DT>(amax);
  const int held = max(ScaleBounds<DT>::lo, min(ScaleBounds<DT>::hi, exponent_of(old)));
  const int k = fresh ? need : max(held, need);
  const bool grow = !fresh && k > held;
  careful |= k == ScaleBounds<DT>::hi;  // (magnitudes past the pool's range)
  // an old code's place under the wider scale: below 2^-100 every code is zero
  const float shrink = pow2(max(held - k, -100));
  auto put = [&](int t, bool has_row, const Values& y) {
    u32x2* p0 = (u32x2*)(codes + (int64_t)t * D + 8 * ci);
    u32x2* p1 = (u32x2*)(codes + (int64_t)t * D + 8 * ci + D / 2);
    uint32_t c[4] = {0u, 0u, 0u, 0u};
    if (has_row) {
      if (careful) y.careful(c, pow2(-k));
      else y.quick(c, pow2(k));
    } else if (grow) {
      const u32x2 c0 = *p0, c1 = *p1;
      auto again = [&](uint32_t was) {
        const f32x2 lo = decode2_f32<false>(was, shrink), hi = decode2_f32<true>(was, shrink);
        return encode4(lo[0], lo[1], hi[0], hi[1]);
      };
      c[0] = again(c0[0]);
      c[1] = again(c0[1]);
      c[2] = again(c1[0]);
      c[3] = again(c1[1]);
    } else if (!fresh) {
      return;
    }
    *p0 = u32x2{c[0], c[1]};
    *p1 = u32x2{c[2], c[3]};
  };
#pragma unroll
  for (int p = 0; p < KEEP; ++p) put(p * RPP + grp, has[p], x[p]);
  for (int t = 16 + grp; t < a.bs; t += RPP) {
    Values y;
    const bool has_row = later(t, y);
    put(t, has_row, y);
  }
  if (lane == 0) a.scales[2 * hb + is_v] = pow2(k);
}

// Writes block `blk`, if token i is the call's first of it: part `part` (K or V of a
// head) by this wavefront. s_row [kMaxBlockSize], s_earlier: LDS. The whole workgroup
// calls it alike, parts past the last included.
template <int DT, int D, int MODE>
__device__ __forceinline__ void write_block(const QuantArgs& a, int64_t i, int blk, int part, int* s_row,
                                            int* s_earlier) {
  constexpr int NT = kWriteWaves * 64;
  const int tid = threadIdx.x;
  const int64_t base = (int64_t)blk * a.bs;
  const bool active = part < 2 * a.r.num_kv_heads;
  const int h = part >> 1, is_v = part & 1;
  const int64_t hb = (int64_t)h * a.num_blocks + blk;
  float old = 0.f;
  if (active) old = a.scales[2 * hb + is_v];
  // ---- the block's tokens in this call: row + 1 that each takes, 0: none
  __syncthreads();  // (the last block's readers are done)
  for (int t = tid; t < a.bs; t += NT) s_row[t] = 0;
  if (tid == 0) *s_earlier = 0;
  __syncthreads();
  constexpr int SCAN = 8;  // slots of a lane in flight together
  for (int64_t j0 = tid; j0 < a.r.n_tokens; j0 += SCAN * NT) {
    int64_t slot[SCAN];
#pragma unroll
    for (int u = 0; u < SCAN; ++u) slot[u] = j0 + u * NT < a.r.n_tokens ? a.r.slots[j0 + u * NT] : -1;
#pragma unroll
    for (int u = 0; u < SCAN; ++u) {
      const uint64_t o = (uint64_t)slot[u] - (uint64_t)base;
      if (o < (uint64_t)a.bs) {
        atomicMax(&s_row[(int)o], (int)(j0 + u * NT) + 1);
        if (j0 + u * NT < i) *s_earlier = 1;
      }
    }
  }
  __syncthreads();
  if (*s_earlier || !active) return;  // another workgroup's block

  // ---- this wavefront's head, K or V
  if (MODE == kRowsPlain || is_v)
    write_part<DT, D, kRowsPlain>(a, i, hb, h, is_v, old, s_row);
  else
    write_part<DT, D, MODE>(a, i, hb, h, is_v, old, s_row);
}

struct OneBlock {
  int row[kMaxBlockSize], earlier;
};

// Blocks a workgroup is after at a time, with the rows that their tokens take.
struct Wanted {
  int blk[kWanted], earlier[kWanted];
  int64_t tok[kWanted];
  int row[kWantedRows];  // [wanted][block_size]: row + 1, 0: none
  int key[kKeys], of[kKeys];  // open addressing: block (-1: none), the first wanted that names it
};

// Where block `blk` is in the table, or would be: an entry of it or an empty one.
__device__ __forceinline__ int find_key(const Wanted& s, int blk) {
  int p = blk & (kKeys - 1);
  for (int key = s.key[p]; key != blk && key != -1; key = s.key[p]) p = (p + 1) & (kKeys - 1);
  return p;
}

// Writes those of the `count` wanted blocks whose token is the call's first of the block:
// part `part` (K or V of a head) by this wavefront. The whole workgroup calls it alike,
// parts past the last included; blk and tok are set, with no barrier behind them yet.
template <int DT, int D, int MODE>
__device__ __forceinline__ void write_blocks(const QuantArgs& a, int count, int part, Wanted& s) {
  constexpr int NT = kWriteWaves * 64;
  const int tid = threadIdx.x, lane = tid & 63;
  const bool active = part < 2 * a.r.num_kv_heads;
  const int h = part >> 1, is_v = part & 1;
  const int64_t h0 = (int64_t)h * a.num_blocks;
  for (int t = tid; t < count * a.bs; t += NT) s.row[t] = 0;
  if (tid < kWanted) s.earlier[tid] = 0;
  for (int t = tid; t < kKeys; t += NT) {
    s.key[t] = -1;
    s.of[t] = kWanted;
  }
  __syncthreads();
  float old = 0.f;  // lane c: the scale of wanted block c
  if (active && lane < count) old = a.scales[2 * (h0 + s.blk[lane]) + is_v];
  if (tid < count) {
    int p = s.blk[tid] & (kKeys - 1);
    for (;;) {  // (at most 16 of 256 entries are taken)
      const int was = atomicCAS(&s.key[p], -1, s.blk[tid]);
      if (was == -1 || was == s.blk[tid]) break;
      p = (p + 1) & (kKeys - 1);
    }
    atomicMin(&s.of[p], tid);
  }
  __syncthreads();
  // ---- the blocks' tokens in this call
  const int64_t num_slots = a.num_blocks * a.bs;
  constexpr int SCAN = 8;  // slots of a lane in flight together
  for (int64_t j0 = tid; j0 < a.r.n_tokens; j0 += SCAN * NT) {
    int64_t slot[SCAN];
#pragma unroll
    for (int u = 0; u < SCAN; ++u) slot[u] = j0 + u * NT < a.r.n_tokens ? a.r.slots[j0 + u * NT] : -1;
#pragma unroll
    for (int u = 0; u < SCAN; ++u) {
      if ((uint64_t)slot[u] >= (uint64_t)num_slots) continue;  // (slots fit 31 bits)
      const int blk = (int)((uint32_t)slot[u] / (uint32_t)a.bs);
      const int p = find_key(s, blk);
      if (s.key[p] == -1) continue;
      const int c = s.of[p];
      atomicMax(&s.row[c * a.bs + ((int)slot[u] - blk * a.bs)], (int)(j0 + u * NT) + 1);
      if (j0 + u * NT < s.tok[c]) s.earlier[c] = 1;
    }
  }
  __syncthreads();

  // ---- this wavefront's head, K or V
  for (int c = 0; c < count; ++c) {
    const int blk = s.blk[c];
    if (s.earlier[c] || !active || s.of[find_key(s, blk)] != c) continue;  // another's block
    const float was = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(old), c));
    if (MODE == kRowsPlain || is_v)
      write_part<DT, D, kRowsPlain>(a, s.tok[c], h0 + blk, h, is_v, was, s.row + c * a.bs);
    else
      write_part<DT, D, MODE>(a, s.tok[c], h0 + blk, h, is_v, was, s.row + c * a.bs);
  }
}

// A workgroup's place among the n of the write. Those of a prompt that own a block come
// every block_size tokens, and workgroup b runs on XCD b mod 8: in their own order all
// of them would share one or two XCDs (16.5 us for a mixed step's 1,248 tokens, 13.7
// spread out). Each run of 8 is rotated by the sum of its index's octal digits, so that places
// any power of two apart fall on all of them.
__device__ __forceinline__ uint32_t spread_xcds(uint32_t b, uint32_t n) {
  const uint32_t k = b >> 3;
  if (8 * k + 8 > n) return b;  // a last, shorter run
  const uint32_t turn = k + (k >> 3) + (k >> 6) + (k >> 9) + (k >> 12) + (k >> 15) + (k >> 18);
  return 8 * k + ((b + turn) & 7u);
}

// MANY: windows of more than 16 tokens.
template <int DT, int D, int MODE, bool MANY>
__global__ __launch_bounds__(kWriteWaves * 64) void kv_write_q8_kernel(QuantArgs a) {
  __shared__ std::conditional_t<MANY, Wanted, OneBlock> s;
  if constexpr (MODE != kRowsPlain) {
    if (blockIdx.x >= a.n_kv) {
      query_rows<DT, D, MODE>(a.r, (blockIdx.x - a.n_kv) * kWriteWaves + (threadIdx.x >> 6));
      return;
    }
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t group = spread_xcds(blockIdx.x, (uint32_t)a.n_kv);
  const int64_t wi = group / (uint32_t)a.kv_groups;
  const int part = (int)(group - wi * a.kv_groups) * kWriteWaves + (tid >> 6);
  const int64_t num_slots = a.num_blocks * a.bs;
  const int64_t i0 = wi * a.window;
  const int wn = (int)min((int64_t)a.window, a.r.n_tokens - i0);
  // lane l: token first + l of the window; it may own its block unless the token before it
  // is in the same one. What follows is uniform over the workgroup: every wavefront looks at
  // the same window.
  int my_blk = -1;
  auto owners = [&](int64_t first) -> uint64_t {
    const bool in = first + lane < i0 + wn;
    const int64_t my_slot = in ? a.r.slots[first + lane] : -1;
    const int64_t before = in && first + lane > 0 ? a.r.slots[first + lane - 1] : -1;
    const bool valid = my_slot >= 0 && my_slot < num_slots;  // (negative: padding)
    if (my_slot >= num_slots && part == 0) flag_error(a.err, IR_ERR_SLOT_RANGE);
    my_blk = valid ? (int)((uint32_t)my_slot / (uint32_t)a.bs) : -1;  // (slots fit 31 bits)
    const int64_t my_base = (int64_t)my_blk * a.bs;
    return __ballot(valid && !(before >= my_base && before < my_base + a.bs));
  };
  if constexpr (!MANY) {
    for (uint64_t todo = owners(i0); todo; todo &= todo - 1) {
      const int at = __builtin_ctzll(todo);
      write_block<DT, D, MODE>(a, i0 + at, __builtin_amdgcn_readlane(my_blk, at), part, s.row, &s.earlier);
    }
  } else {
    const int most = min(kWanted, kWantedRows / a.bs);
    int count = 0;
    for (int64_t first = i0; first < i0 + wn; first += 64)
      for (uint64_t todo = owners(first); todo; todo &= todo - 1) {
        const int at = __builtin_ctzll(todo), blk = __builtin_amdgcn_readlane(my_blk, at);
        if (tid == 0) {
          s.blk[count] = blk;
          s.tok[count] = first + at;
        }
        if (++count < most) continue;
        write_blocks<DT, D, MODE>(a, count, part, s);
        __syncthreads();  // (its readers are done before the next are set)
        count = 0;
      }
    if (count) write_blocks<DT, D, MODE>(a, count, part, s);
  }
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
  C::store_nt(a.ok + idx * 8 * C::EB, k8);
  C::store_nt(a.ov + idx * 8 * C::EB, v8);
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
  // one token a workgroup until the workgroups fill the device, then as many as keep
  // it filled: in a prompt most tokens own no block, in a decode step each does; past 16
  // they share the reading of the slots
  a.window = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxWindow, a.r.n_tokens * a.kv_groups / kWriteGroups));
  a.n_kv = (a.r.n_tokens + a.window - 1) / a.window * a.kv_groups;
  const int64_t runs = (a.r.num_q_heads + G - 1) / G;
  const int64_t n_q = mode == kRowsPlain ? 0 : (a.r.n_tokens * runs + kWriteWaves - 1) / kWriteWaves;
  IR_REQUIRE(a.r.n_tokens < 0x7fffffff && a.n_kv + n_q <= 0x7fffffff, "%s: too many tokens", name);
  const dim3 grid((unsigned)(a.n_kv + n_q)), block(kWriteWaves * 64);
  const bool many = a.window > 16;
#define IR_WRITE(MODE_)                                                                         \
  do {                                                                                          \
    if (many)                                                                                   \
      hipLaunchKernelGGL((kv_write_q8_kernel<DT, D, MODE_, true>), grid, block, 0, s, a);       \
    else                                                                                        \
      hipLaunchKernelGGL((kv_write_q8_kernel<DT, D, MODE_, false>), grid, block, 0, s, a);      \
  } while (0)
  if (mode == kRowsPlain) IR_WRITE(kRowsPlain);
  else if (mode == kRowsNorm) IR_WRITE(kRowsNorm);
  else IR_WRITE(kRowsRotate);
#undef IR_WRITE
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
                                     int head_dim, int dtype, int q_out_dtype, int32_t* err_flags,
                                     ir_stream_t stream) {
  const char* name = "ir_rope_kv_scatter_q8";
  const int eb = dtype_bytes(dtype);
  IR_REQUIRE(eb > 0, "%s: unknown dtype %d", name, dtype);
  IR_REQUIRE(q_out_dtype == dtype || q_out_dtype == IR_DTYPE_F32, "%s: unknown q_out_dtype %d for dtype %d", name,
             q_out_dtype, dtype);
  IR_REQUIRE(n_tokens >= 0 && num_q_heads >= 0, "%s: bad sizes", name);
  if (n_tokens == 0) return ok();
  int rc = check_pool(name, k_cache, v_cache, scales, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != IR_OK) return rc;
  QuantArgs a = {};
  rc = fill_row_args(name, a.r, q, q_tok_stride, q_head_stride, q_out, qo_tok_stride, qo_head_stride, k, k_tok_stride,
                     k_head_stride, v, v_tok_stride, v_head_stride, q_weight, k_weight, eps, cos, sin, cs_tok_stride,
                     slot_mapping, n_tokens, num_q_heads, num_kv_heads, eb, dtype_bytes(q_out_dtype));
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
