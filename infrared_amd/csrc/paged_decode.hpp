// Device building blocks of the GQA paged decode kernel (one query token per
// sequence, paged_decode.hip).
//
// A "unit" is (sequence, KV head, group of <= 16 query heads of that KV head):
// the K/V rows of one KV head serve every query head of the group, so a unit
// reads each of its keys exactly once. A unit's keys are cut into 16-token
// tiles; the wavefronts of a workgroup take a run of tiles round-robin. Per
// tile a wavefront
//   1. loads the 16 K rows and 16 V rows of its KV head straight from the pool
//      with 16-byte loads (each row of one head is head_dim contiguous
//      elements),
//   2. scores S^T[token][head] = K . Q^T with MFMA (rows = 16 tokens, columns =
//      the group's query heads, padded to 16),
//   3. runs the online softmax in base 2 on the MFMA accumulator,
//   4. accumulates O^T[d][head] += V^T . P^T with MFMA (the P^T operand is the
//      lane's own four probabilities, V^T a register-level transpose).
// Loads run DEPTH-1 tiles ahead of the math (a register ring), and the block
// ids of a wavefront's tiles are fetched up front, one per lane, so no tile
// load waits on a block-table read.
//
// Algorithm parity: the one-shot softmax of infrared/model/layers.py:102-118
// over the gathered history (infrared/model/triton_attention.py:110-129), with
// the streaming max/sum update of infrared/model/triton_attention.py:135-177 and
// the exp2 fold of infrared/model/triton_attention.py:249. For 16-bit dtypes
// the probabilities are rounded to the input dtype before the PV product, as
// `softmax(scores.float()).to(q.dtype)` does in the reference. Over an 8-bit cache
// they take two pieces of the dtype, which shows in no output (64 sequences of 512..4096
// keys 33.1 us against 32.7 of one piece; errors of the outputs 0.0017 against 0.0023).
#pragma once

#include <type_traits>

#include "attn_tile.hpp"
#include "e4m3.hpp"

namespace ir {

constexpr int kMaxWaveTiles = 64;  // tiles per wavefront and run (one block id per lane)
constexpr int kMaxPartition = 16 * kMaxWaveTiles * 4;  // tokens (4 wavefronts)

struct DecodeArgs {
  const void* q;
  int64_t q_seq, q_head;  // elements
  const void* kc;
  const void* vc;
  int64_t c_slot, c_head;  // elements
  int64_t num_blocks;
  int bs;
  const int32_t* bt;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* ctx;
  void* out;
  int64_t o_seq, o_head;  // elements
  int num_seqs, num_q_heads, num_kv_heads, n_rep, n_hg;
  float scale_log2;
  int part_tokens, max_parts;
  int n_ups;          // units per sequence: num_kv_heads * n_hg (planned schedule)
  int32_t* counters;  // [seq][kv_head][head group], zero at rest
  float* ws_o;        // [seq][q_head][part][D]
  float* ws_ml;       // [seq][q_head][part][2]
  int32_t* err;
  // 8-bit caches: (K, V) scales [kv_head][block], 16-byte units of a block's codes
  const f32x2* scales;
  uint32_t block16;
  int merge_later;  // the planned call's partial rows are merged by a launch of their own
};

// Per-lane byte offsets of this lane's K pieces and V rows inside a 16-token
// tile, relative to the tile's first row; constant across tiles when the tile
// is one block's contiguous rows, so a tile load is uniform base + offset.
template <int DT, int D>
struct LaneOffsets {
  uint32_t k[KStage<DT, D>::NI];
  uint32_t v[4];
};

template <int DT, int D>
__device__ __forceinline__ LaneOffsets<DT, D> lane_offsets(int lane, int64_t slot_bytes) {
  typedef TileShape<DT, D> Sh;
  LaneOffsets<DT, D> o;
  const int g = lane >> 4, c = lane & 15;
#pragma unroll
  for (int i = 0; i < KStage<DT, D>::NI; ++i)
    o.k[i] = (uint32_t)(kstage_row<DT, D>(i, lane) * slot_bytes + 16 * kstage_chunk<DT, D>(lane));
#pragma unroll
  for (int r = 0; r < 4; ++r) o.v[r] = (uint32_t)((4 * r + g) * slot_bytes + Sh::TILES * c * Sh::EB);
  return o;
}

// A tile of an 8-bit cache as it is loaded: 16 dense rows of D codes for K and for
// V. K: the wavefront's 16-byte pieces in row order; V: head_dim/16 codes of rows
// 4r+g. Half the bytes of a 16-bit tile, so a wavefront keeps twice as many in
// flight for the same queue; the codes become numbers in registers (head_dim/4
// conversions a lane and tile, against some 300 cycles of memory time a tile and CU).
template <int D>
struct CodeTile {
  static constexpr int NI = D / 64;  // K load instructions
  uint32_t k[4 * NI];
  uint32_t v[4][NI];
};

// What a kernel streams: tiles of the dtype itself, or of codes.
template <int DT, int D, bool Q8>
struct CacheFormat {
  typedef Tile<DT, D> Raw;
  typedef LaneOffsets<DT, D> Offsets;
  static constexpr int EB = TileShape<DT, D>::EB;          // bytes of an element
  static constexpr int STAGE = KStage<DT, D>::BYTES;       // LDS bytes of a K tile
  __device__ __forceinline__ static Offsets offsets(int lane, int64_t slot_bytes) {
    return lane_offsets<DT, D>(lane, slot_bytes);
  }
};
template <int DT, int D>
struct CacheFormat<DT, D, true> {
  typedef CodeTile<D> Raw;
  struct Offsets {
    uint32_t k, v;  // of this lane in a tile
  };
  static constexpr int EB = 1;
  static constexpr int STAGE = 16 * D;
  __device__ __forceinline__ static Offsets offsets(int lane, int64_t) {
    return Offsets{(uint32_t)lane * 16u, (uint32_t)lane * (D / 16)};
  }
};

// A query operand in registers; with QF (an fp32 query of a 16-bit pool) first the 16
// elements of a step as they are loaded, x then rest, and after split() two pieces of the
// dtype times the power of two that unit takes back.
template <int DT, int D, bool QF>
struct QueryRegs {
  uint32_t x[TileShape<DT, D>::KDW];
  __device__ __forceinline__ void split() {}
  __device__ __forceinline__ float scaled(float scale) const { return scale; }
};
template <int DT, int D>
struct QueryRegs<DT, D, true> {
  static constexpr int N = TileShape<DT, D>::KDW;
  uint32_t x[N], rest[N];
  float unit;
  // (all lanes of the wavefront: the four lane groups hold a row together)
  __device__ __forceinline__ void split() {
    float v[2 * N], most = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      v[i] = __uint_as_float(i < N ? x[i] : rest[i - N]);
      most = fmaxf(most, fabsf(v[i]));
    }
    const int up = row_shift(wave_max_groups_swap(most));
    unit = pow2(-up);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Pieces p = split2<DT>(v[2 * i] * pow2(up), v[2 * i + 1] * pow2(up));
      x[i] = p.hi;
      rest[i] = p.lo;
    }
  }
  __device__ __forceinline__ float scaled(float scale) const { return scale * unit; }
};

// Issues a code tile's loads; the tile's first row is at tk / tv.
template <int DT, int D>
__device__ __forceinline__ void issue_codes(const uint8_t* tk, const uint8_t* tv,
                                            const typename CacheFormat<DT, D, true>::Offsets& lo, CodeTile<D>& tl) {
#pragma unroll
  for (int i = 0; i < CodeTile<D>::NI; ++i) {
    const u32x4 x = __builtin_nontemporal_load((const u32x4*)(tk + lo.k + 1024 * i));
    tl.k[4 * i + 0] = x[0];
    tl.k[4 * i + 1] = x[1];
    tl.k[4 * i + 2] = x[2];
    tl.k[4 * i + 3] = x[3];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if constexpr (D == 128) {
      const u32x2 x = __builtin_nontemporal_load((const u32x2*)(tv + lo.v + 4 * D * r));
      tl.v[r][0] = x[0];
      tl.v[r][1] = x[1];
    } else {
      tl.v[r][0] = __builtin_nontemporal_load((const uint32_t*)(tv + lo.v + 4 * D * r));
    }
  }
}

// Issues the loads of the tile starting at key t0 and returns a 4-bit mask of
// which of this lane's keys 4r+g (r = 0..3) may be used (the keys whose scores
// and V rows this lane holds, see staged_token). Every load is issued
// unconditionally and nothing else touches memory here: an unusable key (bad
// block id, past the context) reads row 0 of the pool instead and is masked in
// the math, and a bad block id only sets `bad` (reported once after the loop).
// That keeps the hardware wait counts exact, with no load-free or
// extra-memory-op path.
// BS16: `bid` is the tile's wave-uniform block id; otherwise every lane
// resolves its own keys through the block table.
template <int DT, int D, bool BS16>
__device__ __forceinline__ uint32_t load_tile(const DecodeArgs& a, const int32_t* bt_row, int32_t bid,
                                              const uint8_t* kc, const uint8_t* vc, const LaneOffsets<DT, D>& lo,
                                              int t0, int t_end, int lane, Tile<DT, D>& tl, bool& bad) {
  typedef TileShape<DT, D> Sh;
  const int g = lane >> 4, c = lane & 15;
  const int64_t slot_bytes = a.c_slot * Sh::EB;
  if constexpr (BS16) {
    // The whole tile lies in one block, and every row of a block is inside the
    // pool even past the context end. The tile base is wave-uniform.
    const int blk = t0 / a.bs;
    const bool ok = bid >= 0 && (int64_t)bid < a.num_blocks;
    bad |= !ok;
    const int64_t base = ok ? (int64_t)bid * a.bs + (t0 - blk * a.bs) : 0;
    const uint8_t* tk = kc + base * slot_bytes;
    const uint8_t* tv = vc + base * slot_bytes;
#pragma unroll
    for (int i = 0; i < KStage<DT, D>::NI; ++i) {
      const u32x4 x = __builtin_nontemporal_load((const u32x4*)(tk + lo.k[i]));
      tl.k[4 * i + 0] = x[0];
      tl.k[4 * i + 1] = x[1];
      tl.k[4 * i + 2] = x[2];
      tl.k[4 * i + 3] = x[3];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) load_dwords_nt<Sh::VDW, true>(tv + lo.v[r], tl.v[r]);
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) m |= (ok && t0 + 4 * r + g < t_end) ? (1u << r) : 0u;
    return m;
  } else {
    kstage_load<DT, D, true>(
        [&](int t) {
          const int tk = t0 + t;
          const int64_t ks = tk < t_end ? token_slot_or_neg(bt_row, tk, a.bs, a.num_blocks) : 0;
          bad |= ks < 0;
          return kc + (ks >= 0 ? ks : 0) * slot_bytes;
        },
        lane, tl.k);
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int tv = t0 + 4 * r + g;
      const int64_t vs = tv < t_end ? token_slot_or_neg(bt_row, tv, a.bs, a.num_blocks) : -1;
      load_v_nt<DT, D, true>(vc + (vs >= 0 ? vs : 0) * slot_bytes, c, tl.v[r]);
      m |= vs >= 0 ? (1u << r) : 0u;
    }
    return m;
  }
}

// kmask: which of this lane's keys 4r+g are usable; a tile whose keys are
// all usable in every lane takes the unmasked path. col_on: whether this
// lane's query column attends the tile at all (a unit shared by two sequences
// runs each one's private tiles with the other's columns off). An off column
// gets -inf scores, so zero probabilities; the V rows stay, since a lane's V
// operand serves every column of the PV product.
template <int DT, int D>
__device__ __forceinline__ void compute_tile(const Tile<DT, D>& tl, const uint32_t (&qr)[TileShape<DT, D>::KDW],
                                             uint32_t kmask, float scale_log2, uint8_t* kst, int lane, State<D>& st,
                                             bool col_on = true) {
  uint32_t kop[TileShape<DT, D>::KDW];
  kstage_transpose<DT, D>(kst, lane, tl.k, kop);
  const f32x4 s = qk_tile<DT, D>(kop, qr);
  float sv[4];
  bool vok[4];
  if (__all(kmask == 0xfu)) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vok[r] = true;
      sv[r] = col_on ? s[r] * scale_log2 : kNegInf;
    }
    softmax_pv<DT, D, true>(sv, tl.v, vok, st);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vok[r] = (kmask >> r) & 1u;
      sv[r] = vok[r] && col_on ? s[r] * scale_log2 : kNegInf;
    }
    softmax_pv<DT, D, false>(sv, tl.v, vok, st);
  }
}

// The same for a tile of codes. The K codes go through LDS as they are and turn into
// the operand there: lane group g of step j holds elements 64 j + 16 g .. + 15 of its
// key (load_query_codes: the same of the query), one 16-byte read each. They are used
// without their scale, which multiplies the score beside scale_log2 (scale * log2 e); the
// V codes are multiplied by theirs, both exact.
//
// QF: a 16-bit pool's query is fp32 and held in two pieces of the dtype, its rounded value and
// that of what it leaves, off by 2^-18 of an element (f16: 2^-24, or 2^-39 of the row's
// largest where the pieces are subnormal) instead of 2^-9 (2^-12).
template <int DT, int D, bool QF>
__device__ __forceinline__ void compute_codes(const CodeTile<D>& tl, const QueryRegs<DT, D, QF>& q, uint32_t kmask,
                                              float scale_log2, float k_scale, float v_scale, uint8_t* kst, int lane,
                                              State<D>& st, bool col_on = true) {
  typedef TileShape<DT, D> Sh;
  constexpr int CPR = D / 16;  // 16-byte chunks per row
  const float score_scale = q.scaled(scale_log2) * k_scale;
  const int g = lane >> 4, t = staged_token(lane & 15);
#pragma unroll
  for (int i = 0; i < CodeTile<D>::NI; ++i) {
    const int row = (64 * i + lane) / CPR, ch = lane % CPR;
    *(u32x4*)(kst + row * D + 16 * (ch ^ (row % CPR))) =
        u32x4{tl.k[4 * i], tl.k[4 * i + 1], tl.k[4 * i + 2], tl.k[4 * i + 3]};
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  uint32_t kop[Sh::KDW];
#pragma unroll
  for (int j = 0; j < CodeTile<D>::NI; ++j) {
    const u32x4 x = *(const u32x4*)(kst + t * D + 16 * ((4 * j + g) ^ (t % CPR)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (Sh::k16) {
        kop[8 * j + 2 * i] = decode2<DT, false>(x[i], 1.f);
        kop[8 * j + 2 * i + 1] = decode2<DT, true>(x[i], 1.f);
      } else {
        const f32x2 lo = decode2_f32<false>(x[i], 1.f), hi = decode2_f32<true>(x[i], 1.f);
        kop[16 * j + 4 * i] = __float_as_uint(lo[0]);
        kop[16 * j + 4 * i + 1] = __float_as_uint(lo[1]);
        kop[16 * j + 4 * i + 2] = __float_as_uint(hi[0]);
        kop[16 * j + 4 * i + 3] = __float_as_uint(hi[1]);
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  f32x4 s = qk_tile<DT, D>(kop, q.x);
  if constexpr (QF) s += qk_tile<DT, D>(kop, q.rest);
  uint32_t v[4][Sh::VDW];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < CodeTile<D>::NI; ++i) {
      if constexpr (Sh::k16) {
        v[r][2 * i] = decode2<DT, false>(tl.v[r][i], v_scale);
        v[r][2 * i + 1] = decode2<DT, true>(tl.v[r][i], v_scale);
      } else {
        const f32x2 lo = decode2_f32<false>(tl.v[r][i], v_scale), hi = decode2_f32<true>(tl.v[r][i], v_scale);
        v[r][4 * i] = __float_as_uint(lo[0]);
        v[r][4 * i + 1] = __float_as_uint(lo[1]);
        v[r][4 * i + 2] = __float_as_uint(hi[0]);
        v[r][4 * i + 3] = __float_as_uint(hi[1]);
      }
    }
  float sv[4];
  bool vok[4];
  if (__all(kmask == 0xfu)) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vok[r] = true;
      sv[r] = col_on ? s[r] * score_scale : kNegInf;
    }
    softmax_pv<DT, D, true, true>(sv, v, vok, st);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vok[r] = (kmask >> r) & 1u;
      sv[r] = vok[r] && col_on ? s[r] * score_scale : kNegInf;
    }
    softmax_pv<DT, D, false, true>(sv, v, vok, st);
  }
}

// Context length of `seq`, clamped to what its block table can hold (flagged).
__device__ __forceinline__ int clamp_ctx(const DecodeArgs& a, int seq, bool report) {
  int ctx = a.ctx[seq];
  const int cap = a.max_blocks * a.bs;
  if (ctx < 0 || ctx > cap) {
    if (report) flag_error(a.err, IR_ERR_CONTEXT_RANGE);
    ctx = ctx < 0 ? 0 : cap;
  }
  return ctx;
}

// Accumulates this wavefront's share of the unit's tiles [tile_lo, tile_hi)
// (wavefront w takes tiles tile_lo + w, tile_lo + w + NW, ...) into st. Keys
// at or past t_end are masked. Runs of up to NW * kMaxWaveTiles tiles: each
// run fetches its block ids once, one per lane.
template <int DT, int D, bool BS16, int NW, int DEPTH, bool Q8, bool QF>
__device__ __forceinline__ void attend_tiles(const DecodeArgs& a, const int32_t* bt_row, const uint8_t* kc,
                                             const uint8_t* vc, const f32x2* scales,
                                             const typename CacheFormat<DT, D, Q8>::Offsets& lo,
                                             const QueryRegs<DT, D, QF>& qr, int tile_lo, int tile_hi, int t_end,
                                             uint8_t* kst, int lane, int w, State<D>& st, bool& bad) {
  static_assert(BS16 || !Q8, "a block of codes holds whole tiles");
  typedef typename CacheFormat<DT, D, Q8>::Raw Raw;
  constexpr int RUN = NW * kMaxWaveTiles;
  for (int r0 = tile_lo; r0 < tile_hi; r0 += RUN) {
    const int ntiles = min(tile_hi - r0, RUN);
    const int my_tiles = ntiles > w ? (ntiles - w + NW - 1) / NW : 0;
    if (my_tiles <= 0) break;
    const int t_begin = 16 * r0;
    int32_t bid_lane = 0;
    if constexpr (BS16) {
      if (lane < my_tiles) bid_lane = bt_row[(t_begin + 16 * (w + NW * lane)) / a.bs];
    }
    f32x2 sc = {0.f, 0.f};  // scales of this lane's tile
    if constexpr (Q8) {
      if (lane < my_tiles && bid_lane >= 0 && (int64_t)bid_lane < a.num_blocks) sc = scales[bid_lane];
    }
    auto issue = [&](int i, Raw& tl) -> uint32_t {
      const int32_t bid = BS16 ? __builtin_amdgcn_readlane(bid_lane, i) : 0;
      if constexpr (Q8) {
        const int g = lane >> 4, t0 = t_begin + 16 * (w + NW * i), blk = t0 / a.bs;
        const bool ok = bid >= 0 && (int64_t)bid < a.num_blocks;
        bad |= !ok;
        const int64_t at = ok ? ((int64_t)bid * a.bs + (t0 - blk * a.bs)) * D : 0;
        issue_codes<DT, D>(kc + at, vc + at, lo, tl);
        uint32_t m = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) m |= (ok && t0 + 4 * r + g < t_end) ? (1u << r) : 0u;
        return m;
      } else
        return load_tile<DT, D, BS16>(a, bt_row, bid, kc, vc, lo, t_begin + 16 * (w + NW * i), t_end, lane, tl, bad);
    };
    // Register ring of DEPTH tiles: while one tile is in the math, the next
    // DEPTH-1 tiles' loads are in flight.
    const int last = my_tiles - 1;
    Raw ring[DEPTH];
    uint32_t mk[DEPTH];
    auto compute = [&](const Raw& tl, int i, uint32_t mask) {
      if constexpr (Q8) {
        const int ii = min(i, last);
        const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc[0]), ii));
        const float vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc[1]), ii));
        compute_codes<DT, D, QF>(tl, qr, mask, a.scale_log2, ks, vs, kst, lane, st);
      } else
        compute_tile<DT, D>(tl, qr.x, mask, a.scale_log2, kst, lane, st);
    };
#pragma unroll
    for (int r = 0; r < DEPTH; ++r) mk[r] = issue(min(r, last), ring[r]);
    int i = 0;
    // Steady state: every issue is a real tile, so the body is straight-line
    // and the loads' wait counts are exact (a conditional issue here makes the
    // compiler drain the ring every tile: 59 -> 67 us on 64 sequences).
    for (; i + 2 * DEPTH <= my_tiles; i += DEPTH) {
#pragma unroll
      for (int r = 0; r < DEPTH; ++r) {
        compute(ring[r], i + r, mk[r]);
        mk[r] = issue(i + r + DEPTH, ring[r]);
      }
    }
    // The last tiles: nothing is issued past the end (the merge after the loop
    // reuses the ring's registers and would wait for such loads); a slot past
    // the end is computed with an empty key mask, which changes nothing.
    for (; i < my_tiles; i += DEPTH) {
#pragma unroll
      for (int r = 0; r < DEPTH; ++r) {
        compute(ring[r], i + r, i + r < my_tiles ? mk[r] : 0u);
        if (i + r + DEPTH <= last) mk[r] = issue(i + r + DEPTH, ring[r]);
      }
    }
  }
}

// Q^T operand of (seq, query head qh), same k-slot assignment as the K loads;
// padded heads are zero.
template <int DT, int D>
__device__ __forceinline__ void load_query(const DecodeArgs& a, int seq, int qh, bool head_ok, int g,
                                           uint32_t (&qr)[TileShape<DT, D>::KDW]) {
  if (head_ok)
    load_k<DT, D>((const uint8_t*)a.q + ((int64_t)seq * a.q_seq + (int64_t)qh * a.q_head) * TileShape<DT, D>::EB, g,
                  qr);
  else
    zero_dwords(qr);
}

// The query operand that goes with code tiles (compute_codes), before its split().
template <int DT, int D, bool QF>
__device__ __forceinline__ void load_query_codes(const DecodeArgs& a, int seq, int qh, bool head_ok, int g,
                                                 QueryRegs<DT, D, QF>& q) {
  typedef TileShape<DT, D> Sh;
  constexpr int EB = QF ? 4 : Sh::EB;
  constexpr int DW = 4 * EB;  // dwords of 16 elements
  const uint8_t* row = (const uint8_t*)a.q + ((int64_t)seq * a.q_seq + (int64_t)qh * a.q_head + 16 * g) * EB;
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int i = 0; i < DW; i += 4) {
      const u32x4 x = head_ok ? *(const u32x4*)(row + 64 * j * EB + 4 * i) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = DW * j + i + e;
        if constexpr (QF) {
          if (at >= Sh::KDW) q.rest[at - Sh::KDW] = x[e];
          else q.x[at] = x[e];
        } else {
          q.x[at] = x[e];
        }
      }
    }
}

template <int DT, int D, bool Q8, bool QF>
__device__ __forceinline__ void load_query_for(const DecodeArgs& a, int seq, int qh, bool head_ok, int g,
                                               QueryRegs<DT, D, QF>& q) {
  static_assert(Q8 || !QF, "16-bit caches take queries of their dtype");
  if constexpr (Q8) load_query_codes<DT, D>(a, seq, qh, head_ok, g, q);
  else load_query<DT, D>(a, seq, qh, head_ok, g, q.x);
}

// Writes the workgroup's merged (normalised) result for heads head0..head0+nh.
template <int DT, int D, int NW>
__device__ __forceinline__ void store_merged(const DecodeArgs& a, const MergeSmem<NW, D>& sm, int seq, int head0,
                                             int nh) {
  constexpr int EB = TileShape<DT, D>::EB;
  for (int it = threadIdx.x; it < nh * (D / 4); it += NW * 64) {
    const int hc = it / (D / 4);
    const int d0 = (it - hc * (D / 4)) * 4;
    float M, L, o[4];
    merge_column<NW, D>(sm, hc, d0, M, L, o);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    store4<DT>((uint8_t*)a.out + ((int64_t)seq * a.o_seq + (int64_t)(head0 + hc) * a.o_head + d0) * EB, o, inv);
  }
}

// Log-sum-exp merge of n partial rows (acc at o[k * o_step], (max, sum) at
// ml[k * ml_step]) for 4 outputs d0..d0+3; `ld` reads one fp32.
template <typename Ld>
__device__ __forceinline__ void lse_merge(const float* o, int64_t o_step, const float* ml, int64_t ml_step, int n,
                                          Ld ld, float (&acc)[4], float& L) {
  float M = kNegInf;
  for (int p = 0; p < n; ++p) M = fmaxf(M, ld(ml + p * ml_step));
  L = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[k] = 0.f;
  for (int p = 0; p < n; ++p) {
    const float mp = ld(ml + p * ml_step);
    const float lp = ld(ml + p * ml_step + 1);
    const float wt = mp == kNegInf ? 0.f : fast_exp2(mp - M);
    L += wt * lp;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += wt * ld(o + p * o_step + k);
  }
}

}  // namespace ir
