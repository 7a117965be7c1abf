// The kernel of the row-wise calls whose keys and values go to a 4-bit pool, or whose
// angles come from positions with several axes: one pass over the step's rows, the row
// mathematics norm_rope.hpp's.
//
// A wavefront takes one token and 64 / (head_dim / 16) of its rows (q, then k, then v) at
// a time, its lanes holding their part of the token's angles in registers for all of
// them. Bound by memory: every row is read once and written once (4,096 tokens of 28 + 2 x 4 rows
// of 128 in bf16, rotated by axes into a 16-bit pool: 14.0 us, 5.4 TB/s; 64 tokens, normed too, 3.3 us,
// the launch and two trips).
#pragma once

#include <algorithm>

#include "e2m1.hpp"
#include "norm_rope.hpp"

namespace ir {

enum { kAnglesNone = 0, kAnglesTables = 1, kAnglesPositions = 2 };
enum { kToRows = 0, kToCache = 1, kToCodes4 = 2 };  // where keys go; values go with them, or nowhere

constexpr int kMaxPairs = 128;  // of a head
constexpr int kTurnWaves = 4;  // of a workgroup, a token each
// Of rows given the same slot of a 4-bit pool the last is written (a mixture of two would have one's codes
// at the other's scales). In a launch of up to kWaveScan tokens each wavefront reads the slots behind its
// own (1,024 tokens of 4 heads of 128: 0.7 us of 3.7); in a longer one a workgroup, of kScanWaves, reads those
// behind all its tokens' (find_later; 4,096 tokens: 0.9 us of 5.1, 8,192: 1.7 of 7.4; 2,048 take 4.7 us either
// way, 1,216 4.1 and 4.5, 3,000 6.3 and 4.8). That is n^2 / 4 bytes in all, so a call of more than kScanTokens
// is several launches, in order (65,536 tokens in bf16: 60 us, 66 in launches of 8,192 and 67 of 32,768).
constexpr int kWaveScan = 2048, kScanWaves = 16, kScanTokens = 16384;

struct TurnArgs {
  RowArgs r;
  // kAnglesPositions
  const int64_t* pos;
  int64_t pos_axis;
  int num_axes;
  const ir_rotary_pair* pairs;
  float scaling;
  int head_dim;
  // kToRows, bytes
  uint8_t* ko;
  int64_t ko_tok, ko_head;
  // kToCache (bytes), kToCodes4 (dense)
  uint8_t* kc;
  uint8_t* vc;
  int64_t c_slot, c_head;
  uint8_t* scales;
  int64_t num_slots;
  int64_t tok0, tok_end;  // the launch's tokens
  int chunk_rows;         // rows of a wavefront
  int32_t* err;
};

// cos and sin of a token's pairs, one pair a lane, to the wavefront's LDS. position *
// step modulo 2^64 is the angle as a fraction of a turn: the wrap-around is the reduction,
// exact however far the position, and the signed upper half of it (rounded: 2^-33 turns) is half
// a turn at most, as an fp32 number off by 2^-24 of itself.
__device__ __forceinline__ void angles_of(const TurnArgs& a, int64_t tok, int lane, int pairs, float* cs) {
  for (int j = lane; j < pairs; j += 64) {
    const u32x4 p = *(const u32x4*)(a.pairs + j);
    const uint64_t step = ((uint64_t)p[1] << 32) | p[0];
    const int axis = max(0, min((int)p[2], a.num_axes - 1));
    const uint64_t turn = (uint64_t)a.pos[axis * a.pos_axis + tok] * step + 0x80000000u;
    float s, c;
    sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
    cs[j] = c * a.scaling;
    cs[kMaxPairs + j] = s * a.scaling;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Which of the first kScanWaves of n slots, the workgroup's tokens', come again later, a bit each (every thread
// of the workgroup calls). A map of the slots' low bits tells most of the others apart.
__device__ __forceinline__ uint32_t find_later(const int64_t* slots, int n) {
  constexpr int NW = kScanWaves, NT = NW * 64, AHEAD = 4, BITS = 8192;
  static_assert(NW * NW <= NT && BITS / 32 <= NT, "a thread for each pair of tokens and each word of the map");
  __shared__ uint32_t s_map[BITS / 32], s_own[NW], s_later;
  const int tid = threadIdx.x;
  auto key = [](int64_t slot) { return (uint64_t)slot >> 32 ? ~0u : (uint32_t)slot; };  // (a pool's are below 2^31)
  int64_t x[AHEAD];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = slots[min(j0 + tid + NT * i, n - 1)];
  };
  const uint32_t own = key(slots[min(tid, n - 1)]);
  load(NW);
  if (tid < BITS / 32) s_map[tid] = 0;
  if (tid == 0) s_later = 0;
  __syncthreads();
  if (tid < NW) {
    s_own[tid] = own;
    atomicOr(&s_map[own % BITS / 32], 1u << (own % 32));
  }
  __syncthreads();
  if (tid < NW * NW) {
    const int k = tid % NW, m = tid / NW;
    if (k < m && m < n && s_own[k] == s_own[m]) atomicOr(&s_later, 1u << k);
  }
  for (int j0 = NW; j0 < n; j0 += NT * AHEAD) {
    if (j0 > NW) load(j0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (j0 + NT * i >= n) break;
      const uint32_t y = key(x[i]);
      if (s_map[y % BITS / 32] >> (y % 32) & 1u) {
        uint32_t later = 0;
        for (int k = 0; k < NW; ++k) later |= s_own[k] == y ? 1u << k : 0u;
        if (later) atomicOr(&s_later, later);
      }
    }
  }
  __syncthreads();
  return s_later;
}

// D 0: a.head_dim (rows without norms only). NW wavefronts, a token each.
template <int DT, int D, int MODE, int ANG, int DST, int NW>
__global__ __launch_bounds__(NW * 64) void turn_rows_kernel(TurnArgs a) {
  typedef Chunk8<DT> C;
  static_assert(D != 0 || (MODE == kRowsTurn && DST == kToRows), "the head's width is known for norms and pools");
  __shared__ __attribute__((aligned(16))) float s_cs[ANG == kAnglesPositions ? NW : 1][2 * kMaxPairs];
  const int hd = D ? D : a.head_dim, lpr = hd / 16, half = hd / 2 * C::EB;
  const int G = 64 / lpr;  // rows of a wavefront at a time
  const int lane = threadIdx.x & 63, grp = lane / lpr, ci = lane - grp * lpr;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr bool SCAN = NW == kScanWaves;
  static_assert(!SCAN || DST == kToCodes4, "only a 4-bit pool's writes need it");
  const uint32_t block = DST == kToCodes4 && !SCAN && gridDim.y == 1 ? near_block(blockIdx.x) : blockIdx.x;
  const int64_t tok = a.tok0 + (int64_t)block * NW + w;
  const int nq = MODE == kRowsPlain ? 0 : a.r.num_q_heads, nkv = a.r.num_kv_heads;
  const int rows = nq + (DST == kToRows ? nkv : 2 * nkv);
  const int row0 = blockIdx.y * a.chunk_rows;
  const int row_end = min(rows, row0 + a.chunk_rows);
  bool kv_ok = true;
  if constexpr (SCAN) {
    if (row_end > nq) kv_ok = !(find_later(a.r.slots + tok - w, (int)(a.tok_end - tok) + w) >> w & 1u);
  }
  if (tok >= a.tok_end) return;
  int64_t slot = 0;
  if constexpr (DST != kToRows) {
    slot = a.r.slots[tok];
    kv_ok = kv_ok && slot >= 0 && slot < a.num_slots;
    if (slot >= a.num_slots && lane == 0 && row0 == 0) flag_error(a.err, IR_ERR_SLOT_RANGE);
  }
  if constexpr (DST == kToCodes4 && !SCAN) {
    if (row_end > nq) {
      const int64_t* slots = a.r.slots + a.tok0;
      const int n = (int)(a.tok_end - a.tok0);
      bool later = false;
      for (int j = (int)(tok - a.tok0) + 1 + lane; j < n; j += 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) later |= slots[min(j + 64 * i, n - 1)] == slot;
      }
      if (__any(later)) kv_ok = false;
    }
  }
  Angles<DT, D, MODE> t;
  if constexpr (ANG == kAnglesTables) t.load(a.r.cos + tok * a.r.cs_tok, a.r.sin + tok * a.r.cs_tok, ci);
  if constexpr (ANG == kAnglesPositions) {
    angles_of(a, tok, lane, hd / 2, s_cs[w]);
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const f32x4 c = *(const f32x4*)&s_cs[w][8 * ci + e], s = *(const f32x4*)&s_cs[w][kMaxPairs + 8 * ci + e];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t.c[e + i] = t.c[8 + e + i] = c[i];
        t.s[e + i] = t.s[8 + e + i] = s[i];
      }
    }
  }
  typename C::Raw wraw[2][2];  // norm weights of q and k
  if constexpr (MODE == kRowsNorm) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* p = (i ? a.r.k_weight : a.r.q_weight) + ci * 8 * C::EB;
      C::raw_load(p, wraw[i][0]);
      C::raw_load(p + half, wraw[i][1]);
    }
  }
  for (int row = row0 + grp; row < row_end && grp < G; row += G) {
    const bool is_q = MODE != kRowsPlain && row < nq, is_v = row >= nq + nkv;
    const int h = is_q ? row : is_v ? row - nq - nkv : row - nq;
    const uint8_t* src = (is_q   ? a.r.q + tok * a.r.q_tok + h * a.r.q_head
                          : is_v ? a.r.v + tok * a.r.v_tok + h * a.r.v_head
                                 : a.r.k + tok * a.r.k_tok + h * a.r.k_head) +
                         ci * 8 * C::EB;
    typename C::Raw lo, hi;
    C::raw_load(src, lo);
    C::raw_load(src + half, hi);
    if (!is_q && !kv_ok) continue;  // (a row's lanes go together)
    if constexpr (DST == kToCache) {
      if (is_v) {
        uint8_t* dst = a.vc + slot * a.c_slot + h * a.c_head + ci * 8 * C::EB;
        C::raw_store_nt(dst, lo);
        C::raw_store_nt(dst + half, hi);
        continue;
      }
    }
    float x[16], wt[16];
    auto unpack = [](const typename C::Raw& l, const typename C::Raw& u, float(&to)[16]) {
      float p[8], q[8];
      C::unpack(l, p);
      C::unpack(u, q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        to[e] = p[e];
        to[8 + e] = q[e];
      }
    };
    unpack(lo, hi, x);
    if constexpr (MODE != kRowsPlain) {
      if (!is_v) {
        if constexpr (MODE == kRowsNorm) unpack(wraw[is_q ? 0 : 1][0], wraw[is_q ? 0 : 1][1], wt);
        transform_row<DT, D, MODE>(x, wt, a.r.eps, t);
      }
    }
    if constexpr (DST == kToCodes4) {
      if (!is_q) {
        const int64_t tile = (int64_t)((uint64_t)(uint32_t)h * (uint32_t)(a.num_slots >> 4)) + (slot >> 4);
        store_row_e2m1<DT, D>(x, (is_v ? a.vc : a.kc) + tile * Tile4<D>::CODES, a.scales + tile * Tile4<D>::SCALES,
                              (int)(slot & 15), ci, is_v);
        continue;
      }
    }
    float x0[8], x1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x0[e] = x[e];
      x1[e] = x[8 + e];
    }
    if (is_q && a.r.qo_wide) {
      typedef Chunk8<IR_DTYPE_F32> W;
      uint8_t* dst = a.r.qo + tok * a.r.qo_tok + h * a.r.qo_head + ci * 32;
      W::store_nt(dst, x0);
      W::store_nt(dst + hd * 2, x1);
      continue;
    }
    uint8_t* dst = (is_q               ? a.r.qo + tok * a.r.qo_tok + h * a.r.qo_head
                    : DST == kToCache ? a.kc + slot * a.c_slot + h * a.c_head
                                      : a.ko + tok * a.ko_tok + h * a.ko_head) +
                   ci * 8 * C::EB;
    C::store_nt(dst, x0);
    C::store_nt(dst + half, x1);
  }
}

// Wavefronts of a token: one for all its rows once the tokens alone fill the device, which
// then have their angles once a token; below that one for each run of rows, so that a
// decode step's few tokens are a single pass (qk_norm_rope.hip has both measured).
constexpr int64_t kTurnTokensForDevice = 2048;

template <int DT, int D, int MODE, int ANG, int DST, int NW>
void launch_tokens(const TurnArgs& a, int runs, hipStream_t s) {
  int64_t blocks = (a.tok_end - a.tok0 + NW - 1) / NW;
  if (DST == kToCodes4 && NW == kTurnWaves && runs == 1) blocks = near_blocks(blocks);
  hipLaunchKernelGGL((turn_rows_kernel<DT, D, MODE, ANG, DST, NW>), dim3((unsigned)blocks, runs), dim3(NW * 64), 0, s,
                     a);
}

template <int DT, int D, int MODE, int ANG, int DST>
int launch_turn(const char* name, TurnArgs a, hipStream_t s) {
  const int rows = a.r.num_q_heads + (DST == kToRows ? 1 : 2) * a.r.num_kv_heads;
  if (rows == 0) return ok();
  const int g = 64 / ((D ? D : a.head_dim) / 16);
  const int runs = a.r.n_tokens >= kTurnTokensForDevice ? 1 : (rows + g - 1) / g;
  a.chunk_rows = runs == 1 ? rows : g;
  IR_REQUIRE(a.r.n_tokens <= 0x7fffffff, "%s: too many tokens", name);
  IR_REQUIRE(runs <= 65535, "%s: too many heads", name);
  const int64_t step = DST == kToCodes4 ? kScanTokens : a.r.n_tokens;
  for (a.tok0 = 0; a.tok0 < a.r.n_tokens; a.tok0 = a.tok_end) {
    a.tok_end = std::min(a.tok0 + step, a.r.n_tokens);
    if (DST == kToCodes4 && a.tok_end - a.tok0 > kWaveScan)
      launch_tokens<DT, D, MODE, ANG, DST, DST == kToCodes4 ? kScanWaves : kTurnWaves>(a, runs, s);
    else
      launch_tokens<DT, D, MODE, ANG, DST, kTurnWaves>(a, runs, s);
  }
  return check_launch(name);
}

}  // namespace ir
