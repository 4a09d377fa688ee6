// bf16 flash attention for sm_100a in which token i sees the keys [lo_i, hi_i): packed requests (documents), a prefix
// with causal or frame-causal tokens behind it, windows.  QK^T and PV are tcgen05 kind::f16 MMAs with S, P and O in
// TMEM; Q, K and V are read by TMA straight from the caller's rows, and key heads may be shared by groups of query heads.
// No counterpart in the reference, whose backends attend to the whole sequence (tfvideo/attention.py:29-54).
//
// o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(q_i k_j / sqrt(128) - m_i), one pass over the keys with the running
// maximum m and sum l in 32 bits.  A row without keys gives zeros.  P is rounded to bf16 for the PV MMA (both operands
// of that MMA have one type, V's); l sums the unrounded P.
//
// A unit of work = two 128-row query tiles (A, B) of one head over the same 128-key steps.  TMEM: S_A, S_B, O_A, O_B of
// 128 columns each, P written over S.  Warps 0-3: softmax of A, 4-7: of B, a thread per query row; warp 8: TMA and the
// next unit; warps 9 and 10: the MMAs of A and of B; warp 11: guards masked V rows (below).  One tile's MMAs run under
// the other's softmax.  A CTA takes units from a counter, so that a unit's loads and its first S run under the end of
// the one before (a CTA for each unit: 8 us of start and end, 162 us against 145 for packed clips of 1 to 2,019 tokens,
// 40 heads, 4.6 units an SM).
//
// A step of both tiles is 4 x 512 cycles of MMA at the bf16 rate, and measures 2,570: S to P takes 1,490, P to the next S
// 1,070 (PV of 64 keys, QK, and 300 of waiting and issuing), which is as long as two turns of the tensor core with
// their 250 cycles of changing hands.  Exponentials are 2 x 1,024 cycles at 16 a cycle, 5 pairs in 16 on the FMA pipe
// instead.  Measured beside this: 16 softmax warps, two threads a row (147 us for those clips: the same chunk takes
// 270 cycles a warp with two warps as 316 with one); one warp for both tiles' MMAs (150 us); P handed over whole (147),
// by quarters (147) or three quarters first (168).  At 37,760 tokens in two requests, 40 heads: 12.1 ms, 1.21 PFLOP/s,
// with the SM clock held at 1.5-1.6 GHz by the power limit (a plain bf16 GEMM sustains 1.39 under it).
//
// All of this is of rows whose scores are bounded (kBoundBf16): q and k of unit variance, |q| |k| about 128.  With
// |q| |k| about 512 every row keeps a running maximum, reads its scores twice and takes no polynomial: 14.7 ms for the two
// requests and 183 us for the clips (143 bounded, in the same run).
//
// Masked keys.  Steps run over the union of the unit's spans and start at its first key, so documents begin on a step.
// Scores of masked keys become -inf before the maximum, whatever K holds there.  V needs more: 0 x NaN is NaN inside
// the MMA, and another request's rows or the memory behind the last one may hold anything.  In a step that hides some
// key from some row, warp 11 sets non-finite elements of the V tile to zero and notes the step; the epilogue adds
// them back, from global memory, to the rows that do see them.
#pragma once

#include <climits>
#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "h3b200.h"

namespace h3 {

// warp-wide: one tile of a 3-D tensor map into shared memory, completing on `bar`
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 rx;\n\t" H3_ELECT
      "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];\n\t}" ::"r"(smem_u32(smem_dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// warp-wide: D[tmem] (+)= A[smem] x B[smem], bf16 x bf16 -> fp32
__device__ __forceinline__ void mma_bf16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 rx;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t" H3_ELECT
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// warp-wide: A from TMEM (lane = row, two consecutive K elements a column)
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 rx;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t" H3_ELECT
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Waits until a barrier's phase completes whether or not another wait of the grid gave up, for at most the same limit:
// copies and MMAs in flight end before a CTA gives back its memory.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity, int code) {
  if (mbar_try_wait(bar, parity)) return;
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait_suspend(bar, parity, kSuspendNs))
    if (globaltimer() - t0 > kWaitLimitNs) {
      set_status(code);
      return;
    }
}
// kind::f16 with bf16 operands and an fp32 accumulator: C format F32 = 1 in bits 4-5, A / B format BF16 = 1 in bits
// 7-9 / 10-12, bit 16 = B is MN-major (its N elements contiguous in shared memory).
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// warp-wide store of one box of a 3-D tensor map from shared memory (the part outside the tensor is not written)
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* smem_src, int x, int y, int z) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 rx;\n\t" H3_ELECT
      "@e cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n\t}" ::"l"(map), "r"(x),
      "r"(y), "r"(z), "r"(smem_u32(smem_src))
      : "memory");
}
// warp-wide: the elected lane's stores so far become a group; all but its last N groups have read their shared memory
__device__ __forceinline__ void tma_store_commit() {
  asm volatile("{\n\t.reg .pred e;\n\t.reg .b32 rx;\n\t" H3_ELECT "@e cp.async.bulk.commit_group;\n\t}" ::: "memory");
}
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("{\n\t.reg .pred e;\n\t.reg .b32 rx;\n\t" H3_ELECT "@e cp.async.bulk.wait_group.read %0;\n\t}" ::"n"(N)
               : "memory");
}

struct AttnBf16Args {
  const __nv_bfloat16* v;    // element (t, h, d) at v + t * ldv + h * hsv + d (the epilogue's repair of masked steps)
  long long ldv, hsv;
  const int* lo;             // spans, or NULL: every key
  const int* hi;
  const float* knorm;        // [key heads][S / 128 tiles]: largest |k|^2 of each 128 keys, or NULL
  const float* knorm1;       // [key heads][S]: of each key
  const int* order;          // [S / 256 tiles]: query tiles by falling number of key steps, or NULL
  int S, group;              // group: query heads that share a key head
  int* next;                 // units handed out beyond each CTA's first, or NULL: a CTA for every unit
  int rows;                  // query rows a unit: 256, or 128 (tile B unused) when that many CTAs still fit at once
  int tiles, heads;          // units: query tiles of that many rows x query heads
  int tile_major;            // units in order of tiles (every head of one, then the next), else of heads
};

// What one CTA works on at a time: two query tiles of one head.  Step j covers keys base + 128 j ..; tile t takes part
// in steps [j0[t], j1[t]).
struct AttnBf16Unit {
  int q0;                        // first query row; -1: no more units
  int h, base, steps;
  int j0[2], j1[2];
  int lo_max[2], hi_min[2];      // over the tile's rows that have keys
  float kk;                      // largest |k|^2 of the unit's keys
};

struct AttnBf16Smem {
  static constexpr int SUB = 128 * 128;            // 128 rows x 64 dims of bf16 (128-byte rows, 128-byte swizzle)
  static constexpr int TILE = 2 * SUB;             // 128 rows x 128 dims
  static constexpr int KST = 2, VST = 2;           // ring depths (a third V tile measured the same)
  static constexpr int STAGE = 32 * 128;           // output on its way: 32 rows x 64 dims a softmax warp
  static constexpr int Q_OFF = 0;                  // tiles A, B
  static constexpr int K_OFF = 2 * TILE;
  static constexpr int V_OFF = K_OFF + KST * TILE;
  static constexpr int STAGE_OFF = V_OFF + VST * TILE;
  static constexpr int BAR_OFF = STAGE_OFF + 8 * STAGE;
  static constexpr int MAX_S = 262144;
  static constexpr int BAD_WORDS = MAX_S / 128 / 32 + 1;   // a bit per step whose V tile held masked non-finite values
  static constexpr int BAD_OFF = BAR_OFF + 256;            // of two units
  static constexpr int UNIT_OFF = BAD_OFF + (2 * BAD_WORDS + 3) / 4 * 16;
  static constexpr int TOTAL = UNIT_OFF + 2 * (int)sizeof(AttnBf16Unit) + 16 + 1024;
};
static_assert(AttnBf16Smem::TOTAL <= 232448, "shared memory of one SM");

constexpr int kAttnBf16Threads = 384;
// Lag of the running maximum (log2 units) before O and l are rescaled: P <= 2^8 is far inside bf16's range, and its
// relative rounding does not depend on the factor.
constexpr float kTauBf16 = 8.0f;
// Scores are bounded by |q| |k|; while twice that bound is below this (log2 units), a row keeps the maximum of its
// first step for good: P and l then stay below 2^98 (and O below fp32's range for values to 2^29), and no later step
// looks for a maximum: 11.2-11.9 ms against 14.7 at the size above, in one run.
constexpr float kBoundBf16 = 80.0f;
// pairs of each 32-key chunk whose exp2 runs on the FMA pipe (bit i: keys 2i, 2i + 1)
constexpr uint32_t kPolyPairsBf16 = 0x2492u;

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN when either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

// 2^x for a pair whose results are normal numbers: exp2_poly_pair's polynomial, without its clamp, and the exponent
// raised by an integer addition.
__device__ __forceinline__ uint64_t exp2_poly_normal(uint64_t x) {
  constexpr float kMagic = 12582912.0f;                                     // 1.5 * 2^23: the sum's low bits are round(x)
  const uint64_t t = add2(x, f32x2_splat(kMagic));
  const uint64_t g = fma2(add2(t, f32x2_splat(-kMagic)), f32x2_splat(-1.0f), x);
  uint64_t p = fma2(f32x2_splat(0.0551716685295105f), g, f32x2_splat(0.2426111400127411f));
  p = fma2(p, g, f32x2_splat(0.6932609677314758f));
  p = fma2(p, g, f32x2_splat(0.9999280571937561f));
  float t0, t1, p0, p1;
  f32x2_unpack(t, t0, t1);
  f32x2_unpack(p, p0, p1);
  return f32x2_pack(__uint_as_float((__float_as_uint(t0) << 23) + __float_as_uint(p0)),
                    __uint_as_float((__float_as_uint(t1) << 23) + __float_as_uint(p1)));
}

// 32 scores of one row -> 16 words of bf16 P = exp2(s * scale - m) (key 2w in the low half of word w); l2 += the
// unrounded P.  POLY (bounded scores, none masked): part of the exponentials as a polynomial; otherwise all on the
// MUFU, whose exp2(-inf) is exactly 0 and exp2(NaN) NaN.
template <bool POLY>
__device__ __forceinline__ void p_chunk_bf16(const uint32_t (&s)[32], uint64_t scale2, float nm, uint32_t (&pw)[16],
                                             uint64_t& l2a, uint64_t& l2b) {
  const uint64_t nm2 = f32x2_splat(nm);
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const uint64_t x = fma2(f32x2_pack(__uint_as_float(s[2 * w]), __uint_as_float(s[2 * w + 1])), scale2, nm2);
    const uint64_t y = POLY && ((kPolyPairsBf16 >> w) & 1u) ? exp2_poly_normal(x) : exp2_mufu_pair(x);
    if (w & 1) l2b = add2(l2b, y);
    else l2a = add2(l2a, y);
    float a, b;
    f32x2_unpack(y, a, b);
    pw[w] = pack_bf16(a, b);
  }
}

// Before the attention, for long sequences: |k|^2 of each key and head, the largest of each 128 (NaN when one is), and the
// span range of each 128 query rows.  Bound by reading K once: 16 lanes a row.
struct AttnBf16Prep {
  const __nv_bfloat16* k;
  long long ld, hs;
  int S;
  const int *lo, *hi;
  float *knorm, *knorm1;
  int2* range;         // [S / 128 tiles]: first and end key of the tile's rows
  int* order;
  int* next;           // to zero
};
__global__ void __launch_bounds__(256) attn_bf16_prep_kernel(const AttnBf16Prep a) {
  __shared__ float red[16];
  __shared__ int2 rr[4];
  const int part = threadIdx.x & 15, row0 = threadIdx.x >> 4;
  launch_dependents();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.next = 0;
  uint4 u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = blockIdx.x * 128 + row0 + 16 * i;
    u[i] = make_uint4(0u, 0u, 0u, 0u);
    if (t < a.S) u[i] = *reinterpret_cast<const uint4*>(a.k + (long long)t * a.ld + blockIdx.y * a.hs + part * 8);
  }
  const bool spans = a.lo && blockIdx.y == 0;
  if (spans && threadIdx.x < 128) {
    const int t = blockIdx.x * 128 + threadIdx.x;
    int lo = t < a.S ? max(a.lo[t], 0) : 0, hi = t < a.S ? min(a.hi[t], a.S) : 0;
    const bool live = lo < hi;
    lo = __reduce_min_sync(~0u, live ? lo : INT_MAX);
    hi = __reduce_max_sync(~0u, live ? hi : 0);
    if ((threadIdx.x & 31) == 0) rr[threadIdx.x >> 5] = make_int2(lo, hi);
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += bf16_lo(w[e]) * bf16_lo(w[e]) + bf16_hi(w[e]) * bf16_hi(w[e]);
#pragma unroll
    for (int o = 8; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    m = max_nan(m, ss);
    const int t = blockIdx.x * 128 + row0 + 16 * i;
    if (part == 0 && t < a.S) a.knorm1[(size_t)blockIdx.y * a.S + t] = ss;
  }
  if (part == 0) red[row0] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max_nan(m, red[i]);
    a.knorm[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = m;
    if (spans)
      a.range[blockIdx.x] = make_int2(min(min(rr[0].x, rr[1].x), min(rr[2].x, rr[3].x)),
                                      max(max(rr[0].y, rr[1].y), max(rr[2].y, rr[3].y)));
  }
}
// The 256-row query tiles (at most 1,024) by falling number of key steps: the longest units start first, so that the
// last ones to start are short.  One block; each thread ranks its tile against all.
__global__ void __launch_bounds__(1024) attn_bf16_order_kernel(const AttnBf16Prep a, int tiles) {
  __shared__ int w[1024];
  const int t = threadIdx.x, n128 = (a.S + 127) >> 7;
  launch_dependents();
  wait_primary();
  int mine = 0;
  if (t < tiles) {
    const int2 x = a.range[2 * t], y = 2 * t + 1 < n128 ? a.range[2 * t + 1] : make_int2(INT_MAX, 0);
    const int lo = min(x.x, y.x), hi = max(x.y, y.y);
    mine = hi > lo ? (hi - lo + 127) >> 7 : 0;
  }
  w[t] = mine;
  __syncthreads();
  if (t >= tiles) return;
  int rank = 0;
  for (int i = 0; i < tiles; ++i) rank += w[i] > mine || (w[i] == mine && i < t);
  a.order[rank] = t;
}

__global__ void __launch_bounds__(kAttnBf16Threads, 1)
    attn_bf16_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                     const AttnBf16Args p) {
  using L = AttnBf16Smem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;            // both tiles' S issued for good, and every softmax warp past its look at Q
  uint64_t* k_full = q_empty + 1;          // [KST]
  uint64_t* k_empty = k_full + L::KST;
  uint64_t* v_full = k_empty + L::KST;     // [VST]
  uint64_t* v_ok = v_full + L::VST;        // [VST]: landed, and its masked non-finite values are zero
  uint64_t* v_empty = v_ok + L::VST;
  uint64_t* s_full = v_empty + L::VST;     // [tile]
  uint64_t* p_full = s_full + 2;           // [tile][half]: P of keys 0-63 / 64-127 written, by four warps
  uint64_t* o_done = p_full + 4;           // [tile]: the unit's last PV
  uint64_t* o_free = o_done + 2;           // [tile]: O is in registers
  uint64_t* turn = o_free + 2;             // [tile]: the other tile's MMAs of this round are issued
  uint64_t* guard_done = turn + 2;         // [unit]: the V guard has seen all of it
  uint64_t* unit_full = guard_done + 2;    // [unit]
  uint64_t* unit_empty = unit_full + 2;
  uint64_t* drained = unit_empty + 2;
  uint32_t* bad = reinterpret_cast<uint32_t*>(smem + L::BAD_OFF);            // [unit][BAD_WORDS]
  AttnBf16Unit* units = reinterpret_cast<AttnBf16Unit*>(smem + L::UNIT_OFF);   // [2]
  int* any_bad = reinterpret_cast<int*>(units + 2);                          // [unit]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(any_bad + 2);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  auto load = [&](int off, const CUtensorMap* map, int row, int head, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, L::TILE);
    tma_load_3d(smem + off, map, 0, row, head, bar);
    tma_load_3d(smem + off + L::SUB, map, 64, row, head, bar);
  };
  // (TMA warp) K and V tiles asked for, over all units
  int nk = 0, nv = 0;
  auto load_k = [&](int row, int h) {
    load(L::K_OFF + nk % L::KST * L::TILE, &tmK, row, h / p.group, &k_full[nk % L::KST]);
    ++nk;
  };
  auto load_v = [&](int row, int h) {
    load(L::V_OFF + nv % L::VST * L::TILE, &tmV, row, h / p.group, &v_full[nv % L::VST]);
    ++nv;
  };
  auto load_q = [&](const AttnBf16Unit& u) {
    load(L::Q_OFF, &tmQ, u.q0, u.h, q_full);
    load(L::Q_OFF + L::TILE, &tmQ, u.q0 + 128, u.h, q_full);   // (zeros past the sequence; unused at 128 rows)
  };
  // Unit n of the list: long ones first where they are known, else the last tiles, which see most under causal spans.
  auto place = [&](AttnBf16Unit& u, int n) {
    u.h = p.tile_major ? n % p.heads : n / p.tiles;
    const int rank = p.tile_major ? n / p.heads : n % p.tiles;
    u.q0 = uniform(p.order ? p.order[rank] : p.tiles - 1 - rank) * p.rows;
  };
  int lo8[8], hi8[8];   // spans of its rows lane, 32 + lane ..
  auto spans = [&](const AttnBf16Unit& u) {
    const int q_end = min(u.q0 + p.rows, p.S);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int query = u.q0 + 32 * i + lane;
      lo8[i] = hi8[i] = 0;
      if (query < q_end) {
        lo8[i] = p.lo ? p.lo[query] : 0;
        hi8[i] = p.hi ? p.hi[query] : p.S;
      }
    }
  };
  auto describe = [&](AttnBf16Unit& u) {
    u.base = INT_MAX;
    int lo_min[2], hi_max[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int v[4] = {INT_MAX, -1, INT_MAX, -1};
#pragma unroll
      for (int i = 4 * t; i < 4 * t + 4; ++i) {
        const int a = max(lo8[i], 0), b = min(hi8[i], p.S);
        if (a < b) {
          v[0] = min(v[0], a);
          v[1] = max(v[1], a);
          v[2] = min(v[2], b);
          v[3] = max(v[3], b);
        }
      }
      lo_min[t] = __reduce_min_sync(~0u, v[0]);
      u.lo_max[t] = __reduce_max_sync(~0u, v[1]);
      u.hi_min[t] = __reduce_min_sync(~0u, v[2]);
      hi_max[t] = __reduce_max_sync(~0u, v[3]);
      u.base = min(u.base, lo_min[t]);
    }
    const int kend = max(hi_max[0], hi_max[1]);
    u.steps = kend > 0 ? (kend - u.base + 127) >> 7 : 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u.j0[t] = hi_max[t] > 0 ? (lo_min[t] - u.base) >> 7 : 0;
      u.j1[t] = hi_max[t] > 0 ? (hi_max[t] - u.base + 127) >> 7 : 0;
    }
    u.kk = 0.f;
    if (p.knorm && u.steps > 0) {
      // exactly the unit's keys, so that its results do not depend, in their rounding, on what lies beside them
      const int t0 = u.base >> 7, t1 = (kend - 1) >> 7;
      const float* one = p.knorm1 + (size_t)(u.h / p.group) * p.S;
      float edge[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = (i < 4 ? t0 : t1) * 128 + (i & 3) * 32 + lane;
        edge[i] = key >= u.base && key < kend ? one[key] : 0.f;
      }
      const float* kn = p.knorm + (size_t)(u.h / p.group) * ((p.S + 127) >> 7);
      for (int i = t0 + 1 + lane; i < t1; i += 32) u.kk = max_nan(u.kk, kn[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) u.kk = max_nan(u.kk, edge[i]);
#pragma unroll
      for (int o = 16; o; o >>= 1) u.kk = max_nan(u.kk, __shfl_xor_sync(~0u, u.kk, o));
    }
  };
  AttnBf16Unit first_unit;   // (TMA warp)
  if (warp == 8) {      // the first unit's loads are on their way before the rest is set up
    wait_primary();     // the preparation's results
    place(first_unit, blockIdx.x);
    spans(first_unit);
    if (lane == 0) {
      mbar_init(q_full, 2);
      mbar_init(q_empty, 10);
      for (int s = 0; s < L::KST; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 2);   // a commit of each MMA warp
      }
      for (int s = 0; s < L::VST; ++s) {
        mbar_init(&v_full[s], 1);
        mbar_init(&v_ok[s], 1);
        mbar_init(&v_empty[s], 2);
      }
      mbar_init(&unit_full[0], 1);
      mbar_init(&unit_full[1], 1);
      fence_barrier_init();
    }
    __syncwarp();
    load_q(first_unit);
    describe(first_unit);
    for (int j = 0; j < min(first_unit.steps, 2); ++j) {
      load_k(first_unit.base + 128 * j, first_unit.h);
      load_v(first_unit.base + 128 * j, first_unit.h);
    }
    if (lane == 0) {
      units[0] = first_unit;
      mbar_arrive(&unit_full[0]);
    }
  }
  static_assert(L::KST == 2 && L::VST == 2, "first loads");
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 4);
      mbar_init(&p_full[2 * t + 1], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_free[t], 4);
      mbar_init(&turn[t], 1);
      mbar_init(&guard_done[t], 1);
      mbar_init(&unit_empty[t], 11);   // MMA, guard and softmax warps
    }
    mbar_init(drained, 2);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  if (warp >= 8) {
    // The softmax warps hold a row's scores: 8 x 32 x 208 registers + 4 x 32 x 88 are the 384 x 168 of the launch.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      // ---------------------------------------------------------------- TMA
      AttnBf16Unit u = first_unit;
      const int all = p.tiles * p.heads;
      bool ok = true;
      int nq = 1;   // Q tiles asked for
      for (int it = 0; ok; ++it) {
        if (it > 0) {
          if (!(ok = __all_sync(~0u, mbar_wait(&unit_empty[it & 1], ((it >> 1) & 1) ^ 1, 300)))) break;
          if (lane == 0) {
            units[it & 1] = u;
            mbar_arrive(&unit_full[it & 1]);
          }
          __syncwarp();
          if (u.q0 < 0) break;
        }
        const int k0 = nk - (it ? 0 : min(u.steps, 2));   // tiles of earlier units
        int n = all;
        for (int j = 0; ok && j < max(u.steps, 1); ++j) {
          if (j < u.steps && k0 + j >= nk) {
            if (!(ok = __all_sync(~0u, mbar_wait(&k_empty[nk % L::KST], ((nk / L::KST) & 1) ^ 1, 301)))) break;
            load_k(u.base + 128 * j, u.h);
          }
          if (it > 0 && j == 0) {
            if (!(ok = __all_sync(~0u, mbar_wait(q_empty, (nq - 1) & 1, 304)))) break;
            load_q(u);
            ++nq;
          }
          // (asked for here, needed behind the loop; earlier would hand units to busy CTAs)
          if (p.next && j == max(u.steps - 3, 0) && lane == 0) n = gridDim.x + atomicAdd(p.next, 1);
          if (j < u.steps && k0 + j >= nv) {
            if (!(ok = __all_sync(~0u, mbar_wait(&v_empty[nv % L::VST], ((nv / L::VST) & 1) ^ 1, 302)))) break;
            load_v(u.base + 128 * j, u.h);
          }
        }
        n = uniform(lane == 0 ? n : 0);
        u.q0 = -1;
        if (n < all) {
          place(u, n);
          spans(u);
          describe(u);
        }
      }
      // nothing may still be landing in this CTA's memory when it ends, after a wait that gave up included
      mbar_drain(q_full, (nq - 1) & 1, 303);
      for (int j = max(nk - L::KST, 0); j < nk; ++j) mbar_drain(&k_full[j % L::KST], (j / L::KST) & 1, 303);
      for (int j = max(nv - L::VST, 0); j < nv; ++j) mbar_drain(&v_full[j % L::VST], (j / L::VST) & 1, 303);
    } else if (warp < 11) {
      // ---------------------------------------------------------------- MMA of one tile
      constexpr uint32_t idesc_s = idesc_bf16(128, 128, false), idesc_o = idesc_bf16(128, 128, true);
      const int t = warp - 9;
      const uint32_t s_tm = tmem + t * 128, o_tm = tmem + 256 + t * 128;
      // descriptors of the first tiles; others differ by 16-byte units in the low bits.  V rows are keys (the K
      // dimension), 64 dims contiguous: MN-major, 8-key groups 1,024 bytes apart, the two 64-dim halves SUB apart
      const uint64_t qd = sdesc_kmajor_sw128(smem_u32(smem + L::Q_OFF + t * L::TILE));
      const uint64_t kd0 = sdesc_kmajor_sw128(smem_u32(smem + L::K_OFF));
      const uint64_t vd0 = make_sdesc(smem_u32(smem + L::V_OFF), L::SUB, 1024, kLayoutSW128);
      auto issue_s = [&](int slot) {   // S = Q K^T: 8 MMAs over 16 dims each
        const uint64_t kd = kd0 + slot * (L::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t off = ((kk >> 2) * L::SUB + (kk & 3) * 32) >> 4;
          mma_bf16_ss(s_tm, qd + off, kd + off, idesc_s, kk != 0);
        }
      };
      auto issue_pv = [&](int slot, int half, bool add) {   // O (+)= P V over 64 keys: 4 MMAs over 16 keys each
        const uint64_t vd = vd0 + slot * (L::TILE >> 4);
#pragma unroll
        for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
          mma_bf16_ts(o_tm, s_tm + kk * 8, vd + kk * (2048 >> 4), idesc_o, add || kk != 0);
      };
      bool ok = true;
      int g0 = 0, r0 = 0, np = 0, no = 0;   // steps and rounds, this tile's P and O of earlier units
      for (int it = 0; ok; ++it) {
        if (!(ok = __all_sync(~0u, mbar_wait(&unit_full[it & 1], (it >> 1) & 1, 309)))) break;
        const AttnBf16Unit& u = units[it & 1];
        const int q0 = uniform(u.q0), steps = uniform(u.steps);
        const int first = uniform(t ? u.j0[1] : u.j0[0]), last = uniform(t ? u.j1[1] : u.j1[0]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&unit_empty[it & 1]);
        if (q0 < 0) break;
        const int q_last = last > first ? last - 1 : 0;   // the last step that reads Q
        ok = __all_sync(~0u, mbar_wait(q_full, it & 1, 310));
        if (steps == 0) {
          tc_commit(q_empty);
          continue;
        }
        for (int j = -1; ok && j < steps; ++j) {
          const int n = j + 1, g = g0 + j;
          // (also for steps this tile has no part in: a ring slot is free once both warps have let go of it)
          if (j >= 0 && !(ok = __all_sync(~0u, mbar_wait(&v_ok[g % L::VST], (g / L::VST) & 1, 311)))) break;
          if (n < steps && !(ok = __all_sync(~0u, mbar_wait(&k_full[(g + 1) % L::KST], ((g + 1) / L::KST) & 1, 312))))
            break;
          const bool pv = j >= first && j < last, qk = n >= first && n < last;
          // The warps take turns, A first.  Left to themselves the two tiles' MMAs interleave and finish together, and
          // both softmaxes then wait for both: 4,160 cycles a step, against 2,920 in turns at that time.  (Passing the
          // turn on before the last MMAs of S are issued: 150 us against 145 for the clips; waiting for P before the
          // turn: 146.)
          if (t + r0 + n > 0 && !(ok = __all_sync(~0u, mbar_wait(&turn[t], (r0 + n - 1 + t) & 1, 316 + t)))) break;
          if (pv) {
            // O of the unit before is in registers
            if (j == first && no > 0 && !(ok = __all_sync(~0u, mbar_wait(&o_free[t], (no - 1) & 1, 318)))) break;
            if (!(ok = __all_sync(~0u, mbar_wait(&p_full[2 * t], (np + j - first) & 1, 313 + t)))) break;
            tc_fence_after();
            issue_pv(g % L::VST, 0, j != first);
            if (!(ok = __all_sync(~0u, mbar_wait(&p_full[2 * t + 1], (np + j - first) & 1, 313 + t)))) break;
            tc_fence_after();
            issue_pv(g % L::VST, 1, true);
            if (n == last) tc_commit(&o_done[t]);
          }
          tc_fence_after();
          if (qk) {   // after PV(j) in issue order: P is read before S overwrites it
            issue_s((g + 1) % L::KST);
            tc_commit(&s_full[t]);
          }
          if (lane == 0) mbar_arrive(&turn[t ^ 1]);
          __syncwarp();
          if (j >= 0) tc_commit(&v_empty[g % L::VST]);
          if (n < steps) tc_commit(&k_empty[(g + 1) % L::KST]);
          if (n == q_last) tc_commit(q_empty);
        }
        g0 += steps;
        r0 += steps + 1;
        np += last - first;
        no += last > first;
      }
      // every MMA has left the tensor core before TMEM and shared memory are given back
      tc_commit(drained);
      mbar_drain(drained, 0, 315);
    } else {
      // ---------------------------------------------------------------- V guard
      bool ok = true;
      int g = 0;
      for (int it = 0; ok; ++it) {
        if (!(ok = __all_sync(~0u, mbar_wait(&unit_full[it & 1], (it >> 1) & 1, 321)))) break;
        const AttnBf16Unit u = units[it & 1];
        if (u.q0 < 0) break;
        // (a unit is published once the softmax warps are past the notes of the one two before it)
        uint32_t* notes = bad + (it & 1) * L::BAD_WORDS;
        for (int i = lane; i < (u.steps + 31) >> 5; i += 32) notes[i] = 0;
        if (lane == 0) any_bad[it & 1] = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&unit_empty[it & 1]);
        for (int j = 0; j < u.steps; ++j, ++g) {
          const int vs = g % L::VST;
          if (!(ok = __all_sync(~0u, mbar_wait(&v_full[vs], (g / L::VST) & 1, 320)))) break;
          const int kb = u.base + 128 * j;
          bool hides = false;   // some key of the step from some live row of a tile
#pragma unroll
          for (int t = 0; t < 2; ++t)
            hides |= j >= u.j0[t] && j < u.j1[t] && (u.lo_max[t] > kb || u.hi_min[t] < kb + 128);
          if (hides) {
            uint4* vt = reinterpret_cast<uint4*>(smem + L::V_OFF + vs * L::TILE);
            uint32_t seen = 0;   // adding one to an exponent of all ones carries into the sign's place
#pragma unroll 8
            for (int i = lane; i < L::TILE / 16; i += 32) {
              const uint4 w = vt[i];
              seen |= ((w.x & 0x7F807F80u) + 0x00800080u) | ((w.y & 0x7F807F80u) + 0x00800080u) |
                      ((w.z & 0x7F807F80u) + 0x00800080u) | ((w.w & 0x7F807F80u) + 0x00800080u);
            }
            if (__any_sync(~0u, (seen & 0x80008000u) != 0)) {
              for (int i = lane; i < L::TILE / 16; i += 32) {
                uint4 x = vt[i];
                uint32_t* w = &x.x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if ((w[e] & 0x7F80u) == 0x7F80u) w[e] &= 0xFFFF0000u;
                  if ((w[e] & 0x7F800000u) == 0x7F800000u) w[e] &= 0x0000FFFFu;
                }
                vt[i] = x;
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the MMA reads these writes
              if (lane == 0) {
                notes[j >> 5] |= 1u << (j & 31);
                any_bad[it & 1] = 1;
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ok[vs]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&guard_done[it & 1]);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: one thread per query row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lane_off + t * 128, o_col = tmem + lane_off + 256 + t * 128;
    const float scale = kLog2e * 0.08838834764831845f;   // log2(e) / sqrt(128)
    const uint64_t scale2 = f32x2_splat(scale);
    uint8_t* stage = smem + L::STAGE_OFF + warp * L::STAGE;
    bool ok = true;
    int ns = 0, no = 0;   // this tile's steps and its units with keys so far
    for (int it = 0; ok; ++it) {
      if (!(ok = __all_sync(~0u, mbar_wait(&unit_full[it & 1], (it >> 1) & 1, 336)))) break;
      const AttnBf16Unit& u = units[it & 1];
      const int q0 = u.q0, h = u.h, base = u.base;
      if (q0 < 0) break;
      const int first = t ? u.j0[1] : u.j0[0], last = t ? u.j1[1] : u.j1[0];
      const int lo_top = t ? u.lo_max[1] : u.lo_max[0], hi_low = t ? u.hi_min[1] : u.hi_min[0];
      const bool any = last > first;
      const int query = q0 + threadIdx.x, q_end = min(q0 + p.rows, p.S);
      int lo = 0, hi = 0;   // this row's span
      if (query < q_end) {
        lo = p.lo ? max(p.lo[query], 0) : 0;
        hi = p.hi ? min(p.hi[query], p.S) : p.S;
      }
      const bool live = lo < hi;
      float m_used = -INFINITY;   // the row's own largest score, not a rounded one: its P is then exactly 1 in bf16 too
      uint64_t l2a = 0, l2b = 0;
      bool bounded = false;
      if (!(ok = __all_sync(~0u, mbar_wait(q_full, it & 1, 334)))) break;
      if (p.knorm && any) {
        float qq = 0.f;
        const uint8_t* qr = smem + L::Q_OFF + t * L::TILE + (threadIdx.x & 127) * 128;
#pragma unroll
        for (int c = 0; c < 16; ++c) {   // (any order of the row's pieces will do)
          const uint4 v = *reinterpret_cast<const uint4*>(qr + (c >> 3) * L::SUB + (((c ^ lane) & 7) << 4));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) qq += bf16_lo(w[e]) * bf16_lo(w[e]) + bf16_hi(w[e]) * bf16_hi(w[e]);
        }
        bounded = __all_sync(~0u, !live || 2.0f * scale * sqrtf(qq) * sqrtf(u.kk) < kBoundBf16);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty);
      auto written = [&](int half) {   // P of 64 keys
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
      };
      for (int j = first; ok && j < last;) {
        // nearly every step of a long row: bounded scores, every key visible, 32 scores at a time with the next on their
        // way (P's words lie over scores that have been read)
        if (bounded && base + 128 * j >= lo_top && !__any_sync(~0u, m_used == -INFINITY)) {
          const int end = min(last, (hi_low - base) >> 7);
          const float nm = -m_used;
#pragma unroll 1
          for (; j < end; ++j, ++ns) {
            if (!(ok = __all_sync(~0u, mbar_wait(&s_full[t], ns & 1, 330 + t)))) break;
            tc_fence_after();
            uint32_t s[2][32];
            tmem_ld32(s_col, s[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_ld_wait();
              if (c < 3) tmem_ld32(s_col + 32 * (c + 1), s[(c + 1) & 1]);
              uint32_t pw[16];
              p_chunk_bf16<true>(s[c & 1], scale2, nm, pw, l2a, l2b);
              tmem_st16(s_col + 16 * c, pw);
              if (c & 1) written(c >> 1);
            }
          }
          if (!ok || j >= last) break;
        }
        const int kb = base + 128 * j;
        if (!(ok = __all_sync(~0u, mbar_wait(&s_full[t], ns & 1, 330 + t)))) break;
        tc_fence_after();
        const bool masked = lo_top > kb || hi_low < kb + 128;
        // 64 scores at a time, twice: for the maximum, and for P
        uint32_t s[2][32];
        auto scores = [&](int half) {
          tmem_ld32(s_col + 64 * half, s[0]);
          tmem_ld32(s_col + 64 * half + 32, s[1]);
          tmem_ld_wait();
          if (masked && live) {   // (a row without keys takes the scores as they are and is zeroed at the end)
            const int k = kb + 64 * half;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t vis = bits_below(hi - k - 32 * c) & ~bits_below(lo - k - 32 * c);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis >> e) & 1u)) s[c][e] = __float_as_uint(-INFINITY);
            }
          }
        };
        if (!bounded || __any_sync(~0u, m_used == -INFINITY)) {
          float mx = -INFINITY;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            scores(half);
            mx = fmaxf(mx, fmaxf(max_chunk(s[0], -INFINITY), max_chunk(s[1], -INFINITY)));
          }
          const float mnew = mx * scale;
          const bool need = m_used == -INFINITY ? mnew > m_used : mnew > m_used + kTauBf16 && !bounded;
          float alpha = 1.0f;
          if (need) {
            alpha = m_used == -INFINITY ? 0.0f : ex2(m_used - mnew);
            m_used = mnew;
            const uint64_t a2 = f32x2_splat(alpha);
            l2a = mul2(l2a, a2);
            l2b = mul2(l2b, a2);
          }
          // O holds the PV of every earlier step here: those MMAs were issued before S of this step by the same thread,
          // and s_full counts everything issued before its commit
          if (j > first && __any_sync(~0u, need)) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(o_col + 16 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(o_col + 16 * c, o);
            }
          }
        }
        const float nm = m_used == -INFINITY ? 0.0f : -m_used;   // no key yet: P = exp2(-inf) = 0
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          scores(half);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pw[16];
            p_chunk_bf16<false>(s[c], scale2, nm, pw, l2a, l2b);
            tmem_st16(s_col + 32 * half + 16 * c, pw);
          }
          written(half);
        }
        ++j, ++ns;
      }
      // ---- epilogue: O / l -> bf16, this thread's row
      if (ok && any) ok = __all_sync(~0u, mbar_wait(&o_done[t], no & 1, 332));
      if (ok) ok = __all_sync(~0u, mbar_wait(&guard_done[it & 1], (it >> 1) & 1, 333));
      if (!ok) break;
      if (any) tc_fence_after();
      float la, lb, lc, ld;
      f32x2_unpack(l2a, la, lb);
      f32x2_unpack(l2b, lc, ld);
      const float inv_l = 1.0f / ((la + lb) + (lc + ld));
      const bool repair = any && live && *(volatile int*)&any_bad[it & 1] != 0;
      const uint32_t* notes = bad + (it & 1) * L::BAD_WORDS;
      const int query0 = q0 + warp * 32;
      // 64 dims at a time through shared memory, swizzled, and out by TMA: whole lines instead of one row a thread
      // (3.7 us of a unit)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t o[2][32];
        if (any) {
#pragma unroll
          for (int c = 0; c < 2; ++c) tmem_ld32(o_col + 64 * half + 32 * c, o[c]);
          tmem_ld_wait();
          if (half == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[t]);
          }
        }
        if (query0 >= q_end) continue;
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[c][e] = live ? __float_as_uint(__uint_as_float(o[c][e]) * inv_l) : 0u;
          if (repair) {   // non-finite V elements this row does see
            for (int j = first; j < last; ++j) {
              if (!((notes[j >> 5] >> (j & 31)) & 1u)) continue;
              const int kb = base + 128 * j;
              for (int key = max(kb, lo); key < min(kb + 128, hi); ++key) {
                const __nv_bfloat16* vr =
                    p.v + (long long)key * p.ldv + (long long)(h / p.group) * p.hsv + 64 * half + 32 * c;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float x = __bfloat162float(vr[e]);
                  if (!isfinite(x)) o[c][e] = __float_as_uint(__uint_as_float(o[c][e]) + x);
                }
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e)
            w[16 * c + e] = pack_bf16(__uint_as_float(o[c][2 * e]), __uint_as_float(o[c][2 * e + 1]));
        }
        tma_store_wait_read<0>();   // the rows that were here have been read
        __syncwarp();
#pragma unroll
        for (int q8 = 0; q8 < 8; ++q8)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((q8 ^ (lane & 7)) << 4)) =
              make_uint4(w[4 * q8], w[4 * q8 + 1], w[4 * q8 + 2], w[4 * q8 + 3]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the store reads these writes
        __syncwarp();
        tma_store_3d(&tmO, stage, 64 * half, query0, h);
        tma_store_commit();
      }
      no += any;
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[it & 1]);
    }
    tma_store_wait_read<0>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace h3
