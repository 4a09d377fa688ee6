// Rotary positions with several axes (time, height, width): the rotation table of a packed sequence, and per-head
// QK-RMSNorm + split-half rotation straight from the positions.  No counterpart in the reference, whose host model
// makes the table (tools/profile_block.py:41-45) and whose kernel takes it ready-made
// (ck.rms_rope_split_half_, tfvideo/minimax_h3.py:296-298).
//
// Pair p of a head (dims p and p + rot/2) belongs to one axis a and is its j-th pair: angle = pos[s, a] *
// theta_a^(-2j / d_a), pairs of the axes one after another.  The angle is formed in 64 bits, in turns
// (pos * freq / 2 pi), and its whole turns are dropped there: a position of a million keeps 2^-33 of a turn, where
// 32 bits would keep 2^-4.  The rest, at most half a turn, is rounded to 32 bits once and goes to sincospi, so cosine
// and sine are within a few 2^-24 of the exact ones at any position.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "h3b200.h"

namespace h3 {

constexpr int kRopeMaxPairs = 64;   // rot <= 128, the head dim

struct RopePos {
  const void* pos;      // element (s, a) at s * ld + a * axis_stride
  long long ld, axis_stride;
  int type;             // H3_POS_*
  int pairs;            // rot / 2
  int end[4];           // end of each axis' pairs
  double power[4][6];   // theta_a^(-2 / d_a) to the powers 1, 2, 4 .. 32
};

__device__ __forceinline__ int rope_axis(const RopePos& r, int p) {   // of pair p
  return (p >= r.end[0]) + (p >= r.end[1]) + (p >= r.end[2]);
}
// Pair p's turns per unit of position: theta_a^(-2j / d_a) / 2 pi for its axis' j-th pair, as a product over the bits of
// j.  The kernel parameters are read at the same place by every lane; a table of 64 frequencies read lane by lane took
// 2 us at the start of a block.
__device__ __forceinline__ double rope_turns(const RopePos& r, int p) {
  const int axis = rope_axis(r, p);
  const int j = p - (axis == 0 ? 0 : axis == 1 ? r.end[0] : axis == 2 ? r.end[1] : r.end[2]);
  double turns = 0.15915494309189533577;   // 1 / (2 pi)
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 6; ++b)
      if (axis == a && (j >> b & 1)) turns *= r.power[a][b];
  return turns;
}

template <int TYPE>   // H3_POS_*
__device__ __forceinline__ double rope_load(const RopePos& r, long long s, int axis) {
  const long long o = s * r.ld + axis * r.axis_stride;
  if (TYPE == H3_POS_I32) return (double)reinterpret_cast<const int*>(r.pos)[o];
  if (TYPE == H3_POS_I64) return (double)reinterpret_cast<const long long*>(r.pos)[o];
  return (double)reinterpret_cast<const float*>(r.pos)[o];
}
// (cos, sin) of position p times `turns` turns
__device__ __forceinline__ float2 rope_cs(double p, double turns) {
  const double x = p * turns;
  float c, sn;
  sincospif(2.0f * (float)(x - rint(x)), &sn, &c);
  return make_float2(c, sn);
}

// out[s, p] = [[c, -s], [s, c]], fp32.  Bound by the 16 bytes written per pair; a thread keeps one pair (its frequency
// stays in a register) and walks over tokens, neighbouring threads neighbouring pairs, so a warp writes 512
// contiguous bytes.
template <int TYPE>
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ RopePos r, int S, float4* out) {
  const int per = 256 / r.pairs;   // tokens a block takes at a time
  const int p = threadIdx.x % r.pairs, t = threadIdx.x / r.pairs;
  if (t >= per) return;
  const int axis = rope_axis(r, p);
  const double turns = rope_turns(r, p);
  for (long long s = (long long)blockIdx.x * per + t; s < S; s += (long long)gridDim.x * per) {
    const float2 cs = rope_cs(rope_load<TYPE>(r, s, axis), turns);
    out[s * r.pairs + p] = make_float4(cs.x, -cs.y, cs.y, cs.x);
  }
}

struct QkNormAxesArgs {
  const __nv_bfloat16 *q, *k;    // element (s, h, d) at s * ld + h * hs + d
  __nv_bfloat16 *oq, *ok;        // as q / k themselves, or apart from them
  long long ldq, hsq, ldk, hsk, ldoq, hsoq, ldok, hsok;
  int S, Hq, Hk;
  const float *qw, *kw;
  float eps;
};

// The sum over the warp of each of G rows' partial sums p, for the lanes with row_of<G>(lane) = row.
template <int G>
__device__ __forceinline__ float warp_sum_rows(const float (&p)[G], int lane) {
  float q[G];
#pragma unroll
  for (int i = 0; i < G; ++i) q[i] = p[i];
#pragma unroll
  for (int w = G / 2, o = 16; w >= 1; w >>= 1, o >>= 1) {   // a lane keeps half of its rows and sends the other half
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float keep = up ? q[w + i] : q[i], send = up ? q[i] : q[w + i];
      q[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
#pragma unroll
  for (int o = 16 / G; o >= 1; o >>= 1) q[0] += __shfl_xor_sync(0xffffffffu, q[0], o);
  return q[0];
}

// y = x / sqrt(mean(x^2) + eps) * w over a head's 128 dims, then the rotation of dims < rot; one rounding to bf16.
// Bound by reading and writing q and k once.  One warp a token; lane l owns dims 4l..4l+3.  Rows go in groups of eight (q
// and k of four heads), the rest in smaller groups, each loaded whole before any of it is written, the first while the
// angles are computed.  A group's sums of squares are reduced over the warp together, one square root a row.  The
// weight and the rotation are one pair of factors a dim and token: o = r (x (w c) + x' (w' s)), x' the pair's other dim,
// fetched as the packed bf16 words.  A lane computes the angles of two pairs (64 over the warp) and fetches the four it
// needs by shuffles, since both halves of the rotated span use the same pairs.  gridDim.y > 1 splits a token's groups
// over blocks when there are too few tokens to fill the GPU.
struct QkRows {
  const __nv_bfloat16* in[2];   // q, k: this token's rows at this lane's dims
  __nv_bfloat16* out[2];
  float f[2][4], g[2][4];       // factors of the dim itself and of its partner
  int src, lane;
};

// G rows: rows h .. of q and of k in turn (KIND 2), or of q (0) or k (1) alone
template <int G, int KIND>
__device__ __forceinline__ void qk_load(const QkNormAxesArgs& a, const QkRows& t, int h, uint2 (&u)[G]) {
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int i = KIND == 2 ? j & 1 : KIND, row = KIND == 2 ? h + (j >> 1) : h + j;
    u[j] = *reinterpret_cast<const uint2*>(t.in[i] + row * (i ? a.hsk : a.hsq));
  }
}
template <int G, int KIND>
__device__ __forceinline__ void qk_finish(const QkNormAxesArgs& a, const QkRows& t, int h, const uint2 (&u)[G]) {
  float p[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const float x0 = bf16_lo(u[j].x), x1 = bf16_hi(u[j].x), x2 = bf16_lo(u[j].y), x3 = bf16_hi(u[j].y);
    p[j] = fmaf(x0, x0, x1 * x1) + fmaf(x2, x2, x3 * x3);
  }
  const float rmine = rsqrtf(fmaf(warp_sum_rows<G>(p, t.lane), 0.0078125f, a.eps));
#pragma unroll
  for (int j = 0; j < G; ++j) {
    // row j's sum is held by the lanes whose top bits, from bit 4 down, are j's from its highest down
    const int holder = G == 8 ? ((j >> 2) << 4) | ((j >> 1 & 1) << 3) | ((j & 1) << 2)
                     : G == 4 ? ((j >> 1) << 4) | ((j & 1) << 3)
                     : G == 2 ? j << 4 : 0;
    const float r = G == 1 ? rmine : __shfl_sync(0xffffffffu, rmine, holder);
    const uint32_t v0 = __shfl_sync(0xffffffffu, u[j].x, t.src), v1 = __shfl_sync(0xffffffffu, u[j].y, t.src);
    const int i = KIND == 2 ? j & 1 : KIND, row = KIND == 2 ? h + (j >> 1) : h + j;
    const float x[4] = {bf16_lo(u[j].x), bf16_hi(u[j].x), bf16_lo(u[j].y), bf16_hi(u[j].y)};
    const float y[4] = {bf16_lo(v0), bf16_hi(v0), bf16_lo(v1), bf16_hi(v1)};
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = r * fmaf(x[e], t.f[i][e], y[e] * t.g[i][e]);
    *reinterpret_cast<uint2*>(t.out[i] + row * (i ? a.hsok : a.hsoq)) =
        make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
  }
}
template <int G, int KIND>
__device__ __forceinline__ void qk_rows(const QkNormAxesArgs& a, const QkRows& t, int h) {
  uint2 u[G];
  qk_load<G, KIND>(a, t, h, u);
  qk_finish<G, KIND>(a, t, h, u);
}

// FEW: at most seven heads, as many of k as of q (one GPU's share of the heads): all of a token's rows are on their way
// before the angles, where the groups after the first would each wait for memory again.  (launch bounds: 80 registers,
// three blocks an SM, 44 bytes spilled, 4 with FEW; unbounded or four blocks measured 411 and 307 us against 264 at
// 37,760 tokens, 40 heads)
template <int TYPE, bool FEW>
__global__ void __launch_bounds__(256, 3) qknorm_rope_axes_kernel(const __grid_constant__ QkNormAxesArgs a,
                                                                     const __grid_constant__ RopePos r) {
  __shared__ double s_turns[kRopeMaxPairs];
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const bool mine = s < a.S;
  const int half = r.pairs, hq = half >> 2;
  const int d0 = lane * 4;
  const bool first = d0 < half, rotated = d0 < 2 * half;
  QkRows t;
  t.lane = lane;
  t.src = first ? lane + hq : (rotated ? lane - hq : lane);
  t.in[0] = a.q + s * a.ldq + d0;
  t.in[1] = a.k + s * a.ldk + d0;
  t.out[0] = a.oq + s * a.ldoq + d0;
  t.out[1] = a.ok + s * a.ldok + d0;
  const int both = min(a.Hq, a.Hk), four = both & ~3;
  int h = blockIdx.y * 4;
  uint2 u[8], u4[4], u2[2];
  if (mine && h < four) qk_load<8, 2>(a, t, h, u);
  if (FEW && mine && (both & 2)) qk_load<4, 2>(a, t, four, u4);
  if (FEW && mine && (both & 1)) qk_load<2, 2>(a, t, both - 1, u2);
  double pos[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) pos[e] = mine ? rope_load<TYPE>(r, s, rope_axis(r, min(2 * lane + e, half - 1))) : 0.0;
  if (threadIdx.x < half) s_turns[threadIdx.x] = rope_turns(r, threadIdx.x);
  __syncthreads();
  if (!mine) return;
  float2 cs[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) cs[e] = rope_cs(pos[e], s_turns[min(2 * lane + e, half - 1)]);
  const int p0 = first ? d0 : (rotated ? d0 - half : 0);
  float ca[4], cb[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int from = (p0 >> 1) + (e >> 1);
    const float c = __shfl_sync(0xffffffffu, cs[e & 1].x, from), sn = __shfl_sync(0xffffffffu, cs[e & 1].y, from);
    ca[e] = rotated ? c : 1.0f;
    cb[e] = rotated ? (first ? -sn : sn) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 w4 = *reinterpret_cast<const float4*>((i ? a.kw : a.qw) + d0);
    const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t.f[i][e] = w[e] * ca[e];
      t.g[i][e] = __shfl_sync(0xffffffffu, w[e], t.src) * cb[e];
    }
  }
  if (FEW) {
    if (four) qk_finish<8, 2>(a, t, 0, u);
    if (both & 2) qk_finish<4, 2>(a, t, four, u4);
    if (both & 1) qk_finish<2, 2>(a, t, both - 1, u2);
    return;
  }
  const int step = gridDim.y * 4;
  if (h < four) {
    qk_finish<8, 2>(a, t, h, u);
    for (h += step; h < four; h += step) qk_rows<8, 2>(a, t, h);
  }
  if (blockIdx.y != gridDim.y - 1) return;   // the last block of a token takes what is left
  h = four;
  if (both & 2) { qk_rows<4, 2>(a, t, h); h += 2; }
  if (both & 1) { qk_rows<2, 2>(a, t, h); ++h; }
  auto alone = [&](auto kind, int heads) {   // heads of the longer of q and k
    constexpr int K = decltype(kind)::value;
    for (; h + 8 <= heads; h += 8) qk_rows<8, K>(a, t, h);
    if (heads - h & 4) { qk_rows<4, K>(a, t, h); h += 4; }
    if (heads - h & 2) { qk_rows<2, K>(a, t, h); h += 2; }
    if (heads - h & 1) qk_rows<1, K>(a, t, h);
  };
  if (a.Hq > a.Hk) alone(std::integral_constant<int, 0>{}, a.Hq);
  else if (a.Hk > a.Hq) alone(std::integral_constant<int, 1>{}, a.Hk);
}

}  // namespace h3
