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
  uint8_t axis[kRopeMaxPairs];
  double turns[kRopeMaxPairs];   // turns per unit of position of pair p
};

// (cos, sin) of the pair's angle at token s
__device__ __forceinline__ float2 rope_cs(const RopePos& r, int s, int axis, double turns) {
  const long long o = (long long)s * r.ld + axis * r.axis_stride;
  double p;
  if (r.type == H3_POS_I32) p = (double)reinterpret_cast<const int*>(r.pos)[o];
  else if (r.type == H3_POS_I64) p = (double)reinterpret_cast<const long long*>(r.pos)[o];
  else p = (double)reinterpret_cast<const float*>(r.pos)[o];
  const double x = p * turns;
  float c, sn;
  sincospif(2.0f * (float)(x - rint(x)), &sn, &c);
  return make_float2(c, sn);
}

// out[s, p] = [[c, -s], [s, c]], fp32.  Bound by the 16 bytes written per pair; a thread keeps one pair (its frequency
// stays in a register) and walks over tokens, neighbouring threads neighbouring pairs, so a warp writes 512
// contiguous bytes.
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ RopePos r, int S, float4* out) {
  const int per = 256 / r.pairs;   // tokens a block takes at a time
  const int p = threadIdx.x % r.pairs, t = threadIdx.x / r.pairs;
  if (t >= per) return;
  const int axis = r.axis[p];
  const double turns = r.turns[p];
  for (long long s = (long long)blockIdx.x * per + t; s < S; s += (long long)gridDim.x * per) {
    const float2 cs = rope_cs(r, (int)s, axis, turns);
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

// y = x / sqrt(mean(x^2) + eps) * w over a head's 128 dims, then the rotation of dims < rot; one rounding to bf16.
// Bound by reading and writing q and k once.  One warp takes a token's head rows (q heads, then k heads) in groups of
// eight, all eight in flight before the first is written; lane l owns dims 4l..4l+3.  The eight sums of squares are
// reduced over the warp transposed (warp_sum8_transposed), one sqrt and division per row.  A lane computes the
// angles of two pairs (64 over the warp) and fetches the four it needs by shuffles, since both halves of the rotated
// span use the same pairs.  gridDim.y > 1 splits a token's groups over blocks when there are too few tokens to fill
// the GPU.
__global__ void __launch_bounds__(256) qknorm_rope_axes_kernel(const __grid_constant__ QkNormAxesArgs a,
                                                               const __grid_constant__ RopePos r) {
  __shared__ double s_turns[kRopeMaxPairs];
  __shared__ int s_axis[kRopeMaxPairs];
  if (threadIdx.x < r.pairs) {   // lanes reading different entries of a kernel parameter would serialise: once a block
    s_turns[threadIdx.x] = r.turns[threadIdx.x];
    s_axis[threadIdx.x] = r.axis[threadIdx.x];
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (s >= a.S) return;
  const int half = r.pairs, hq = half >> 2;
  const int d0 = lane * 4;
  const bool first = d0 < half, rotated = d0 < 2 * half;
  const int src = first ? lane + hq : (rotated ? lane - hq : lane);
  const int rows = a.Hq + a.Hk;

  float2 mine[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int p = min(2 * lane + e, half - 1);
    mine[e] = rope_cs(r, s, s_axis[p], s_turns[p]);
  }
  float ca[4], cb[4];   // o = ca * y + cb * y_partner
  const int p0 = first ? d0 : (rotated ? d0 - half : 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int from = (p0 >> 1) + (e >> 1);
    ca[e] = __shfl_sync(0xffffffffu, mine[e & 1].x, from);
    const float sn = __shfl_sync(0xffffffffu, mine[e & 1].y, from);
    cb[e] = first ? -sn : sn;
  }
  const float4 qw4 = *reinterpret_cast<const float4*>(a.qw + d0), kw4 = *reinterpret_cast<const float4*>(a.kw + d0);
  const float qw[4] = {qw4.x, qw4.y, qw4.z, qw4.w}, kw[4] = {kw4.x, kw4.y, kw4.z, kw4.w};
  const __nv_bfloat16* qrow = a.q + s * a.ldq + d0;
  const __nv_bfloat16* krow = a.k + s * a.ldk + d0;
  __nv_bfloat16* oqrow = a.oq + s * a.ldoq + d0;
  __nv_bfloat16* okrow = a.ok + s * a.ldok + d0;

  for (int r0 = blockIdx.y * 8; r0 < rows; r0 += gridDim.y * 8) {
    uint2 u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = r0 + j;
      u[j] = make_uint2(0u, 0u);
      if (i < a.Hq) u[j] = *reinterpret_cast<const uint2*>(qrow + i * a.hsq);
      else if (i < rows) u[j] = *reinterpret_cast<const uint2*>(krow + (i - a.Hq) * a.hsk);
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = sumsq4(u[j]);
    const float ss = warp_sum8_transposed(p, lane);
    const float rmine = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(ss * 0.0078125f, a.eps)));
#pragma unroll
    for (int j = 0; j < 8; ++j) {   // row j's sum is held by lane 16 (j>>2) + 8 (j>>1 & 1) + 4 (j & 1)
      const int i = r0 + j;
      const float rj = __shfl_sync(0xffffffffu, rmine, ((j >> 2) << 4) | (((j >> 1) & 1) << 3) | ((j & 1) << 2));
      if (i < a.Hq)
        *reinterpret_cast<uint2*>(oqrow + i * a.hsoq) = qk_row(u[j], qw, ca, cb, rotated, src, rj);
      else if (i < rows)
        *reinterpret_cast<uint2*>(okrow + (i - a.Hq) * a.hsok) = qk_row(u[j], kw, ca, cb, rotated, src, rj);
    }
  }
}

}  // namespace h3
