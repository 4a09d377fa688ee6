// Low-rank adapters of several requests beside a shared projection: out_m = y_m + B_a (scale_a A_a x_m), a = rows[m]
// (no adapter outside [0, n)).  No counterpart in the reference, which merges adapters into the weights before they are
// quantised (tfvideo/comfy_nodes.py:95-166): one set at a time, re-converting the model for each.
//
// Two kernels on tcgen05 (kind::f16, fp32 accumulators): shrink, T_m = scale_a A_a x_m, which reads x once, and
// expand, out = y + T B^T, which reads y and writes out once; T is M x R.  Both are bound by those bytes: a row of
// y, x and out is 2 (K + 2 N) bytes for 2 R (K + N) FLOP, R FLOP a byte, against about 250 at the measured rates.
// T is rounded to bf16 once (its sums are in 32 bits): 2^-8 of the adapter's part, which is added to y in 32 bits.
//
// Rows come in any order.  A 128-row tile works through the adapters that occur in it, and each row takes only its own
// adapter's product, from an accumulator of that adapter alone: another request's weights never reach it, non-finite
// ones included.  Rows without an adapter are copied (or left, in place) bit for bit.
#pragma once

#include "attention_bf16.cuh"
#include "common.cuh"
#include "h3b200.h"

namespace h3 {

struct AdapterArgs {
  const int* rows;      // [M]
  const float* scale;   // [n], or NULL: 1
  __nv_bfloat16* t;     // [M, Rp]
  int M, K, N, n;
  int Rp;               // rank rounded up to 16
  int inplace;          // expand: out is y
  int* next;            // expand: units handed out beyond each CTA's first; shrink sets it to zero
  int width;            // expand: 128-column tiles a unit
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {   // addr: cluster_addr of another CTA's shared memory
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

// warp-wide: transaction bytes expected on a barrier without an arrival
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .pred e;\n\t.reg .b32 rx;\n\t" H3_ELECT
               "@e mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n\t}" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}
// warp-wide: one arrival
__device__ __forceinline__ void mbar_arrive_warp(uint64_t* bar) {
  asm volatile("{\n\t.reg .pred e;\n\t.reg .b32 rx;\n\t" H3_ELECT
               "@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
// Programmatic dependent launch: the next kernel of the stream may start its blocks once every block of this one got
// here, and waits in wait_primary for this one's end (memory included) before it touches what this one wrote.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// One warp: the distinct adapters of rows m0 .. m0 + 127 in rising order; returns how many.  place (may be NULL): each
// row's place in that list, 255 without an adapter.
__device__ __forceinline__ int tile_adapters(const AdapterArgs& a, int m0, int lane, int* list, uint8_t* place) {
  int id[4], at[4] = {255, 255, 255, 255};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + 32 * i + lane;
    id[i] = m < a.M ? a.rows[m] : -1;
    if (id[i] < 0 || id[i] >= a.n) id[i] = INT_MAX;
  }
  int count = 0, last = -1;
  for (;;) {
    int next = INT_MAX;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (id[i] > last) next = min(next, id[i]);
    next = __reduce_min_sync(~0u, next);
    if (next == INT_MAX) break;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (id[i] == next) at[i] = count;
    if (lane == 0) list[count] = next;
    ++count;
    last = next;
  }
  if (place) {
#pragma unroll
    for (int i = 0; i < 4; ++i) place[32 * i + lane] = (uint8_t)at[i];
  }
  __syncwarp();
  return count;
}

// ------------------------------------------------------------------------------------------------ shrink
// blockIdx.x: 128-row tile; the CTAs of a cluster (gridDim.y, 1 to 8) share the tile's K range, and add their partial
// sums over distributed shared memory in a fixed order.  Stages of 64 K elements: the x tile (128 rows of 128 bytes)
// and, stacked as the MMA's N rows, the A rows of up to G adapters; a tile with more adapters walks x again for the
// next G (from L2).  Warps 0-3: epilogue, a thread per row; warp 4: TMA; warp 5: MMA.
struct ShrinkSmem {
  static constexpr int X = 128 * 128, SLOT = 2 * X;
  __host__ __device__ static constexpr int group(int rp) { return 128 / rp; }
  // two CTAs an SM when there are many, one deeper one when a tile is split
  __host__ __device__ static constexpr int stages(int rp, int splits) { return splits > 1 ? (rp > 64 ? 4 : 5) : 3; }
  static constexpr int MAX_STAGES = 5;
  __host__ __device__ static constexpr int red_row(int rp) { return rp * 4 + 16; }   // padded: threads hold rows
  __host__ __device__ static constexpr int total(int rp, int splits) {
    return 1024 + stages(rp, splits) * SLOT + (splits > 1 ? 128 * red_row(rp) : 0) + 1024;
  }
};

__global__ void __launch_bounds__(192)
    adapter_shrink_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA,
                          const AdapterArgs a) {
  using L = ShrinkSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int slot = L::SLOT;
  const int splits = gridDim.y;
  const int G = L::group(a.Rp), stages = L::stages(a.Rp, splits);
  uint8_t* red = smem + stages * slot;
  uint64_t* full = reinterpret_cast<uint64_t*>(red + (splits > 1 ? 128 * L::red_row(a.Rp) : 0));
  uint64_t* empty = full + L::MAX_STAGES;
  uint64_t* acc_full = empty + L::MAX_STAGES;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drained = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  int* count_s = reinterpret_cast<int*>(tmem_slot + 1);
  int* list = count_s + 1;   // [128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.x * 128;
  constexpr uint32_t ncols = 128;
  const int chunks = (a.K + 63) >> 6;
  const int c0 = (int)((long long)chunks * blockIdx.y / splits), c1 = (int)((long long)chunks * (blockIdx.y + 1) / splits);
  const int ahead = min(stages, c1 - c0);   // x tiles asked for before the tile's adapters are known

  if (warp == 4) {
    if (lane == 0) {
      for (int s = 0; s < L::MAX_STAGES; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      mbar_init(acc_full, 1);
      mbar_init(acc_empty, 4);
      mbar_init(drained, 1);
      fence_barrier_init();
    }
    __syncwarp();
    for (int i = 0; i < ahead; ++i) {
      mbar_expect_tx(&full[i], L::X);
      tma_load_3d(smem + i * slot, &tmX, (c0 + i) * 64, m0, 0, &full[i]);
    }
  }
  if (warp == 0) {
    const int c = tile_adapters(a, m0, lane, list, nullptr);
    if (lane == 0) *count_s = c;
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, ncols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int count = *count_s;
  const int passes = (count + G - 1) / G;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.next = 0;
  launch_dependents();   // (the next kernel's blocks wait for this one to end before they read T)

  if (warp == 4) {
    int it = 0;
    bool ok = true;
    for (int p = 0; ok && p < passes; ++p) {
      const int cnt = min(G, count - p * G);
      for (int c = c0; c < c1; ++c, ++it) {
        const int st = it % stages;
        ok = __all_sync(~0u, mbar_wait(&empty[st], ((it / stages) & 1) ^ 1, 401));
        if (!ok) break;
        uint8_t* s = smem + st * slot;
        mbar_arrive_expect_tx(&full[st], (it < ahead ? 0 : L::X) + cnt * a.Rp * 128);
        if (it >= ahead) tma_load_3d(s, &tmX, c * 64, m0, 0, &full[st]);
        for (int g = 0; g < cnt; ++g)
          tma_load_3d(s + L::X + g * a.Rp * 128, &tmA, c * 64, 0, list[p * G + g], &full[st]);
      }
    }
    // what is still landing: the last stages, and x tiles that no adapter asked for
    for (; it < ahead; ++it) mbar_arrive_warp(&full[it]);
    for (int j = max(it - stages, 0); j < it; ++j) mbar_drain(&full[j % stages], (j / stages) & 1, 402);
  } else if (warp == 5) {
    int it = 0;
    bool ok = true;
    for (int p = 0; ok && p < passes; ++p) {
      const int cnt = min(G, count - p * G);
      const uint32_t idesc = idesc_bf16(128, cnt * a.Rp, false);
      if (p > 0 && !(ok = __all_sync(~0u, mbar_wait(acc_empty, (p - 1) & 1, 411)))) break;
      for (int c = c0; c < c1; ++c, ++it) {
        const int st = it % stages;
        ok = __all_sync(~0u, mbar_wait(&full[st], (it / stages) & 1, 412));
        if (!ok) break;
        tc_fence_after();
        const uint32_t xa = smem_u32(smem + st * slot), wa = xa + L::X;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_bf16_ss(tmem, sdesc_kmajor_sw128(xa + kk * 32), sdesc_kmajor_sw128(wa + kk * 32), idesc, c != c0 || kk != 0);
        tc_commit(&empty[st]);
      }
      if (ok) tc_commit(acc_full);
    }
    tc_commit(drained);   // every MMA has left the tensor core before TMEM is given back
    mbar_drain(drained, 0, 413);
  } else {
    const int row = threadIdx.x, m = m0 + row;
    int id = m < a.M ? a.rows[m] : -1;
    if (id >= a.n) id = -1;
    const float sc = id >= 0 && a.scale ? a.scale[id] : 1.0f;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    for (int p = 0; p < passes; ++p) {
      const int cnt = min(G, count - p * G);
      if (!__all_sync(~0u, mbar_wait(acc_full, p & 1, 420))) break;
      tc_fence_after();
      for (int g = 0; g < cnt; ++g) {
        const bool mine = id == list[p * G + g];
        if (!__any_sync(~0u, mine)) continue;
        for (int c = 0; c < a.Rp; c += 16) {
          uint32_t v[16];
          tmem_ld16(tmem + lane_off + g * a.Rp + c, v);
          tmem_ld_wait();
          if (mine && splits > 1) {
            float4* d = reinterpret_cast<float4*>(red + row * L::red_row(a.Rp) + c * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              d[e] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]), __uint_as_float(v[4 * e + 2]),
                                 __uint_as_float(v[4 * e + 3]));
          } else if (mine) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              w[e] = pack_bf16(__uint_as_float(v[2 * e]) * sc, __uint_as_float(v[2 * e + 1]) * sc);
            uint4* d = reinterpret_cast<uint4*>(a.t + (size_t)m * a.Rp + c);
            d[0] = make_uint4(w[0], w[1], w[2], w[3]);
            d[1] = make_uint4(w[4], w[5], w[6], w[7]);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    const int per = 128 / splits, pieces = a.Rp >> 3;   // this CTA's rows, eight columns a thread at a time
    for (int i = threadIdx.x; i < per * pieces; i += 192) {
      const int row = blockIdx.y * per + i / pieces, c = (i % pieces) * 8, m = m0 + row;
      const int id = m < a.M ? a.rows[m] : -1;
      if (id < 0 || id >= a.n) continue;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < splits; ++s) {
        const uint32_t at = cluster_addr(red + row * L::red_row(a.Rp) + c * 4, s);
        const float4 u = ld_cluster_f4(at), v = ld_cluster_f4(at + 16);
        f[0] += u.x; f[1] += u.y; f[2] += u.z; f[3] += u.w;
        f[4] += v.x; f[5] += v.y; f[6] += v.z; f[7] += v.w;
      }
      const float sc = a.scale ? a.scale[id] : 1.0f;
      *reinterpret_cast<uint4*>(a.t + (size_t)m * a.Rp + c) =
          make_uint4(pack_bf16(f[0] * sc, f[1] * sc), pack_bf16(f[2] * sc, f[3] * sc), pack_bf16(f[4] * sc, f[5] * sc),
                     pack_bf16(f[6] * sc, f[7] * sc));
    }
    __syncwarp();
    cluster_sync();   // no CTA ends while another still reads its partial sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, ncols);
}

// ------------------------------------------------------------------------------------------------ expand
// Persistent over units of 128 rows x `width` tiles of 128 columns (T and the list of adapters stay over a unit), the
// first by block, the others from a counter: SMs get unequal shares of the memory, and equal runs of tiles ended between
// 371 and 526 us.  y, T and B tiles
// come by TMA through rings, out goes by TMA from where y landed, 32 rows a warp.  Warps 0-3 and 4-7: epilogue of every other
// tile, a thread per row (one such group took 2,900 cycles a tile, twice what memory allows); warp 8: TMA and the
// lists; warp 9: MMA.
struct ExpandSmem {
  static constexpr int SUB = 128 * 128;   // 128 rows x 64 elements
  __host__ __device__ static constexpr int kc(int rp) { return rp > 64 ? 2 : 1; }
  // y tiles in the ring: an even number, so that a slot always belongs to the same epilogue group (a barrier that two
  // groups took turns to wait on could be a phase behind for one of them)
  static constexpr int YS = 4;
  __host__ __device__ static constexpr int ts(int rp) { return rp > 64 ? 1 : 2; }   // T tiles
  __host__ __device__ static constexpr int total(int rp) {
    return 1024 + (2 * YS + (ts(rp) + 2) * kc(rp)) * SUB + 2048;
  }
};

__global__ void __launch_bounds__(320)
    adapter_expand_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmT,
                          const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmO,
                          const AdapterArgs a) {
  using L = ExpandSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int nys = L::YS;
  const int kc = L::kc(a.Rp), nts = L::ts(a.Rp);
  uint8_t* ys = smem;                         // [nys][2 SUB]
  uint8_t* ts = ys + 2 * nys * L::SUB;        // [nts][kc SUB]
  uint8_t* bs = ts + nts * kc * L::SUB;       // [2][kc SUB]
  uint64_t* y_full = reinterpret_cast<uint64_t*>(bs + 2 * kc * L::SUB);   // [4]
  uint64_t* y_empty = y_full + 4;    // [4]: out has been read from the slot, by each epilogue warp
  uint64_t* t_full = y_empty + 4;    // [2]
  uint64_t* t_empty = t_full + 2;
  uint64_t* b_full = t_empty + 2;    // [2]
  uint64_t* b_empty = b_full + 2;
  uint64_t* acc_full = b_empty + 2;  // [2]: the product of an epilogue group's tile
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* list_full = acc_empty + 2;   // [2]: the adapters of a row tile
  uint64_t* list_empty = list_full + 2;
  uint64_t* drained = list_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  int* unit_s = reinterpret_cast<int*>(tmem_slot + 1);    // [2]: -1 ends
  int* count_s = unit_s + 2;                              // [2]
  int* list_s = count_s + 2;                              // [2][128]: adapters of the unit's rows
  uint8_t* place_s = reinterpret_cast<uint8_t*>(list_s + 256);   // [2][128]: each row's place among them
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ntile = (a.N + 127) >> 7;
  const int strips = (ntile + a.width - 1) / a.width, units = strips * ((a.M + 127) >> 7);
  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < 4; ++s) {
        mbar_init(&y_full[s], 1);
        mbar_init(&y_empty[s], 4);
      }
      for (int s = 0; s < 2; ++s) {
        mbar_init(&t_full[s], 1);
        mbar_init(&t_empty[s], 1);
        mbar_init(&b_full[s], 1);
        mbar_init(&b_empty[s], 1);
        mbar_init(&acc_full[s], 1);
        mbar_init(&acc_empty[s], 4);
        mbar_init(&list_full[s], 1);
        mbar_init(&list_empty[s], 9);
      }
      mbar_init(drained, 1);
      fence_barrier_init();
    }
    __syncwarp();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // a unit's first row and its tiles [x0, x1) of columns
  auto locate = [&](int unit, int& m0, int& x0, int& x1) {
    m0 = unit / strips * 128;
    x0 = unit % strips * a.width;
    x1 = min(x0 + a.width, ntile);
  };

  if (warp == 8) {
    int ny = 0, nt = 0, nb = 0;   // y, T and B tiles asked for
    bool ok = true;
    auto load_y = [&](int m0, int x) {
      const int st = ny % nys;
      if (!(ok = __all_sync(~0u, mbar_wait(&y_empty[st], ((ny / nys) & 1) ^ 1, 451)))) return;
      mbar_arrive_expect_tx(&y_full[st], 2 * L::SUB);
      tma_load_3d(ys + 2 * st * L::SUB, &tmY, x * 128, m0, 0, &y_full[st]);
      tma_load_3d(ys + (2 * st + 1) * L::SUB, &tmY, x * 128 + 64, m0, 0, &y_full[st]);
      ++ny;
    };
    bool waited = false;
    int unit = blockIdx.x;
    for (int it = 0; ok; ++it) {
      int m0 = 0, x0 = 0, x1 = 0;
      if (unit < units) {
        locate(unit, m0, x0, x1);
        // out of place every tile of y is needed: the first is on its way before the adapters are known
        if (!a.inplace) load_y(m0, x0);
      }
      if (!ok || !(ok = __all_sync(~0u, mbar_wait(&list_empty[it & 1], ((it >> 1) & 1) ^ 1, 450)))) break;
      int* list = list_s + (it & 1) * 128;
      const int count = unit < units ? tile_adapters(a, m0, lane, list, place_s + (it & 1) * 128) : 0;
      if (lane == 0) {
        unit_s[it & 1] = unit < units ? unit : -1;
        count_s[it & 1] = count;
        mbar_arrive(&list_full[it & 1]);
      }
      __syncwarp();
      if (unit >= units) break;
      if (!waited) wait_primary();   // before T and the counter
      waited = true;
      if (lane == 0) unit = gridDim.x + atomicAdd(a.next, 1);
      if (count > 0) {
        const int st = nt % nts;
        if (!(ok = __all_sync(~0u, mbar_wait(&t_empty[st], ((nt / nts) & 1) ^ 1, 452)))) break;
        mbar_arrive_expect_tx(&t_full[st], kc * L::SUB);
        for (int c = 0; c < kc; ++c) tma_load_3d(ts + (st * kc + c) * L::SUB, &tmT, 64 * c, m0, 0, &t_full[st]);
        ++nt;
      }
      for (int x = x0; ok && x < x1; ++x) {
        if (a.inplace ? count > 0 : x > x0) load_y(m0, x);   // (in place, a tile without adapters stays as it is)
        for (int i = 0; ok && i < count; ++i, ++nb) {
          const int st = nb & 1;
          if (!(ok = __all_sync(~0u, mbar_wait(&b_empty[st], ((nb >> 1) & 1) ^ 1, 453)))) break;
          mbar_arrive_expect_tx(&b_full[st], kc * L::SUB);
          for (int c = 0; c < kc; ++c)
            tma_load_3d(bs + (st * kc + c) * L::SUB, &tmB, 64 * c, x * 128, list[i], &b_full[st]);
        }
      }
      unit = __shfl_sync(~0u, unit, 0);
    }
    for (int j = max(ny - nys, 0); j < ny; ++j) mbar_drain(&y_full[j % nys], (j / nys) & 1, 454);
    for (int j = max(nt - nts, 0); j < nt; ++j) mbar_drain(&t_full[j % nts], (j / nts) & 1, 454);
    for (int j = max(nb - 2, 0); j < nb; ++j) mbar_drain(&b_full[j & 1], (j >> 1) & 1, 454);
  } else if (warp == 9) {
    constexpr uint32_t idesc = idesc_bf16(128, 128, false);
    int nt = 0, nb = 0, ny = 0;   // T tiles, products and y tiles so far
    int np[2] = {0, 0};           // products of each group's tiles
    bool ok = true;
    for (int it = 0; ok; ++it) {
      if (!(ok = __all_sync(~0u, mbar_wait(&list_full[it & 1], (it >> 1) & 1, 460)))) break;
      const int unit = unit_s[it & 1], count = count_s[it & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_empty[it & 1]);
      if (unit < 0) break;
      int m0, x0, x1;
      locate(unit, m0, x0, x1);
      if (count == 0) {
        if (!a.inplace) ny += x1 - x0;
        continue;
      }
      const int tt = nt % nts;
      if (!(ok = __all_sync(~0u, mbar_wait(&t_full[tt], (nt / nts) & 1, 461)))) break;
      const uint32_t ta = smem_u32(ts + tt * kc * L::SUB);
      for (int x = x0; ok && x < x1; ++x, ++ny) {
        const int g = ny & 1;
        for (int i = 0; i < count; ++i, ++nb) {
          const int st = nb & 1, k = g ? np[1]++ : np[0]++;
          ok = __all_sync(~0u, mbar_wait(&b_full[st], (nb >> 1) & 1, 462)) &&
               __all_sync(~0u, mbar_wait(&acc_empty[g], (k & 1) ^ 1, 463));
          if (!ok) break;
          tc_fence_after();
          const uint32_t ba = smem_u32(bs + st * kc * L::SUB);
          for (int kk = 0; kk < a.Rp / 16; ++kk) {
            const uint32_t off = (kk >> 2) * L::SUB + (kk & 3) * 32;
            mma_bf16_ss(tmem + g * 128, sdesc_kmajor_sw128(ta + off), sdesc_kmajor_sw128(ba + off), idesc, kk != 0);
          }
          tc_commit(&acc_full[g]);
          tc_commit(&b_empty[st]);
        }
      }
      if (!ok) break;
      tc_commit(&t_empty[tt]);
      ++nt;
    }
    tc_commit(drained);   // every MMA has left the tensor core before TMEM is given back
    mbar_drain(drained, 0, 464);
  } else {
    const int row = threadIdx.x & 127, group = warp >> 2;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    int ny = 0, np = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      if (!(ok = __all_sync(~0u, mbar_wait(&list_full[it & 1], (it >> 1) & 1, 440)))) break;
      const int unit = unit_s[it & 1], count = count_s[it & 1];
      if (unit < 0) break;
      const int own = place_s[(it & 1) * 128 + row];
      int m0, x0, x1;
      locate(unit, m0, x0, x1);
      const int r0 = m0 + (warp & 3) * 32;
      for (int x = x0; x < x1 && (count > 0 || !a.inplace); ++x, ++ny) {
        if ((ny & 1) != group) continue;   // the other group's tile
        const int st = ny % nys;
        uint8_t* yt = ys + 2 * st * L::SUB;
        if (!(ok = __all_sync(~0u, mbar_wait(&y_full[st], (ny / nys) & 1, 441)))) break;
        for (int i = 0; i < count; ++i, ++np) {
          if (!(ok = __all_sync(~0u, mbar_wait(&acc_full[group], np & 1, 442)))) break;
          tc_fence_after();
          const bool mine = own == i;
          if (__any_sync(~0u, mine)) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t d[32];
              tmem_ld32(tmem + lane_off + group * 128 + 32 * c, d);
              tmem_ld_wait();
              if (mine) {
                uint8_t* sub = yt + (c >> 1) * L::SUB + row * 128;   // 16-byte pieces, swizzled as TMA wrote them
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  uint4* at = reinterpret_cast<uint4*>(sub + ((((c & 1) * 4 + q) ^ (row & 7)) << 4));
                  uint4 u = *at;
                  uint32_t* w = &u.x;
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    w[e] = pack_bf16(bf16_lo(w[e]) + __uint_as_float(d[8 * q + 2 * e]),
                                     bf16_hi(w[e]) + __uint_as_float(d[8 * q + 2 * e + 1]));
                  *at = u;
                }
              }
              __syncwarp();
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[group]);
        }
        if (!ok) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the store reads these writes
        __syncwarp();
        if (r0 < a.M) {
          const uint8_t* from = yt + (warp & 3) * 32 * 128;
          tma_store_3d(&tmO, from, x * 128, r0, 0);
          if (x * 128 + 64 < a.N) tma_store_3d(&tmO, from + L::SUB, x * 128 + 64, r0, 0);
        }
        tma_store_commit();
        tma_store_wait_read<0>();
        if (lane == 0) mbar_arrive(&y_empty[st]);
        __syncwarp();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_empty[it & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 256);
}

}  // namespace h3
