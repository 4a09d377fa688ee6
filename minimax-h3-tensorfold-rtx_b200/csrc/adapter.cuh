// Low-rank adapters of several requests beside a shared projection: out_m = y_m + B_a (scale_a A_a x_m), a = rows[m]
// (no adapter outside [0, n)).  No counterpart in the reference, which merges adapters into the weights before they are
// quantised (tfvideo/comfy_nodes.py:95-166): one set at a time, re-converting the model for each.
//
// plan: rows sorted by adapter into tiles of at most 128 rows, so that every tile is one adapter's (rows come in any
// order; without it a tile of six adapters took six passes).  shrink: T = scale_a A_a x of each tile, reading x once.
// expand: out = y + T B_a^T, reading y and writing out once.  Both products are tcgen05 kind::f16 with fp32
// accumulators, and both are bound by the bytes of x, y and out: 2 (K + 2 N) a row for 2 R (K + N) FLOP, about R FLOP a
// byte against 250 at the measured rates.  T is rounded to bf16 once (its sums are in 32 bits): 2^-8 of the adapter's
// part, which is added to y in 32 bits.
//
// A tile whose rows follow one another moves by TMA boxes, any other by 16-byte asynchronous copies and stores of
// single rows (TMA's gather4 took 90 cycles for each four rows, ten times too slow).  A row meets its own adapter's
// weights only, so another request's never reach it, non-finite ones included; rows without an adapter are copied (or
// left, in place) bit for bit.  With one adapter there is no plan: tiles are the rows in order, and rows without the
// adapter are left out in the epilogue.
#pragma once

#include "attention_bf16.cuh"
#include "common.cuh"
#include "h3b200.h"

namespace h3 {

struct AdapterArgs {
  const int* rows;      // [M]
  const float* scale;   // [n], or NULL: 1
  __nv_bfloat16* t;     // [M, Rp]: a tile's rows from its first place in perm on (without a plan, from its first row)
  const __nv_bfloat16 *x, *y;
  __nv_bfloat16* out;
  long long ldx, ldy, ldo;
  // the plan, or NULL without one: tiles {adapter (-1: none), first place in perm, rows, first row when its rows follow
  // one another, else -1}, how many, and the sorted rows
  const int4* tile;
  const int* total;
  const int* perm;
  int M, K, N, n;
  int Rp;               // rank rounded up to 16
  int inplace;          // expand: out is y
  int early;            // expand: need not wait for shrink to write rows without an adapter (no rows of x)
  int stages;           // shrink: ring depth
  int* next;            // expand: units handed out beyond each CTA's first
  int width;            // expand: 128-column tiles a unit
};

// 16 bytes of global into shared memory, asynchronously; zeros unless `in`
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// the calling lane's arrival, once its asynchronous copies so far have landed
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int ld_cluster_i32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {   // addr: cluster_addr of another CTA's shared memory
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

// ------------------------------------------------------------------------------------------------ plan
// One block takes 2,048 rows, cuts each run of one adapter every 128 rows, and appends the tiles to the list.  Rows in
// more runs than they fill tiles are sorted by (adapter, row) first (bitonic: strides below 64 in the registers of a
// warp, the others in shared memory; 8 us for 2,048, which part-filled tiles of a few runs do not cost; a call of 300 rows
// in four runs takes 15 us instead of 20 as they are).
constexpr int kPlanRows = 2048;
constexpr int kPlanCluster = 8;             // blocks that may be one cluster
constexpr int kPlanRuns = 8;                // runs that a block takes as they are, however few its rows
constexpr int kPlanMaxAdapters = 1 << 20;   // (adapter, row) in 32 bits

struct PlanArgs {
  const int* rows;
  int M, n;
  int4* tile;
  int* total;   // zero, and `next` too, unless there is one block or one cluster of them
  int* next;
  int* perm;
  int cluster;
};

__global__ void __launch_bounds__(1024) adapter_plan_kernel(const PlanArgs a) {
  __shared__ uint32_t key[kPlanRows];
  __shared__ int cut[kPlanRows];
  __shared__ int part[32];
  __shared__ int base, mine;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = blockIdx.x * kPlanRows, rows = min(kPlanRows, a.M - r0);
  launch_dependents();
  int size = 64;
  while (size < rows) size *= 2;
  for (int i = tid; i < size; i += 1024) {
    uint32_t k = ~0u;
    if (i < rows) {
      const int id = a.rows[r0 + i];
      k = (uint32_t)(id < 0 || id >= a.n ? 0 : id + 1) << 11 | (uint32_t)i;
    }
    key[i] = k;
  }
  __syncthreads();
  auto head = [&](int i) { return i < rows && (i == 0 || key[i] >> 11 != key[i - 1] >> 11); };
  const int runs = __syncthreads_count(head(2 * tid)) + __syncthreads_count(head(2 * tid + 1));
  if (runs > max(rows / 128, kPlanRuns)) {
    const int e0 = 64 * warp + lane, e1 = e0 + 32;   // this lane's elements
    const bool in = 64 * warp < size;
    uint32_t v0 = in ? key[e0] : 0, v1 = in ? key[e1] : 0;
    for (int k = 2; k <= size; k *= 2) {
      if (k > 64) {
        if (in) {
          key[e0] = v0;
          key[e1] = v1;
        }
        __syncthreads();
        for (int s = 31 - __clz(k / 2); s >= 6; --s) {   // stride 2^s, one pair a thread
          const int j = 1 << s, i = (tid >> s << (s + 1)) + (tid & (j - 1));
          if (tid < size / 2) {
            const uint32_t x = key[i], y = key[i + j];
            if ((x > y) == ((i & k) == 0)) {
              key[i] = y;
              key[i + j] = x;
            }
          }
          __syncthreads();
        }
        if (in) {
          v0 = key[e0];
          v1 = key[e1];
        }
      }
      if (k > 32) {
        const bool up = (e0 & k) == 0;
        const uint32_t x = min(v0, v1), y = max(v0, v1);
        v0 = up ? x : y;
        v1 = up ? y : x;
      }
      for (int j = min(k / 2, 16); j > 0; j /= 2) {
        const uint32_t o0 = __shfl_xor_sync(~0u, v0, j), o1 = __shfl_xor_sync(~0u, v1, j);
        const bool low = (lane & j) == 0;
        v0 = ((e0 & k) == 0) == low ? min(v0, o0) : max(v0, o0);
        v1 = ((e1 & k) == 0) == low ? min(v1, o1) : max(v1, o1);
      }
    }
    if (in) {
      key[e0] = v0;
      key[e1] = v1;
    }
    __syncthreads();
  }
  // each place's start of its adapter's run (a running maximum), two places a thread
  const int i0 = 2 * tid, i1 = i0 + 1;
  auto scan = [&](int v, auto join) {   // over a warp, this lane's included
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v = join(v, u);
    }
    return v;
  };
  auto before_me = [&](int v) {         // of the lane before, 0 for the first
    const int u = __shfl_up_sync(~0u, v, 1);
    return lane == 0 ? 0 : u;
  };
  auto most = [](int x, int y) { return max(x, y); };
  auto plus = [](int x, int y) { return x + y; };
  const int h0 = head(i0) ? i0 : 0, h1 = head(i1) ? i1 : 0;
  const int run = scan(max(h0, h1), most);
  if (lane == 31) part[warp] = run;
  __syncthreads();
  const int warps_run = __shfl_sync(~0u, before_me(scan(part[lane], most)), warp);
  const int s0 = max(max(before_me(run), warps_run), h0), s1 = max(s0, h1);
  const int c0 = i0 < rows && ((i0 - s0) & 127) == 0, c1 = i1 < rows && ((i1 - s1) & 127) == 0;
  __syncthreads();
  // the cuts' places in the list (a running sum)
  const int sum = scan(c0 + c1, plus);
  if (lane == 31) part[warp] = sum;
  __syncthreads();
  const int all = scan(part[lane], plus);
  const int at = sum - c0 - c1 + __shfl_sync(~0u, before_me(all), warp), tiles = __shfl_sync(~0u, all, 31);
  if (c0) cut[at] = i0;
  if (c1) cut[at + c0] = i1;
  // The blocks' places in the list: of one cluster, one after another by what each other block counts (2 us less than
  // with the counters zeroed first); else as they come (the tiles' order does not change what they compute).
  if (gridDim.x == 1) {
    if (tid == 0) {
      base = 0;
      *a.total = tiles;
      *a.next = 0;
    }
  } else if (a.cluster) {
    if (tid == 0) mine = tiles;
    cluster_sync();
    if (warp == 0) {
      const int n = lane < gridDim.x ? ld_cluster_i32(cluster_addr(&mine, lane)) : 0, upto = scan(n, plus);
      if (lane == blockIdx.x) base = upto - n;
      if (blockIdx.x == 0 && lane == 31) {
        *a.total = upto;
        *a.next = 0;
      }
    }
    cluster_sync();   // (no block ends while another still reads its count)
  } else if (tid == 0) {
    base = atomicAdd(a.total, tiles);
  }
  __syncthreads();
  for (int i = tid; i < rows; i += 1024) a.perm[r0 + i] = r0 + (int)(key[i] & (kPlanRows - 1));
  for (int t = tid; t < tiles; t += 1024) {
    const int b = cut[t], e = t + 1 < tiles ? cut[t + 1] : rows;
    const int first = r0 + (int)(key[b] & (kPlanRows - 1)), last = r0 + (int)(key[e - 1] & (kPlanRows - 1));
    a.tile[base + t] = make_int4((int)(key[b] >> 11) - 1, r0 + b, e - b, last - first == e - b - 1 ? first : -1);
  }
}

// A tile as the kernels take it: its adapter (-1: none), rows, and its first row when they follow one another (else -1).
struct TileInfo {
  int adapter, begin, count, first;
};
__device__ __forceinline__ TileInfo tile_info(const AdapterArgs& a, int t) {
  if (!a.tile) return {0, t * 128, min(128, a.M - t * 128), t * 128};
  const int4 v = a.tile[t];
  return {uniform(v.x), uniform(v.y), uniform(v.z), uniform(v.w)};
}
// Rows a lane copies of a tile whose rows do not follow one another: G of them from r0 on, every fourth (a lane's eighth
// of 128 bytes); -1 past the last.
template <int G>
struct LaneRows {
  int row[G];
  __device__ __forceinline__ void read(const int* rows, int count, int r0, int lane) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int r = r0 + 4 * i + (lane >> 3);
      row[i] = r < count ? rows[r] : -1;
    }
  }
  // 64 elements of each row, from column x on, into a swizzled tile of 128-byte rows; columns past `width` are zeros
  __device__ __forceinline__ void copy(uint8_t* tile, int r0, const __nv_bfloat16* base, long long ld, int x, int width,
                                       int lane) const {
    const int col = x + (lane & 7) * 8;
    const bool in = col < width;
    const __nv_bfloat16* from = base + (in ? col : 0);
    const uint32_t to = smem_u32(tile);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int r = r0 + 4 * i + (lane >> 3);
      if (row[i] >= 0) copy16_async(to + r * 128 + (((lane & 7) ^ (r & 7)) << 4), from + row[i] * ld, in);
    }
  }
};

// ------------------------------------------------------------------------------------------------ shrink
// blockIdx.x: tile; the CTAs of a cluster (gridDim.y, 1 to 8) share the tile's K range, and add their partial sums over
// distributed shared memory in a fixed order.  Stages of 64 K elements: the x tile (128 rows of 128 bytes; a box may
// bring rows behind the tile's last, whose T is never used) and the adapter's A rows.  Warps 0-3: the x rows where they
// do not follow one another, then the epilogue, a thread per row; warp 4: TMA; warp 5: MMA.
struct ShrinkSmem {
  static constexpr int X = 128 * 128, MAX_STAGES = 8;
  __host__ __device__ static constexpr int slot(int rp) { return X + rp * 128; }
  __host__ __device__ static constexpr int red_row(int rp) { return rp * 4 + 16; }   // padded: threads hold rows
  __host__ __device__ static constexpr int red(int rp, int splits) { return splits > 1 ? 128 * red_row(rp) : 0; }
  // as many stages as fit when that many CTAs share an SM
  __host__ __device__ static constexpr int stages(int rp, int splits, int ctas) {
    const int n = (233472 / ctas - 1024 - 2048 - red(rp, splits)) / slot(rp);
    return n < MAX_STAGES ? n : MAX_STAGES;
  }
  __host__ __device__ static constexpr int total(int rp, int splits, int stages) {
    return 1024 + stages * slot(rp) + red(rp, splits) + 1024;
  }
};

__global__ void __launch_bounds__(192)
    adapter_shrink_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA,
                          const AdapterArgs a) {
  using L = ShrinkSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int splits = gridDim.y;
  const int slot = L::slot(a.Rp), stages = a.stages;
  uint8_t* red = smem + stages * slot;
  uint64_t* full = reinterpret_cast<uint64_t*>(red + L::red(a.Rp, splits));
  uint64_t* empty = full + L::MAX_STAGES;
  uint64_t* acc_full = empty + L::MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  int* skip_s = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  constexpr uint32_t ncols = 128;
  if (a.tile) wait_primary();   // the plan
  else if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.next = 0;
  launch_dependents();   // (the next kernel's blocks wait for this one to end before they read T)
  if (a.tile && blockIdx.x >= *a.total) return;   // (every CTA of the cluster)
  const TileInfo tile = tile_info(a, blockIdx.x);
  if (tile.adapter < 0) return;
  const int chunks = (a.K + 63) >> 6;
  const int c0 = (int)((long long)chunks * blockIdx.y / splits), c1 = (int)((long long)chunks * (blockIdx.y + 1) / splits);

  if (warp == 4) {
    if (lane == 0) {
      for (int s = 0; s < L::MAX_STAGES; ++s) {
        mbar_init(&full[s], tile.first >= 0 ? 1 : 129);   // TMA's bytes, and every copying lane
        mbar_init(&empty[s], 1);
      }
      mbar_init(acc_full, 1);
      fence_barrier_init();
    }
    __syncwarp();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, ncols);
    tmem_relinquish();
  }
  if (warp == 0 && !a.tile) {   // without a plan a tile may hold no row that has the adapter
    int any = 0;
    for (int i = lane; i < tile.count; i += 32) any |= a.rows[tile.begin + i] == 0;
    any = __any_sync(~0u, any);
    if (lane == 0) *skip_s = !any;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const bool skip = !a.tile && *skip_s;   // the same in every CTA of the cluster

  if (skip) {
  } else if (warp == 4) {
    int it = 0;
    const int bytes = (tile.first >= 0 ? L::X : 0) + a.Rp * 128;
    for (int c = c0; c < c1; ++c, ++it) {
      const int st = it % stages;
      if (!__all_sync(~0u, mbar_wait(&empty[st], ((it / stages) & 1) ^ 1, 401))) break;
      uint8_t* s = smem + st * slot;
      mbar_arrive_expect_tx(&full[st], bytes);
      tma_load_3d(s + L::X, &tmA, c * 64, 0, tile.adapter, &full[st]);
      if (tile.first >= 0) tma_load_3d(s, &tmX, c * 64, tile.first, 0, &full[st]);
    }
    for (int j = max(it - stages, 0); j < it; ++j) mbar_drain(&full[j % stages], (j / stages) & 1, 402);
  } else if (warp == 5) {
    const uint32_t idesc = idesc_bf16(128, a.Rp, false);
    bool ok = true;
    for (int c = c0, it = 0; c < c1; ++c, ++it) {
      const int st = it % stages;
      ok = __all_sync(~0u, mbar_wait(&full[st], (it / stages) & 1, 412));
      if (!ok) break;
      if (tile.first < 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // x came by ordinary writes
      tc_fence_after();
      const uint32_t xa = smem_u32(smem + st * slot), wa = xa + L::X;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_bf16_ss(tmem, sdesc_kmajor_sw128(xa + kk * 32), sdesc_kmajor_sw128(wa + kk * 32), idesc, c != c0 || kk != 0);
      tc_commit(&empty[st]);
    }
    tc_commit(acc_full);
    mbar_drain(acc_full, 0, 413);   // every MMA has left the tensor core before TMEM is given back
  } else {
    const int row = threadIdx.x;
    const float sc = a.scale ? a.scale[tile.adapter] : 1.0f;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    if (tile.first < 0) {
      LaneRows<8> rows;
      rows.read(a.perm + tile.begin, tile.count, 32 * warp, lane);
      for (int c = c0, it = 0; c < c1; ++c, ++it) {
        const int st = it % stages;
        if (!__all_sync(~0u, mbar_wait(&empty[st], ((it / stages) & 1) ^ 1, 403))) break;
        rows.copy(smem + st * slot, 32 * warp, a.x, a.ldx, c * 64, a.K, lane);
        copies_arrive(&full[st]);
      }
    }
    if (__all_sync(~0u, mbar_wait(acc_full, 0, 420))) {
      tc_fence_after();
      for (int c = 0; c < a.Rp; c += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + lane_off + c, v);
        tmem_ld_wait();
        if (splits > 1) {
          float4* d = reinterpret_cast<float4*>(red + row * L::red_row(a.Rp) + c * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            d[e] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]), __uint_as_float(v[4 * e + 2]),
                               __uint_as_float(v[4 * e + 3]));
        } else {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pack_bf16(__uint_as_float(v[2 * e]) * sc, __uint_as_float(v[2 * e + 1]) * sc);
          if (row < tile.count) {   // (the rows behind are the next tile's)
            uint4* d = reinterpret_cast<uint4*>(a.t + ((size_t)tile.begin + row) * a.Rp + c);
            d[0] = make_uint4(w[0], w[1], w[2], w[3]);
            d[1] = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      }
    }
    tc_fence_before();
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    const int per = 128 / splits, pieces = a.Rp >> 3;   // this CTA's rows, eight columns a thread at a time
    const float sc = a.scale ? a.scale[tile.adapter] : 1.0f;
    for (int i = threadIdx.x; i < per * pieces; i += 192) {
      const int row = blockIdx.y * per + i / pieces, c = (i % pieces) * 8;
      if (row >= tile.count) break;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < splits; ++s) {
        const uint32_t at = cluster_addr(red + row * L::red_row(a.Rp) + c * 4, s);
        const float4 u = ld_cluster_f4(at), v = ld_cluster_f4(at + 16);
        f[0] += u.x; f[1] += u.y; f[2] += u.z; f[3] += u.w;
        f[4] += v.x; f[5] += v.y; f[6] += v.z; f[7] += v.w;
      }
      *reinterpret_cast<uint4*>(a.t + ((size_t)tile.begin + row) * a.Rp + c) =
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
// Persistent over units of one row tile x `width` tiles of 128 columns (T stays over a unit), the first by block, the
// others from a counter: SMs get unequal shares of the memory, and equal runs of tiles ended between 371 and 526 us.
// y, T and B tiles come by TMA through rings, out goes by TMA from where y landed, 32 rows a warp.  Warps 0-3 and 4-7:
// epilogue of every other tile, a thread per row (one such group took 2,900 cycles a tile, twice what memory allows);
// warp 8: TMA; warp 9: MMA; warps 10-13: y rows that do not follow one another.
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

// Shrink lets the expand kernel's blocks start before its own hold their TMEM (2 us of a small call).  They cannot take
// it from them and wait for them at once: no SM has the shared memory for a block of each.
constexpr bool never_share_an_sm() {
  for (int rp = 16; rp <= 128; rp += 16)
    for (int splits = 1; splits <= 2; ++splits)
      for (int ctas = 1; ctas <= (splits > 1 ? 2 : 3); ++ctas) {
        const int stages = ShrinkSmem::stages(rp, splits, ctas);
        if (stages >= 1 && ShrinkSmem::total(rp, splits, stages) + ExpandSmem::total(rp) <= 233472) return false;
      }
  return true;
}
static_assert(never_share_an_sm(), "a block of each kernel on one SM");

__global__ void __launch_bounds__(448)
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
  int* rows_s = reinterpret_cast<int*>(bs + 2 * kc * L::SUB);     // [2][128]: the rows of a unit
  uint64_t* y_full = reinterpret_cast<uint64_t*>(rows_s + 256);   // [4]
  uint64_t* y_empty = y_full + 4;    // [4]: out has been read from the slot, by each epilogue warp
  uint64_t* t_full = y_empty + 4;    // [2]
  uint64_t* t_empty = t_full + 2;
  uint64_t* b_full = t_empty + 2;    // [2]
  uint64_t* b_empty = b_full + 2;
  uint64_t* acc_full = b_empty + 2;  // [2]: the product of an epilogue group's tile
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* unit_full = acc_empty + 2;   // [2]: what the next unit is
  uint64_t* unit_empty = unit_full + 2;
  uint64_t* drained = unit_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  int* unit_s = reinterpret_cast<int*>(tmem_slot + 1);    // [2]: -1 ends
  int* kind_s = unit_s + 2;                               // [2]: 0 nothing to do, 1 y to out, 2 with an adapter
  int* first_s = kind_s + 2;                              // [2]: first row when the rows follow one another, else -1
  int* count_s = first_s + 2;                             // [2]: rows
  uint32_t* has_s = reinterpret_cast<uint32_t*>(count_s + 2);   // [2][4]: the rows that have the adapter
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int ntile = (a.N + 127) >> 7;
  const int strips = (ntile + a.width - 1) / a.width;

  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < 4; ++s) {
        mbar_init(&y_full[s], 129);   // TMA's bytes, and each lane of the copying warps
        mbar_init(&y_empty[s], 4);
      }
      for (int s = 0; s < 2; ++s) {
        mbar_init(&t_full[s], 1);
        mbar_init(&t_empty[s], 1);
        mbar_init(&b_full[s], 1);
        mbar_init(&b_empty[s], 1);
        mbar_init(&acc_full[s], 1);
        mbar_init(&acc_empty[s], 4);
        mbar_init(&unit_full[s], 1);
        mbar_init(&unit_empty[s], 13);
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
  const uint32_t tmem = uniform(*tmem_slot);
  auto cols = [&](int unit, int& x0, int& x1) {   // a unit's tiles [x0, x1) of columns
    x0 = unit % strips * a.width;
    x1 = min(x0 + a.width, ntile);
  };

  if (warp == 8) {
    int ny = 0, nt = 0, nb = 0;   // y, T and B tiles asked for
    bool ok = true, waited = false;
    if (a.tile || !a.early) {
      wait_primary();             // (the plan is older than the kernel before this one)
      waited = true;
    }
    const int units = (a.tile ? *a.total : (a.M + 127) >> 7) * strips;
    int unit = blockIdx.x;
    for (int it = 0; ok; ++it) {
      const int b = it & 1;
      if (!(ok = __all_sync(~0u, mbar_wait(&unit_empty[b], ((it >> 1) & 1) ^ 1, 450)))) break;
      TileInfo tile = {-1, 0, 0, 0};
      int x0 = 0, x1 = 0, kind = 0;
      auto load_y = [&](int x) {
        const int st = ny % nys;
        if (!(ok = __all_sync(~0u, mbar_wait(&y_empty[st], ((ny / nys) & 1) ^ 1, 451)))) return;
        mbar_arrive_expect_tx(&y_full[st], tile.first >= 0 ? 2 * L::SUB : 0);
        if (tile.first >= 0) {
          tma_load_3d(ys + 2 * st * L::SUB, &tmY, x * 128, tile.first, 0, &y_full[st]);
          tma_load_3d(ys + (2 * st + 1) * L::SUB, &tmY, x * 128 + 64, tile.first, 0, &y_full[st]);
        }
        ++ny;
      };
      if (unit < units) {
        tile = tile_info(a, unit / strips);
        cols(unit, x0, x1);
        if (tile.first < 0) {
#pragma unroll
          for (int i = lane; i < 128; i += 32) rows_s[128 * b + i] = i < tile.count ? a.perm[tile.begin + i] : -1;
        }
        // out of place every tile of y is needed: the first is on its way before its rows' adapters are known
        if (!a.inplace) load_y(x0);
        bool has[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = 32 * q + lane;
          has[q] = i < tile.count && (a.tile ? tile.adapter >= 0 : a.rows[tile.begin + i] == 0);
        }
        uint32_t any = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t w = __ballot_sync(~0u, has[q]);
          if (lane == 0) has_s[4 * b + q] = w;
          any |= w;
        }
        kind = any ? 2 : !a.inplace;
      }
      if (!ok) break;
      __syncwarp();   // every lane's rows_s before lane 0 lets the other warps read them
      if (lane == 0) {
        unit_s[b] = unit < units ? unit : -1;
        kind_s[b] = kind;
        first_s[b] = tile.first;
        count_s[b] = tile.count;
        mbar_arrive(&unit_full[b]);
      }
      __syncwarp();
      if (unit >= units) break;
      if (!waited) wait_primary();   // before T and the counter
      waited = true;
      if (lane == 0) unit = gridDim.x + atomicAdd(a.next, 1);
      if (kind == 2) {
        const int st = nt % nts;
        if (!(ok = __all_sync(~0u, mbar_wait(&t_empty[st], ((nt / nts) & 1) ^ 1, 452)))) break;
        mbar_arrive_expect_tx(&t_full[st], kc * L::SUB);
        // (with rows of the next tiles, whose products are not used; zeros past the last)
        for (int c = 0; c < kc; ++c) tma_load_3d(ts + (st * kc + c) * L::SUB, &tmT, 64 * c, tile.begin, 0, &t_full[st]);
        ++nt;
      }
      for (int x = x0; ok && x < x1 && kind > 0; ++x) {
        if (a.inplace || x > x0) load_y(x);
        if (!ok || kind < 2) continue;
        const int st = nb & 1;
        if (!(ok = __all_sync(~0u, mbar_wait(&b_empty[st], ((nb >> 1) & 1) ^ 1, 453)))) break;
        mbar_arrive_expect_tx(&b_full[st], kc * L::SUB);
        for (int c = 0; c < kc; ++c)
          tma_load_3d(bs + (st * kc + c) * L::SUB, &tmB, 64 * c, x * 128, tile.adapter, &b_full[st]);
        ++nb;
      }
      unit = uniform(lane == 0 ? unit : 0);
    }
    if (!waited) wait_primary();   // (a call ends after all its kernels)
    for (int j = max(ny - nys, 0); j < ny; ++j) mbar_drain(&y_full[j % nys], (j / nys) & 1, 454);
    for (int j = max(nt - nts, 0); j < nt; ++j) mbar_drain(&t_full[j % nts], (j / nts) & 1, 454);
    for (int j = max(nb - 2, 0); j < nb; ++j) mbar_drain(&b_full[j & 1], (j >> 1) & 1, 454);
  } else if (warp == 9) {
    constexpr uint32_t idesc = idesc_bf16(128, 128, false);
    int nt = 0, nb = 0, ny = 0;   // T tiles, products and y tiles so far
    int np[2] = {0, 0};           // products of each group's tiles
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int b = it & 1;
      if (!(ok = __all_sync(~0u, mbar_wait(&unit_full[b], (it >> 1) & 1, 460)))) break;
      const int unit = uniform(unit_s[b]), kind = uniform(kind_s[b]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[b]);
      if (unit < 0) break;
      int x0, x1;
      cols(unit, x0, x1);
      if (kind < 2) {
        if (kind == 1) ny += x1 - x0;
        continue;
      }
      const int tt = nt % nts;
      if (!(ok = __all_sync(~0u, mbar_wait(&t_full[tt], (nt / nts) & 1, 461)))) break;
      const uint32_t ta = smem_u32(ts + tt * kc * L::SUB);
      for (int x = x0; x < x1; ++x, ++ny, ++nb) {
        const int g = ny & 1, st = nb & 1, k = g ? np[1]++ : np[0]++;
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
      if (!ok) break;
      tc_commit(&t_empty[tt]);
      ++nt;
    }
    tc_commit(drained);   // every MMA has left the tensor core before TMEM is given back
    mbar_drain(drained, 0, 464);
  } else if (warp >= 10) {
    int ny = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int b = it & 1;
      if (!(ok = __all_sync(~0u, mbar_wait(&unit_full[b], (it >> 1) & 1, 470)))) break;
      const int unit = unit_s[b], kind = kind_s[b], first = first_s[b], count = count_s[b];
      if (unit < 0) break;
      LaneRows<8> rows;
      if (first < 0) rows.read(rows_s + 128 * b, count, 32 * (warp - 10), lane);
      __syncwarp();
      int x0, x1;
      cols(unit, x0, x1);
      for (int x = x0; x < x1 && kind > 0; ++x, ++ny) {
        const int st = ny % nys;
        if (!(ok = __all_sync(~0u, mbar_wait(&y_empty[st], ((ny / nys) & 1) ^ 1, 471)))) break;
        if (first < 0) {
          for (int i = 0; i < 2; ++i)
            rows.copy(ys + (2 * st + i) * L::SUB, 32 * (warp - 10), a.y, a.ldy, x * 128 + 64 * i, a.N, lane);
        }
        copies_arrive(&y_full[st]);   // (at once, when there are none)
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&unit_empty[b]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    const int row = threadIdx.x & 127, group = warp >> 2, quad = warp & 3;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    int ny = 0, np = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int b = it & 1;
      if (!(ok = __all_sync(~0u, mbar_wait(&unit_full[b], (it >> 1) & 1, 440)))) break;
      const int unit = unit_s[b], kind = kind_s[b], first = first_s[b], count = count_s[b];
      if (unit < 0) break;
      const uint32_t has = has_s[4 * b + quad];
      const bool mine = (has >> lane) & 1u;
      int x0, x1;
      cols(unit, x0, x1);
      for (int x = x0; x < x1 && kind > 0; ++x, ++ny) {
        if ((ny & 1) != group) continue;   // the other group's tile
        const int st = ny % nys;
        uint8_t* yt = ys + 2 * st * L::SUB;
        if (!(ok = __all_sync(~0u, mbar_wait(&y_full[st], (ny / nys) & 1, 441)))) break;
        if (kind == 2) {
          if (!(ok = __all_sync(~0u, mbar_wait(&acc_full[group], np & 1, 442)))) break;
          ++np;
          tc_fence_after();
          if (has) {
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
        // this warp's rows out: a box of 32 while it holds no others (rows past the matrix are not written), else row
        // by row, 256 bytes each
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // TMA reads these writes, and writes here next
        __syncwarp();
        const uint8_t* from = yt + quad * 32 * 128;
        if (first >= 0 && (quad * 32 + 32 <= count || first + count == a.M)) {
          if (first + quad * 32 < a.M) {
            tma_store_3d(&tmO, from, x * 128, first + quad * 32, 0);
            if (x * 128 + 64 < a.N) tma_store_3d(&tmO, from + L::SUB, x * 128 + 64, first + quad * 32, 0);
          }
          tma_store_commit();
          tma_store_wait_read<0>();
        } else {
          const int col = x * 128 + (lane & 15) * 8;
          const uint8_t* sub = from + ((lane >> 3) & 1) * L::SUB;
#pragma unroll 4
          for (int r = lane >> 4; r < min(32, count - quad * 32); r += 2) {
            const int at = first >= 0 ? first + quad * 32 + r : rows_s[128 * b + quad * 32 + r];
            if (col < a.N)
              *reinterpret_cast<uint4*>(a.out + (long long)at * a.ldo + col) =
                  *reinterpret_cast<const uint4*>(sub + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&y_empty[st]);
        __syncwarp();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 256);
}

}  // namespace h3
