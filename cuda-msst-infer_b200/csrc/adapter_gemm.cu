// adapter_gemm.cu — a shared projection with the low-rank adapters of many requests
// beside it: y[t] = W x[t] + bias + s_a B_a (A_a x[t]), a = row_adapter[t].
//
// Two launches.  adapter_down_kernel computes u[t] = A_a x[t] for every row that has an
// adapter; adapter_gemm_kernel computes W x and adds B_a (s_a u) as a few more K steps
// of the same accumulators, so the low-rank term costs no pass over the output.
//
// Both work on tiles of BT rows (32 to 256) and on the list of the distinct adapters
// of a tile.  An adapter's part of the extra K steps is a slice of 16 rank values
// (ceil(rank / 16) slices an adapter): B_a's columns on one side, on the other U', which
// holds s_a u for the rows whose adapter is a and zeros for all others.  So requests
// may be mixed row by row: a tile costs as many slices as it has adapters.
//
// The weights are the MMA's M side (128 of their rows) and the rows of x its N side: with
// few rows the instruction then still covers 4 KB of weights, where an M side of rows
// would be padded to 128 and the one issuing thread, at about 60 cycles an MMA, would
// bound the pass (K = N = 4096: 8 us of issue for 32 columns a CTA, against the 5.2 us
// that reading W takes).  Few tiles are split along K over a cluster, whose CTAs add
// their parts through distributed shared memory in rank order.
//
// u is rounded to the operands' 16 bits once, as U' feeds the tensor cores; it is summed
// in fp32 before that (split-K parts of the first launch in order).
#include <algorithm>

#include "common.cuh"
#include "operators.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr uint32_t kWTile = 128 * 128;       // 128 weight rows x 64 columns of 16 bits
constexpr int kSliceRows = 16;               // rank values of a slice

// The plan of a call, the same for both launches.
struct Plan {
  int bt;           // rows of x a tile
  int tiles;        // ceil(rows / bt)
  int n_tiles;      // ceil(N / 128)
  int kblocks;      // ceil(K / 64)
  int chunks;       // slices an adapter
  // first launch: CTAs along the rows (of 32 * 8 / down_kw rows), along a tile's adapters and
  // along K; warps of a CTA along K; 8-value rank pieces of a pass
  int down_x, down_y, down_split, down_kw, down_nt;
  int split;        // CTAs of a cluster along K in the second launch
  int x_box;        // rows of x a TMA box brings (bt, fewer when there are fewer rows)
  int list_ld;      // ints of a tile's list
};

// A tile's list: [0] distinct adapters, [1] whether the tile's rows differ, [2 ..] the adapters.
__host__ __device__ inline size_t list_offset(const AdapterGemmParams& p, const Plan& pl) {
  return (size_t)pl.down_split * p.rows * p.rank * sizeof(float);
}

__device__ __forceinline__ int row_id(const AdapterGemmParams& p, long long t) {
  if (t >= p.rows) return -1;
  const int a = __ldg(p.row_adapter + t);
  return a >= 0 && a < p.adapters ? a : -1;
}

// ---------------------------------------------------------------------------
// First launch: u[t] = A_a x[t].  Bound: reading x once (and, for few rows, the adapters' A_a).
// mma.sync m16n8k16 on fragments loaded straight from global memory: a lane takes 8
// consecutive columns of a row (16 bytes; four lanes read 64 consecutive bytes), which serve
// two K steps, x and A_a in the same order.  No barrier, no staging: a launch this short
// is bound by latency, and many small CTAs hide it best.  (A tcgen05 form with 128-row A
// slices took 35 us for 8192 rows of 4096 columns, mostly set-up and drain.)
// A warp owns 32 rows; the warps of a CTA split K (down_kw of them) and rows.  For every
// distinct adapter of its rows it computes all 32 x rank products from the rows that have
// the adapter and keeps those.
// The last tiles' worth of blocks write the lists of the second launch's row tiles.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The list of row tile `tile`: its adapters in order of first appearance.
__device__ void write_list(const AdapterGemmParams& p, const Plan& pl, int tile) {
  __shared__ int s_id[256], s_count[8], s_mixed;
  const int r = threadIdx.x, warp = r >> 5, lane = r & 31;
  const long long t = (long long)tile * pl.bt + r;
  const bool in = r < pl.bt && t < p.rows;
  const int id = in ? row_id(p, t) : -1;
  s_id[r] = id;
  if (in && id < 0 && __ldg(p.row_adapter + t) != -1) record_error(kErrAdapter);
  if (r == 0) s_mixed = 0;
  __syncthreads();
  if (in && id != s_id[0]) s_mixed = 1;
  bool first = id >= 0;
  for (int x = 0; x < r && first; ++x) first = s_id[x] != id;
  const unsigned firsts = __ballot_sync(0xffffffffu, first);
  if (lane == 0) s_count[warp] = __popc(firsts);
  __syncthreads();
  int at = __popc(firsts & ((1u << lane) - 1u)), count = 0;
  for (int x = 0; x < 8; ++x) {
    if (x < warp) at += s_count[x];
    count += s_count[x];
  }
  int* list = reinterpret_cast<int*>(static_cast<uint8_t*>(p.ws) + list_offset(p, pl)) + (size_t)tile * pl.list_ld;
  if (first) list[2 + at] = id;
  if (r == 0) {
    list[0] = count;
    list[1] = s_mixed;
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(256)
    adapter_down_kernel(const __grid_constant__ AdapterGemmParams p, const __grid_constant__ Plan pl) {
  extern __shared__ __align__(16) float s_part[];  // [8 warps][32 rows][NT * 8]
  dependents_may_start();
  if (blockIdx.x >= pl.down_x) {
    if (blockIdx.y == 0 && blockIdx.z == 0) write_list(p, pl, blockIdx.x - pl.down_x);
    return;
  }
  constexpr int kR = NT * 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kw = pl.down_kw, kwarp = warp % kw, group = warp / kw;
  const long long t0 = ((long long)blockIdx.x * (8 / kw) + group) * 32;
  if (t0 >= p.rows) return;
  const int id = row_id(p, t0 + lane);
  const unsigned same = __match_any_sync(0xffffffffu, id);
  unsigned firsts = __ballot_sync(0xffffffffu, id >= 0 && __ffs(same) - 1 == lane);
  const int steps = (p.K + 31) / 32, parts = pl.down_split * kw, me = blockIdx.z * kw + kwarp;
  const int s0 = (int)((long long)steps * me / parts), s1 = (int)((long long)steps * (me + 1) / parts);
  const int row = lane >> 2, quad = lane & 3;
  const T* x = static_cast<const T*>(p.x) + t0 * p.ldx + quad * 8;
  for (int li = 0; firsts; ++li, firsts &= firsts - 1) {
    if (li % pl.down_y != blockIdx.y) continue;
    const int src = __ffs(firsts) - 1;
    const int a = __shfl_sync(0xffffffffu, id, src);
    const unsigned mine = __shfl_sync(0xffffffffu, same, src);  // the rows that have adapter a
    for (int r0 = 0; r0 < p.rank; r0 += kR) {
      const T* la = static_cast<const T*>(p.lora_a) + ((size_t)a * p.rank + r0) * p.K + quad * 8;
      float acc[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2 * NT * 4; ++i) (&acc[0][0][0])[i] = 0.f;
#pragma unroll 2
      for (int s = s0; s < s1; ++s) {
        const bool in = s * 32 + quad * 8 < p.K;
        uint4 xv[4], av[NT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xv[i] = make_uint4(0u, 0u, 0u, 0u);
          if (in && (mine >> (row + 8 * i) & 1))
            xv[i] = *reinterpret_cast<const uint4*>(x + (row + 8 * i) * p.ldx + s * 32);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          av[j] = make_uint4(0u, 0u, 0u, 0u);
          if (in && r0 + j * 8 < p.rank)
            av[j] = __ldg(reinterpret_cast<const uint4*>(la + (size_t)(j * 8 + row) * p.K + s * 32));
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mma16816<T>(acc[i][j], xv[2 * i].x, xv[2 * i + 1].x, xv[2 * i].y, xv[2 * i + 1].y, av[j].x, av[j].y);
            mma16816<T>(acc[i][j], xv[2 * i].z, xv[2 * i + 1].z, xv[2 * i].w, xv[2 * i + 1].w, av[j].z, av[j].w);
          }
      }
      float* part = s_part + (size_t)warp * 32 * kR;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float* at = part + (16 * i + row) * kR + j * 8 + quad * 2;
          *reinterpret_cast<float2*>(at) = make_float2(acc[i][j][0], acc[i][j][1]);
          *reinterpret_cast<float2*>(at + 8 * kR) = make_float2(acc[i][j][2], acc[i][j][3]);
        }
      // the warps that share these rows meet; their parts are added in K order
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(kw * 32) : "memory");
      const float* parts0 = s_part + (size_t)group * kw * 32 * kR;
      const int r_left = min(kR, p.rank - r0);
      float* u = static_cast<float*>(p.ws) + ((size_t)blockIdx.z * p.rows + t0) * p.rank + r0;
      for (int e = kwarp * 32 + lane; e < 32 * kR; e += kw * 32) {
        const int t = e / kR, r = e % kR;
        if (!(mine >> t & 1) || r >= r_left) continue;
        float sum = 0.f;
        for (int k = 0; k < kw; ++k) sum += parts0[(size_t)k * 32 * kR + e];
        u[(size_t)t * p.rank + r] = sum;
      }
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(kw * 32) : "memory");
    }
  }
}

// ---------------------------------------------------------------------------
// Second launch: tiles of 128 weight rows x BT rows of x.  448 threads: warp 0 TMA, warp 1
// MMA, warps 2-5 U' of the slices, warps 6-13 epilogue (lane = weight row, so that 32 lanes
// write 64 consecutive bytes of an output row).  Up to one tile a CTA the accumulators
// are single, else double: the epilogue of a tile overlaps the next one's main loop.
// A ring stage holds 64 columns of W and x, or 4 slices of B_a and U'.
// ---------------------------------------------------------------------------
template <int BT>
struct GemmCfgA {
  static constexpr uint32_t kX = BT * 128;
  static constexpr uint32_t kStage = kWTile + kX;
  static constexpr int kStages = BT == 256 ? 4 : (BT == 128 ? 6 : (BT == 64 ? 8 : 9));
  static constexpr size_t kSmem = kStages * kStage + 512;
  static constexpr uint32_t kTmem = 2 * BT;
  static_assert(4 * kStages * 8 + 48 + 16 * 4 <= 512, "barriers");
  static_assert(kStages * kStage >= BT * 128 * 4, "the split-K exchange reuses the ring");
};
constexpr int kThreadsA = 448;

// Non-finite values of a 16-byte piece of B_a, which would reach every row of the tile as
// 0 * Inf: replaced by zeros here; the epilogue adds them to their own rows.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint4& v) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & kExp) == kExp) w[i] &= 0xffff0000u, found = true;
    if ((w[i] >> 16 & kExp) == kExp) w[i] &= 0x0000ffffu, found = true;
  }
  return found;
}

template <typename T, int BT>
__global__ void __launch_bounds__(kThreadsA, 1)
    adapter_gemm_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                        const __grid_constant__ CUtensorMap bmap, const __grid_constant__ AdapterGemmParams p,
                        const __grid_constant__ Plan pl) {
  using C = GemmCfgA<BT>;
  constexpr uint32_t kIsBf16 = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStage);
  uint64_t* empty = full + C::kStages;
  uint64_t* u_go = empty + C::kStages;    // [stages] the stage is free for U' (producer)
  uint64_t* u_full = u_go + C::kStages;   // [stages] U' written, B_a's slices landed
  uint64_t* acc_full = u_full + C::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [tile count % 16] = tile count + 1 where values of B_a were left out (U' runs ahead of
  // the epilogue by fewer tiles than the ring has stages, plus the two accumulators)
  volatile int* s_dropped = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = pl.split > 1 ? (int)cluster_ctarank() : 0;
  const int tile0 = pl.split > 1 ? blockIdx.x / pl.split : blockIdx.x;
  const int step = pl.split > 1 ? pl.tiles * pl.n_tiles : gridDim.x;
  const int total = pl.tiles * pl.n_tiles;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&u_go[i], 1);
      mbar_init(&u_full[i], 128);
    }
    for (int i = 0; i < 16; ++i) s_dropped[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 256);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&xmap);
    tma_prefetch_desc(&wmap);
    tma_prefetch_desc(&bmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The first launch may still run: what reads its results waits for it first.  Plain loads
  // (not the read-only path, which may hold older values).
  const int* lists = reinterpret_cast<const int*>(static_cast<const uint8_t*>(p.ws) + list_offset(p, pl));
  const int kb0 = pl.kblocks * rank / pl.split, kb1 = pl.kblocks * (rank + 1) / pl.split;
  // this CTA's slices of a tile whose list is `list`
  auto slice_range = [&](const int* list, int& s0, int& s1) {
    const int n = list[0] * pl.chunks;
    s0 = n * rank / pl.split;
    s1 = n * (rank + 1) / pl.split;
  };

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < total; tile += step) {
        const int tt = tile / pl.n_tiles, n0 = (tile - tt * pl.n_tiles) * 128;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % C::kStages;
          if (!mbar_wait(&empty[st], ((it / C::kStages) & 1) ^ 1, kErrTimeoutSmemEmpty, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + st * C::kStage;
          mbar_arrive_expect_tx(&full[st], kWTile + (uint32_t)pl.x_box * 128u);
          tma_load_2d(dst, &wmap, &full[st], kb * 64, n0);
          tma_load_2d(dst + kWTile, &xmap, &full[st], kb * 64, tt * BT);
        }
        // the lists are the first launch's: wait for it only now that W and x are on their way
        if (tile == tile0) wait_for_previous();
        const int* list = lists + (size_t)tt * pl.list_ld;
        int s0, s1;
        slice_range(list, s0, s1);
        for (; ok && s0 < s1; s0 += 4, ++it) {
          const int st = it % C::kStages, n = min(4, s1 - s0);
          if (!mbar_wait(&empty[st], ((it / C::kStages) & 1) ^ 1, kErrTimeoutSmemEmpty, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive(&u_go[st]);
          mbar_arrive_expect_tx(&full[st], (uint32_t)n * 4096u);
          for (int i = 0; i < n; ++i)
            tma_load_3d(smem + st * C::kStage + i * 4096, &bmap, &full[st], ((s0 + i) % pl.chunks) * kSliceRows, n0,
                        list[2 + (s0 + i) / pl.chunks]);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_f16(kIsBf16, BT, 0);
      int it = 0, n = 0;
      uint32_t uses = 0;  // parity of each stage's uses for slices
      bool ok = true;
      for (int tile = tile0; ok && tile < total; tile += step, ++n) {
        const int tt = tile / pl.n_tiles, buf = n & 1;
        const uint32_t acc = tmem + (uint32_t)(buf * BT);
        if (!mbar_wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1, kErrTimeoutTmemEmpty, abort_flag)) break;
        tc_fence_after();
        int s0, s1;
        if (n > 0) slice_range(lists + (size_t)tt * pl.list_ld, s0, s1);  // fetched ahead of its use
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % C::kStages;
          if (!mbar_wait(&full[st], (it / C::kStages) & 1, kErrTimeoutTmaFull, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t dw = sw128_desc(smem_u32(smem + st * C::kStage), 16, 1024);
          const uint64_t dx = sw128_desc(smem_u32(smem + st * C::kStage + kWTile), 16, 1024);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16_ss(acc, dw + 2 * kk, dx + 2 * kk, idesc, kb > kb0 || kk > 0);
          umma_commit(&empty[st]);
        }
        if (n == 0) {
          wait_for_previous();
          slice_range(lists + (size_t)tt * pl.list_ld, s0, s1);
        }
        for (; ok && s0 < s1; s0 += 4, ++it) {
          const int st = it % C::kStages, m = min(4, s1 - s0);
          if (!mbar_wait(&u_full[st], uses >> st & 1, kErrTimeoutTmaFull, abort_flag)) {
            ok = false;
            break;
          }
          uses ^= 1u << st;
          tc_fence_after();
          const uint64_t dw = sw32_desc(smem_u32(smem + st * C::kStage));
          const uint64_t dx = sw32_desc(smem_u32(smem + st * C::kStage + kWTile));
          for (int i = 0; i < m; ++i)
            umma_f16_ss(acc, dw + (uint64_t)(i * (4096 >> 4)), dx + (uint64_t)(i * (BT * 32 >> 4)), idesc, 1u);
          umma_commit(&empty[st]);
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------ U' of the slices
    // These warps follow the ring by its slice stages alone: a stage is theirs once the
    // producer says so, and is not used again before the MMA has had their U'.
    // A thread writes rows i0 and i0 + 128 of all slices.  Their values are fetched and
    // rounded before the stage is waited for, so that the wait covers the loads.
    constexpr int kPer = BT > 128 ? 2 : 1;
    const int i0 = threadIdx.x - 64;
    int it = 0, n = 0;
    uint32_t uses = 0;
    bool ok = true;
    const size_t part = (size_t)p.rows * p.rank;
    wait_for_previous();
    for (int tile = tile0; ok && tile < total; tile += step, ++n) {
      const int tt = tile / pl.n_tiles;
      const int* list = lists + (size_t)tt * pl.list_ld;
      int s0, s1;
      slice_range(list, s0, s1);
      it += kb1 - kb0;
      int id[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) id[e] = row_id(p, (long long)tt * BT + i0 + e * 128);
      for (; s0 < s1; s0 += 4, ++it) {
        const int st = it % C::kStages, m = min(4, s1 - s0);
        uint4 v[kPer][4][2];  // [row][slice][8 values]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int s = s0 + i, a = i < m ? list[2 + s / pl.chunks] : -2, c0 = (s % pl.chunks) * kSliceRows;
#pragma unroll
          for (int e = 0; e < kPer; ++e)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              v[e][i][half] = make_uint4(0u, 0u, 0u, 0u);
              if (id[e] != a || c0 + half * 8 >= p.rank) continue;
              const float* u = static_cast<const float*>(p.ws) + ((size_t)tt * BT + i0 + e * 128) * p.rank + c0 + half * 8;
              float4 lo = *reinterpret_cast<const float4*>(u), hi = *reinterpret_cast<const float4*>(u + 4);
              for (int k = 1; k < pl.down_split; ++k) {
                u += part;
                const float4 l2 = *reinterpret_cast<const float4*>(u), h2 = *reinterpret_cast<const float4*>(u + 4);
                lo = make_float4(lo.x + l2.x, lo.y + l2.y, lo.z + l2.z, lo.w + l2.w);
                hi = make_float4(hi.x + h2.x, hi.y + h2.y, hi.z + h2.z, hi.w + h2.w);
              }
              const float sc = p.scales ? __ldg(p.scales + a) : 1.f;
              v[e][i][half] = make_uint4(pack2<T>(lo.x * sc, lo.y * sc), pack2<T>(lo.z * sc, lo.w * sc),
                                         pack2<T>(hi.x * sc, hi.y * sc), pack2<T>(hi.z * sc, hi.w * sc));
            }
        }
        if (!mbar_wait(&u_go[st], uses >> st & 1, kErrTimeoutSmemEmpty, abort_flag)) {
          ok = false;
          break;
        }
        uses ^= 1u << st;
        uint8_t* base = smem + st * C::kStage;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < kPer; ++e)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int r = i0 + e * 128;
              if (i < m && r < BT)
                *reinterpret_cast<uint4*>(base + kWTile + i * (BT * 32) + r * 32 + ((half ^ (r >> 2 & 1)) << 4)) =
                    v[e][i][half];
            }
        if (!mbar_wait(&full[st], (it / C::kStages) & 1, kErrTimeoutTmaFull, abort_flag)) {
          ok = false;
          break;
        }
        if (list[1]) {
          for (int x = i0; x < m * 256; x += 128) {
            uint4* at = reinterpret_cast<uint4*>(base + x * 16);
            uint4 v = *at;
            if (drop_nonfinite<T>(v)) {
              *at = v;
              s_dropped[n & 15] = n + 1;
            }
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(&u_full[st]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 6) >> 2;
    int n = 0;
    wait_for_previous();
    for (int tile = tile0; tile < total; tile += step, ++n) {
      const int tt = tile / pl.n_tiles, buf = n & 1;
      const int col = (tile - tt * pl.n_tiles) * 128 + q * 32 + lane;  // output column
      const long long t0 = (long long)tt * BT;
      const bool in = col < p.N;
      const float bias = in && p.bias && rank == 0 ? __ldg(p.bias + col) : 0.f;
      if (!mbar_wait(&acc_full[buf], (n >> 1) & 1, kErrTimeoutTmemFull, abort_flag)) break;
      tc_fence_after();
      const bool dropped = s_dropped[n & 15] == n + 1;
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BT);
      constexpr int kCols = BT >= 64 ? BT / 2 : BT;  // columns of this warp
      if (BT >= 64 || half == 0) {
        for (int c = half * kCols; c < (half + 1) * kCols; c += 32) {
          uint32_t v[32];
          tmem_ld32(acc + (uint32_t)c, v);
          tmem_ld_wait(v);
          if (dropped && in) {
            // the values left out of B_a, into the rows that have the adapter
            const int* list = lists + (size_t)tt * pl.list_ld;
            int s0, s1;
            slice_range(list, s0, s1);
            for (int s = s0; s < s1; ++s) {
              const int a = list[2 + s / pl.chunks];
              const int c0 = (s % pl.chunks) * kSliceRows, c1 = min(c0 + kSliceRows, p.rank);
              const T* bw = static_cast<const T*>(p.lora_b) + ((size_t)a * p.N + col) * p.rank;
              for (int r = c0; r < c1; ++r) {
                const float bv = to_f32(bw[r]);
                if (isfinite(bv)) continue;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (row_id(p, t0 + c + i) == a) {
                    float u = 0.f;
                    for (int k = 0; k < pl.down_split; ++k)
                      u += static_cast<const float*>(p.ws)[((size_t)k * p.rows + t0 + c + i) * p.rank + r];
                    u = to_f32(from_f32<T>(u * (p.scales ? __ldg(p.scales + a) : 1.f)));
                    v[i] = __float_as_uint(__uint_as_float(v[i]) + u * bv);
                  }
              }
            }
          }
          if (pl.split > 1) {
            float* ex = reinterpret_cast<float*>(smem) + c * 128 + q * 32 + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i) ex[i * 128] = __uint_as_float(v[i]) + bias;
          } else if (in) {
            T* out = static_cast<T*>(p.out) + (t0 + c) * p.ldo + col;
            const int left = (int)min(32LL, p.rows - (t0 + c));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < left) out[i * p.ldo] = from_f32<T>(__uint_as_float(v[i]) + bias);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[buf]);
    }
  }

  if (pl.split > 1) {
    // every CTA of the cluster adds up its share of the tile's rows, in rank order
    __syncwarp();
    cluster_sync_all();
    const int tt = tile0 / pl.n_tiles, n0 = (tile0 - tt * pl.n_tiles) * 128;
    const int r0 = BT * rank / pl.split, r1 = BT * (rank + 1) / pl.split;
    const uint32_t base = smem_u32(smem);
    for (int x = threadIdx.x; x < (r1 - r0) * 32; x += kThreadsA) {
      const int r = r0 + (x >> 5), c = (x & 31) * 4;
      const long long t = (long long)tt * BT + r;
      if (t >= p.rows || n0 + c >= p.N) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < pl.split; ++k) {
        float4 v;
        const uint32_t at = mapa_shared(base + (uint32_t)(r * 128 + c) * 4u, (uint32_t)k);
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "r"(at)
                     : "memory");
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + t * p.ldo + n0 + c) =
          make_uint2(pack2<T>(sum.x, sum.y), pack2<T>(sum.z, sum.w));
    }
    __syncwarp();
    cluster_sync_all();  // the parts stay until all have read them
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

Plan make_plan(int rows, int K, int N, int adapters, int rank, int num_sms) {
  Plan pl{};
  pl.bt = rows <= 32 ? 32 : (rows <= 64 ? 64 : (rows <= 128 ? 128 : 256));
  pl.tiles = (rows + pl.bt - 1) / pl.bt;
  pl.n_tiles = (N + 127) / 128;
  pl.kblocks = (K + 63) / 64;
  pl.chunks = (rank + kSliceRows - 1) / kSliceRows;
  // first launch: at least 4 K steps of 32 a warp, about two CTAs an SM
  const int steps = (K + 31) / 32;
  pl.down_kw = 1;
  while (pl.down_kw < 8 && pl.down_kw * 2 * 4 <= steps) pl.down_kw *= 2;
  const int rows_cta = 32 * (8 / pl.down_kw);
  pl.down_x = adapters ? (rows + rows_cta - 1) / rows_cta : 0;
  const int want = 2 * num_sms;
  pl.down_split = std::max(1, std::min({want / std::max(pl.down_x, 1), 8, steps / (pl.down_kw * 4)}));
  pl.down_y = std::max(1, std::min({want / std::max(pl.down_x * pl.down_split, 1), 32, adapters}));
  pl.down_nt = rank <= 8 ? 1 : (rank <= 16 ? 2 : (rank <= 32 ? 4 : 8));
  pl.split = 1;
  while (pl.split < 8 && (long long)pl.tiles * pl.n_tiles * pl.split * 2 <= num_sms && pl.split * 2 <= pl.kblocks)
    pl.split *= 2;
  pl.x_box = std::min(pl.bt, (rows + 7) / 8 * 8);
  pl.list_ld = (pl.bt + 2 + 3) / 4 * 4;
  return pl;
}

// 16-bit [count, rows, cols] in boxes of box_cols x box_rows
CUtensorMap map_3d(const void* base, uint64_t cols, uint64_t rows, uint64_t count, uint32_t box_cols,
                   uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  const uint64_t dims[3] = {cols, rows, count};
  const uint64_t strides[2] = {cols * 2, cols * rows * 2};
  const uint32_t box[3] = {box_cols, box_rows, 1};
  return make_tensor_map(base, 3, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_UINT16, swizzle);
}

template <typename T, int NT>
cudaError_t launch_down(const AdapterGemmParams& p, const Plan& pl, cudaStream_t s) {
  static std::atomic<unsigned long long> configured;
  constexpr int smem = 8 * 32 * NT * 8 * (int)sizeof(float);
  cudaError_t e = ensure_smem_limit(adapter_down_kernel<T, NT>, smem, configured);
  if (e != cudaSuccess) return e;
  const double m = p.rows, k = p.K, r = p.rank;
  LaunchScope scope("adapter_down", 2.0 * m * r * k, 2.0 * (m * k + p.adapters * r * k) + 4.0 * m * r, s);
  adapter_down_kernel<T, NT><<<dim3(pl.down_x + pl.tiles, pl.down_y, pl.down_split), 256, smem, s>>>(p, pl);
  return cudaGetLastError();
}

template <typename T, int BT>
cudaError_t launch_bt(const AdapterGemmParams& p, const Plan& pl, int num_sms, cudaStream_t s) {
  static std::atomic<unsigned long long> configured;
  cudaError_t e = ensure_smem_limit(adapter_gemm_kernel<T, BT>, (int)GemmCfgA<BT>::kSmem, configured);
  if (e != cudaSuccess) return e;
  const double m = p.rows, k = p.K, n = p.N, r = p.rank;
  const CUtensorMap mx = map_2d(p.x, (uint64_t)p.rows, (uint64_t)p.K, (uint64_t)p.ldx, (uint32_t)pl.x_box);
  const CUtensorMap mw = map_2d(p.w, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)p.K, 128);
  // without adapters no row has one and the map is not read
  const CUtensorMap mb = p.adapters ? map_3d(p.lora_b, (uint64_t)p.rank, (uint64_t)p.N, (uint64_t)p.adapters,
                                             kSliceRows, 128, CU_TENSOR_MAP_SWIZZLE_32B)
                                    : mx;
  e = pl.down_nt == 1   ? launch_down<T, 1>(p, pl, s)
      : pl.down_nt == 2 ? launch_down<T, 2>(p, pl, s)
      : pl.down_nt == 4 ? launch_down<T, 4>(p, pl, s)
                        : launch_down<T, 8>(p, pl, s);
  if (e != cudaSuccess) return e;
  LaunchScope scope("adapter_gemm", 2.0 * m * n * (k + r), 2.0 * (m * k + n * k + m * n + p.adapters * r * n), s);
  const long long tiles = (long long)pl.tiles * pl.n_tiles;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(pl.split > 1 ? tiles * pl.split : std::min<long long>(tiles, num_sms)));
  cfg.blockDim = dim3(kThreadsA);
  cfg.dynamicSmemBytes = GemmCfgA<BT>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)pl.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = pl.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, adapter_gemm_kernel<T, BT>, mx, mw, mb, p, pl);
}

template <typename T>
cudaError_t launch_t(const AdapterGemmParams& p, int num_sms, cudaStream_t s) {
  if (p.rows == 0) return cudaSuccess;
  const Plan pl = make_plan(p.rows, p.K, p.N, p.adapters, p.rank, num_sms);
  switch (pl.bt) {
    case 32:
      return launch_bt<T, 32>(p, pl, num_sms, s);
    case 64:
      return launch_bt<T, 64>(p, pl, num_sms, s);
    case 128:
      return launch_bt<T, 128>(p, pl, num_sms, s);
    default:
      return launch_bt<T, 256>(p, pl, num_sms, s);
  }
}

}  // namespace

long long adapter_gemm_workspace(int rows, int K, int N, int adapters, int rank, int num_sms) {
  if (rows == 0) return 0;
  const Plan pl = make_plan(rows, K, N, adapters, rank, num_sms);
  return (long long)pl.down_split * rows * rank * 4 + (long long)pl.tiles * pl.list_ld * 4;
}

cudaError_t launch_adapter_gemm(const AdapterGemmParams& p, int bf16, int num_sms, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, num_sms, stream) : launch_t<__half>(p, num_sms, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(adapter_gemm_device_error)

}  // namespace msst
