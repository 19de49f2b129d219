// adapter_gemm.cu — a shared projection with the low-rank adapters of many requests
// beside it: y[t] = W x[t] + bias + s_a B_a (A_a x[t]), a = row_adapter[t].
//
// Two launches.  adapter_down_kernel computes u[t] = A_a x[t] for every row that has an
// adapter; adapter_gemm_kernel computes W x and adds B_a (s_a u) as a few more K steps
// of the same accumulators, so the low-rank term costs no pass over the output.
//
// The second works on row tiles (32, 64 or 128 rows) and on the list of the distinct adapters
// of a tile.  An adapter's part of the extra K steps is a slice of 16 rank values
// (ceil(rank / 16) slices an adapter): B_a's columns on one side, on the other U', which
// holds s_a u for the rows whose adapter is a and zeros for all others.  So requests
// may be mixed row by row: a tile costs as many slices as it has adapters.
//
// Which side of the MMA the rows take, and the split along K: make_plan.
//
// u is rounded to the operands' 16 bits once, as U' feeds the tensor cores; it is summed
// in fp32 before that (split-K parts of the first launch in order).  What U' cannot hold in fp16,
// the part of s_a u beyond +-65504, is multiplied by B_a in fp32 and added to the accumulators by
// the epilogue, before the one rounding of y; so are products of B_a's infinities and NaN, which
// would reach other rows of a tile as 0 * Inf.  Both are rare and slow: left_out.
#include <algorithm>

#include "common.cuh"
#include "operators.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr int kSliceRows = 16;               // rank values of a slice

// The plan of a call, the same for both launches.
struct Plan {
  int rows_on_m;    // second launch: rows of x on the MMA's M side
  int bt;           // rows of x a tile
  int tiles;        // ceil(rows / bt)
  int n_tiles;      // ceil(N / weight rows a tile)
  int kblocks;      // ceil(K / 64)
  int chunks;       // slices an adapter
  // first launch: CTAs along the rows (of 32 * kDownWarps / down_kw rows), along a tile's adapters and
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
// mma.sync m16n8k16; each warp streams its rows through a ring of its own in shared memory
// (cp.async, whole 128-byte lines, three stages of 64 columns in flight: 144 KB an SM with the three CTAs
// that fit up to rank 16, 96 KB with two above, whose accumulators take 202 and 252 registers) and
// takes A_a, which stays in L2, straight from global memory one step ahead.  No barrier
// until the end.  8192 rows of 4096 columns, rank 32: 40 us alone, about half of it under the
// second launch (188 alone, 210 to 214 for both); 32 rows, 16 adapters: 10 us.  (Forms that held x in registers kept too little in flight: 37 us for
// 8192 rows of 4096 columns; a tcgen05 form with 128-row slices of A_a took 35 us.)
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
  __shared__ int s_id[128], s_count[4], s_mixed;
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
  for (int x = 0; x < 4; ++x) {
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}

constexpr int kDownWarps = 4;
constexpr int kDownStages = 4;
constexpr uint32_t kDownStage = 32 * 128;  // 32 rows x 64 columns
constexpr int kDownSmem = kDownWarps * kDownStages * (int)kDownStage;  // 64 KB: up to three CTAs an SM

template <typename T, int NT>
__global__ void __launch_bounds__(32 * kDownWarps)
    adapter_down_kernel(const __grid_constant__ AdapterGemmParams p, const __grid_constant__ Plan pl) {
  extern __shared__ __align__(128) uint8_t s_ring[];  // [warps][stages][32 rows][128 bytes]
  dependents_may_start();
  if (blockIdx.x >= pl.down_x) {
    if (blockIdx.y == 0 && blockIdx.z == 0) write_list(p, pl, blockIdx.x - pl.down_x);
    return;
  }
  constexpr int kR = NT * 8;
  static_assert(32 * kR * 4 <= kDownStages * kDownStage, "the results reuse the ring");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kw = pl.down_kw, kwarp = warp % kw, group = warp / kw;
  const long long t0 = ((long long)blockIdx.x * (kDownWarps / kw) + group) * 32;
  if (t0 >= p.rows) return;
  const int id = row_id(p, t0 + lane);
  const unsigned same = __match_any_sync(0xffffffffu, id);
  unsigned firsts = __ballot_sync(0xffffffffu, id >= 0 && __ffs(same) - 1 == lane);
  const int steps = (p.K + 63) / 64, parts = pl.down_split * kw, me = blockIdx.z * kw + kwarp;
  const int s0 = (int)((long long)steps * me / parts), s1 = (int)((long long)steps * (me + 1) / parts);
  const int row = lane >> 2, quad = lane & 3;
  uint8_t* ring = s_ring + (size_t)warp * kDownStages * kDownStage;
  const uint32_t ring_u = smem_u32(ring);
  // copies: 8 lanes a row's 128 bytes; pieces of odd rows swap halves, so that the reads
  // below (8 rows x 4 pieces at a time) meet no bank twice
  const int crow = lane >> 3, cpiece = lane & 7;
  for (int li = 0; firsts; ++li, firsts &= firsts - 1) {
    if (li % pl.down_y != blockIdx.y) continue;
    const int src = __ffs(firsts) - 1;
    const int a = __shfl_sync(0xffffffffu, id, src);
    const unsigned mine = __shfl_sync(0xffffffffu, same, src);  // the rows that have adapter a
    for (int r0 = 0; r0 < p.rank; r0 += kR) {
      auto fetch = [&](int s) {
        if (s < s1) {
          const uint32_t dst = ring_u + (uint32_t)(s % kDownStages) * kDownStage;
          const T* x = static_cast<const T*>(p.x) + t0 * p.ldx + s * 64 + cpiece * 8;
          const bool in = s * 64 + cpiece * 8 < p.K;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + crow;
            const bool take = in && (mine >> r & 1);
            cp_async16(dst + (uint32_t)(r * 128 + ((cpiece ^ (r & 1) << 2) << 4)), take ? x + r * p.ldx : p.x, take);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const T* la = static_cast<const T*>(p.lora_a) + ((size_t)a * p.rank + r0 + row) * p.K + quad * 8;
      // this lane's 8 columns of each 32 of step s, rank values j * 8 + row
      auto load_a = [&](int s, uint4 (&v)[2][NT]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            v[h][j] = make_uint4(0u, 0u, 0u, 0u);
            if (s < s1 && s * 64 + h * 32 + quad * 8 < p.K && r0 + j * 8 < p.rank)
              v[h][j] = __ldg(reinterpret_cast<const uint4*>(la + (size_t)j * 8 * p.K + s * 64 + h * 32));
          }
      };
      float acc[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2 * NT * 4; ++i) (&acc[0][0][0])[i] = 0.f;
#pragma unroll
      for (int i = 0; i < kDownStages - 1; ++i) fetch(s0 + i);
      uint4 next[2][NT];
      load_a(s0, next);
      for (int s = s0; s < s1; ++s) {
        uint4 av[2][NT];
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) (&av[0][0])[i] = (&next[0][0])[i];
        load_a(s + 1, next);
        asm volatile("cp.async.wait_group %0;" ::"n"(kDownStages - 2) : "memory");
        __syncwarp();
        const uint8_t* st = ring + (s % kDownStages) * kDownStage;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 xv[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            xv[i] = *reinterpret_cast<const uint4*>(st + (row + 8 * i) * 128 + (((h * 4 + quad) ^ (row & 1) << 2) << 4));
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 &x0 = xv[2 * i], &x1 = xv[2 * i + 1], &w = av[h][j];
              mma16816<T>(acc[i][j], x0.x, x1.x, x0.y, x1.y, w.x, w.y);
              mma16816<T>(acc[i][j], x0.z, x1.z, x0.w, x1.w, w.z, w.w);
            }
        }
        __syncwarp();
        fetch(s + kDownStages - 1);  // into the stage read in the last step
      }
      float* part = reinterpret_cast<float*>(ring);
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
      const int r_left = min(kR, p.rank - r0);
      float* u = static_cast<float*>(p.ws) + ((size_t)blockIdx.z * p.rows + t0) * p.rank + r0;
      for (int e = kwarp * 32 + lane; e < 32 * kR; e += kw * 32) {
        const int t = e / kR, r = e % kR;
        if (!(mine >> t & 1) || r >= r_left) continue;
        float sum = 0.f;
        for (int k = 0; k < kw; ++k)
          sum += reinterpret_cast<const float*>(s_ring + (size_t)(group * kw + k) * kDownStages * kDownStage)[e];
        u[(size_t)t * p.rank + r] = sum;
      }
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(kw * 32) : "memory");
    }
  }
}

// ---------------------------------------------------------------------------
// Second launch: tiles of 128 on the M side by BT on the N side.  kRowsOnM: rows of x by
// weight rows, else weight rows by rows of x.  448 threads: warp 0 TMA, warp 1 MMA, warps 2-5
// U' of the slices, warps 6-13 epilogue.  The accumulators are double: the epilogue of a
// tile overlaps the next one's main loop.  A ring stage holds 64 columns of W and x, or 4
// slices of B_a and U'.
// Bound: the tensor cores for large K (8192 rows, K = N = 4096: 210 to 214 us with the first
// launch, 1320 TFLOP/s); 48060 rows, K = 384, N = 1536: 71 to 74 us (2.55 TB/s), 64 of them this one's, tensor pipe
// 51 % busy; latency for few rows (32 rows, 16 adapters, K = N = 4096: 20 us).
// ---------------------------------------------------------------------------
constexpr uint32_t kMTile = 128 * 128;       // the M side: 128 rows x 64 columns of 16 bits

template <int BT, bool kRowsOnM>
struct GemmCfgA {
  static constexpr int kRows = kRowsOnM ? 128 : BT, kCols = kRowsOnM ? BT : 128;
  static constexpr uint32_t kStage = kMTile + BT * 128;
  static constexpr int kStages = BT == 256 ? 4 : (BT == 128 ? 6 : (BT == 64 ? 8 : 9));
  // a slice (32 bytes a row) and where the slices of U' and B_a lie in a stage
  static constexpr uint32_t kUSlice = kRows * 32, kBSlice = kCols * 32;
  static constexpr uint32_t kUAt = kRowsOnM ? 0 : kMTile, kBAt = kRowsOnM ? kMTile : 0;
  static constexpr uint32_t kStaging = kRowsOnM ? 8 * 2048 : 0;  // 32 x 32 outputs a warp
  static constexpr size_t kSmem = kStages * kStage + kStaging + 512;
  static constexpr uint32_t kTmem = 2 * BT;
  static_assert(4 * kStages * 8 + 56 + 16 * 4 <= 512, "barriers");
  static_assert(kRowsOnM || kStages * kStage >= BT * 128 * 4, "the split-K exchange reuses the ring");
};
constexpr int kThreadsA = 448;

// The exponent of a 16-bit type's infinities and NaN; its largest magnitude is one below.
template <typename T>
constexpr uint32_t kExpBits = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
// Non-finite values of a 16-byte piece of B_a, which would reach every row of the tile as
// 0 * Inf: replaced by zeros here; the epilogue adds them to their own rows.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint4& v) {
  constexpr uint32_t kExp = kExpBits<T>;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & kExp) == kExp) w[i] &= 0xffff0000u, found = true;
    if ((w[i] >> 16 & kExp) == kExp) w[i] &= 0x0000ffffu, found = true;
  }
  return found;
}
// 16-bit maxima of the magnitudes of a piece's 8 values: at or above kExp where one is not finite.
__device__ __forceinline__ uint32_t magnitudes(const uint4& v) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(v.x & kAbs, v.y & kAbs), __vmaxu2(v.z & kAbs, v.w & kAbs));
}

// The next four slices of a tile's list: adapter (-2 past the end) and slice of that adapter.
// Read a stage ahead by counting: with two divisions and a wait for the list at every slice, in the
// one producing thread, a slice took about 0.5 us instead of 0.2 (32 rows, K = N = 4096).
struct Slices {
  const int* at;
  int c, chunks, left;
  int id[4], part[4];
  __device__ __forceinline__ Slices(const int* list, int s0, int s1, int n) : chunks(n), left(s1 - s0) {
    at = list + 2 + s0 / n;
    c = s0 % n;
    next();
  }
  __device__ __forceinline__ void next() {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      id[i] = left > 0 ? *at : -2;
      part[i] = c;
      --left;
      if (++c == chunks) c = 0, ++at;
    }
  }
};

// s_a u as U' holds it: rounded, the largest finite value where that gives an infinity.
template <typename T>
__device__ __forceinline__ bool clamp_infinities(uint4& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7fffu) == kExpBits<T>) w[i] -= 1u, found = true;
    if ((w[i] >> 16 & 0x7fffu) == kExpBits<T>) w[i] -= 0x10000u, found = true;
  }
  return found;
}

// What the operands of slices [s0, s1) of the tile's list leave out of y[t, col]: the products of the
// part of s_a u beyond what U' holds, and, where the tile's rows differ (`mixed`), those of the values
// that drop_nonfinite took out of B_a.
template <typename T>
__device__ __forceinline__ float left_out(const AdapterGemmParams& p, const Plan& pl, const int* list, int s0, int s1,
                                          bool mixed, long long t, int col) {
  const int a = row_id(p, t);
  float sum = 0.f;
  if (a < 0 || col >= p.N) return sum;
  const float sc = p.scales ? __ldg(p.scales + a) : 1.f;
  const T* bw = static_cast<const T*>(p.lora_b) + ((size_t)a * p.N + col) * p.rank;
  const float* u0 = static_cast<const float*>(p.ws) + t * p.rank;
  for (int s = s0; s < s1; ++s) {
    if (list[2 + s / pl.chunks] != a) continue;
    const int c0 = (s % pl.chunks) * kSliceRows, c1 = min(c0 + kSliceRows, p.rank);
    for (int r = c0; r < c1; ++r) {
      float u = 0.f;
      for (int k = 0; k < pl.down_split; ++k) u += u0[(size_t)k * p.rows * p.rank + r];
      u *= sc;
      const float bv = to_f32(bw[r]);
      if (mixed && !isfinite(bv)) {
        sum += u * bv;
      } else if (isinf(to_f32(from_f32<T>(u)))) {
        const float most = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
        sum += (u - copysignf(most, u)) * bv;
      }
    }
  }
  return sum;
}

// Adds it to the accumulators of columns [c, c_end) of this warp's lanes, at `acc` + c: lane the row t
// and column the output column col + c (kRowsOnM), or lane the output column and column the row t + c.
template <typename T, bool kRowsOnM>
__device__ __noinline__ void add_left_out(const AdapterGemmParams& p, const Plan& pl, const int* list, int s0, int s1,
                                          long long t, int col, uint32_t acc, int c, int c_end) {
  for (; c < c_end; ++c) {
    const float x = left_out<T>(p, pl, list, s0, s1, list[1] != 0, kRowsOnM ? t : t + c, kRowsOnM ? col + c : col);
    if (__any_sync(0xffffffffu, x != 0.f)) {
      const float y = __uint_as_float(tmem_ld1(acc + (uint32_t)c));
      tmem_st1(acc + (uint32_t)c, __float_as_uint(x != 0.f ? y + x : y));
    }
  }
}

template <typename T, int BT, bool kRowsOnM>
__global__ void __launch_bounds__(kThreadsA, 1)
    adapter_gemm_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                        const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap omap,
                        const __grid_constant__ AdapterGemmParams p, const __grid_constant__ Plan pl) {
  using C = GemmCfgA<BT, kRowsOnM>;
  constexpr uint32_t kIsBf16 = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* staging = smem + C::kStages * C::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::kStaging);
  uint64_t* empty = full + C::kStages;
  uint64_t* u_go = empty + C::kStages;    // [stages] the stage is free for U' (producer)
  uint64_t* u_full = u_go + C::kStages;   // [stages] U' written, B_a's slices landed
  uint64_t* acc_full = u_full + C::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2]
  uint64_t* mma_end = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_end + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [tile count % 16] = tile count + 1 where the operands leave products out (written behind the ring,
  // so ahead of the epilogue by fewer tiles than the ring has stages, plus the two accumulators)
  volatile int* s_left_out = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = kRowsOnM ? 1 : pl.split;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int total = pl.tiles * pl.n_tiles;
  const int tile0 = split > 1 ? blockIdx.x / split : blockIdx.x;
  const int step = split > 1 ? total : gridDim.x;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&u_go[i], 1);
      mbar_init(&u_full[i], 128);
    }
    for (int i = 0; i < 16; ++i) s_left_out[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 256);
    }
    mbar_init(mma_end, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&xmap);
    tma_prefetch_desc(&wmap);
    tma_prefetch_desc(&bmap);
    tma_prefetch_desc(&omap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The first launch may still run: what reads its results waits for it first.
  const int* lists = reinterpret_cast<const int*>(static_cast<const uint8_t*>(p.ws) + list_offset(p, pl));
  const int kb0 = pl.kblocks * rank / split, kb1 = pl.kblocks * (rank + 1) / split;
  // this CTA's slices of a tile whose list is `list`
  auto slice_range = [&](const int* list, int& s0, int& s1) {
    const int n = list[0] * pl.chunks;
    s0 = n * rank / split;
    s1 = n * (rank + 1) / split;
  };

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      const uint32_t bytes = (uint32_t)(pl.x_box + C::kCols) * 128u;
      for (int tile = tile0; ok && tile < total; tile += step) {
        const int tt = tile / pl.n_tiles, n0 = (tile - tt * pl.n_tiles) * C::kCols;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % C::kStages;
          if (!mbar_wait(&empty[st], ((it / C::kStages) & 1) ^ 1, kErrTimeoutSmemEmpty, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + st * C::kStage;
          mbar_arrive_expect_tx(&full[st], bytes);
          tma_load_2d(dst + C::kBAt, &wmap, &full[st], kb * 64, n0);
          tma_load_2d(dst + C::kUAt, &xmap, &full[st], kb * 64, tt * C::kRows);
        }
        // the lists are the first launch's: wait for it only now that W and x are on their way
        if (tile == tile0) wait_for_previous();
        const int* list = lists + (size_t)tt * pl.list_ld;
        int s0, s1;
        slice_range(list, s0, s1);
        Slices sl(list, s0, s1, pl.chunks);
        for (; ok && s0 < s1; s0 += 4, ++it, sl.next()) {
          const int st = it % C::kStages, n = min(4, s1 - s0);
          if (!mbar_wait(&empty[st], ((it / C::kStages) & 1) ^ 1, kErrTimeoutSmemEmpty, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive(&u_go[st]);
          mbar_arrive_expect_tx(&full[st], (uint32_t)n * C::kBSlice);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < n)
              tma_load_3d(smem + st * C::kStage + C::kBAt + i * C::kBSlice, &bmap, &full[st], sl.part[i] * kSliceRows,
                          n0, sl.id[i]);
        }
      }
      mbar_drain_ring(full, C::kStages, it % C::kStages, it / C::kStages & 1);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = umma_idesc_f16(kIsBf16, BT, 0);
      int it = 0, n = 0;
      uint32_t uses = 0;  // parity of each stage's uses for slices
      bool ok = true;
      for (int tile = tile0; ok && tile < total; tile += step, ++n) {
        const int tt = tile / pl.n_tiles, buf = n & 1;
        const uint32_t acc = tmem + (uint32_t)(buf * BT);
        if (!mbar_wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1, kErrTimeoutTmemEmpty, abort_flag)) break;
        tc_fence_after();
        int s0 = 0, s1 = 0;
        if (n > 0) slice_range(lists + (size_t)tt * pl.list_ld, s0, s1);  // fetched ahead of its use
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % C::kStages;
          if (!mbar_wait(&full[st], (it / C::kStages) & 1, kErrTimeoutTmaFull, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t dm = sw128_desc(smem_u32(smem + st * C::kStage), 16, 1024);
          const uint64_t dn = sw128_desc(smem_u32(smem + st * C::kStage + kMTile), 16, 1024);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16_ss(acc, dm + 2 * kk, dn + 2 * kk, idesc, kb > kb0 || kk > 0);
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
          const uint64_t dm = sw32_desc(smem_u32(smem + st * C::kStage));
          const uint64_t dn = sw32_desc(smem_u32(smem + st * C::kStage + kMTile));
          for (int i = 0; i < m; ++i)
            umma_f16_ss(acc, dm + (uint64_t)(i * (4096 >> 4)), dn + (uint64_t)(i * (BT * 32 >> 4)), idesc, 1u);
          umma_commit(&empty[st]);
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
      umma_commit(mma_end);  // TMEM and the ring are not given up under an MMA
      mbar_drain(mma_end, 0);
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------ U' of the slices
    // These warps follow the ring by its slice stages alone: a stage is theirs once the
    // producer says so, and is not used again before the MMA has had their U'.
    // A thread writes its row of all slices.  It fetches its row's s_a u once a tile, 32 rank
    // values at a time, and holds them rounded: fetched as their slice came up, every slice of a
    // mixed tile paid the latency of another thread's loads (0.9 us a slice instead of 0.5).
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
      const long long t = (long long)tt * C::kRows + i0;
      const int id = i0 < C::kRows ? row_id(p, t) : -1;
      const float sc = id >= 0 && p.scales ? __ldg(p.scales + id) : 1.f;
      uint4 held[4];  // slices held0 and held0 + 1 of this row, 8 values each
      int held0;
      bool beyond = false;  // a value of this row is more than U' holds
      auto fetch = [&](int c) {
        float4 f[8] = {};
        const float* u = static_cast<const float*>(p.ws) + t * p.rank + c * kSliceRows;
        const int left = p.rank - c * kSliceRows;
        for (int k = 0; k < pl.down_split; ++k, u += part) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i * 4 >= left) continue;
            const float4 x = *reinterpret_cast<const float4*>(u + 4 * i);
            f[i] = make_float4(f[i].x + x.x, f[i].y + x.y, f[i].z + x.z, f[i].w + x.w);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 lo = f[2 * i], hi = f[2 * i + 1];
          held[i] = make_uint4(pack2<T>(lo.x * sc, lo.y * sc), pack2<T>(lo.z * sc, lo.w * sc),
                               pack2<T>(hi.x * sc, hi.y * sc), pack2<T>(hi.z * sc, hi.w * sc));
        }
        const uint32_t top = __vmaxu2(__vmaxu2(magnitudes(held[0]), magnitudes(held[1])),
                                      __vmaxu2(magnitudes(held[2]), magnitudes(held[3])));
        if ((top & 0xffffu) >= kExpBits<T> || top >> 16 >= kExpBits<T>) {
#pragma unroll
          for (int i = 0; i < 4; ++i) beyond |= clamp_infinities<T>(held[i]);
        }
        held0 = c;
      };
      held0 = -2;
      if (id >= 0 && s0 < s1) fetch(0);
      const bool mixed = list[1] != 0;
      Slices sl(list, s0, s1, pl.chunks);
      for (; s0 < s1; s0 += 4, ++it) {
        const int st = it % C::kStages, m = min(4, s1 - s0);
        uint4 v[4][2];  // [slice][8 values]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = sl.part[i];
          v[i][0] = v[i][1] = make_uint4(0u, 0u, 0u, 0u);
          if (id != sl.id[i]) continue;
          if ((c & ~1) != held0) fetch(c & ~1);
          v[i][0] = c & 1 ? held[2] : held[0];
          v[i][1] = c & 1 ? held[3] : held[1];
        }
        sl.next();
        if (!mbar_wait(&u_go[st], uses >> st & 1, kErrTimeoutSmemEmpty, abort_flag)) {
          ok = false;
          break;
        }
        uses ^= 1u << st;
        uint8_t* base = smem + st * C::kStage;
        if (i0 < C::kRows) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half)
              if (i < m)
                *reinterpret_cast<uint4*>(base + C::kUAt + i * C::kUSlice + i0 * 32 + ((half ^ (i0 >> 2 & 1)) << 4)) =
                    v[i][half];
        }
        if (!mbar_wait(&full[st], (it / C::kStages) & 1, kErrTimeoutTmaFull, abort_flag)) {
          ok = false;
          break;
        }
        if (mixed) {
          // all of a thread's pieces are looked at before the rare rewrite
          constexpr uint32_t kExp = kExpBits<T>;
          uint4* at = reinterpret_cast<uint4*>(base + C::kBAt) + i0;
          uint32_t top = 0;
          for (int i = 0; i < m; ++i) {
#pragma unroll
            for (int x = 0; x < C::kCols / 64; ++x) top = __vmaxu2(top, magnitudes(at[(i * (C::kCols / 64) + x) * 128]));
          }
          if ((top & 0xffffu) >= kExp || top >> 16 >= kExp) {
            for (int x = 0; x < m * (C::kCols / 64); ++x) {
              uint4 b = at[x * 128];
              if (drop_nonfinite<T>(b)) at[x * 128] = b;
            }
            s_left_out[n & 15] = n + 1;
          }
        }
        if (beyond) s_left_out[n & 15] = n + 1;
        fence_proxy_async_smem();
        mbar_arrive(&u_full[st]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    // A warp has lane quarter q of the M side and half of the N side's columns (all of 32).
    const int q = warp & 3, half = (warp - 6) >> 2;
    constexpr int kMine = BT >= 64 ? BT / 2 : BT;
    uint8_t* stg = staging + (warp - 6) * 2048;
    int n = 0;
    wait_for_previous();
    for (int tile = tile0; tile < total; tile += step, ++n) {
      const int tt = tile / pl.n_tiles, buf = n & 1;
      const int n0 = (tile - tt * pl.n_tiles) * C::kCols;
      const long long t0 = (long long)tt * C::kRows;
      const int col = n0 + q * 32 + lane;  // weights on the M side: this lane's output column
      const float bias = !kRowsOnM && p.bias && rank == 0 && col < p.N ? __ldg(p.bias + col) : 0.f;
      if (!mbar_wait_warp(&acc_full[buf], (n >> 1) & 1, kErrTimeoutTmemFull, abort_flag)) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BT);
      if (s_left_out[n & 15] == n + 1 && (BT >= 64 || half == 0)) {
        const int* list = lists + (size_t)tt * pl.list_ld;
        int s0, s1;
        slice_range(list, s0, s1);
        add_left_out<T, kRowsOnM>(p, pl, list, s0, s1, kRowsOnM ? t0 + q * 32 + lane : t0, kRowsOnM ? n0 : col, acc,
                                  half * kMine, (half + 1) * kMine);
      }
      if (BT >= 64 || half == 0) {
        for (int c = half * kMine; c < (half + 1) * kMine; c += 32) {
          if (kRowsOnM && n0 + c >= p.N) break;
          uint32_t v[32];
          tmem_ld32(acc + (uint32_t)c, v);
          tmem_ld_wait(v);
          if (kRowsOnM && p.bias) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              if (n0 + c + i < p.N) {  // N is a multiple of 8
                const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + n0 + c + i));
                v[i] = __float_as_uint(__uint_as_float(v[i]) + b.x);
                v[i + 1] = __float_as_uint(__uint_as_float(v[i + 1]) + b.y);
                v[i + 2] = __float_as_uint(__uint_as_float(v[i + 2]) + b.z);
                v[i + 3] = __float_as_uint(__uint_as_float(v[i + 3]) + b.w);
              }
            }
          }
          if constexpr (kRowsOnM) {
            // 32 rows x 32 columns through swizzled shared memory, out by TMA (which clips)
            if (lane == 0) bulk_wait_read0();
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint4 o;
              o.x = pack2<T>(__uint_as_float(v[8 * u]), __uint_as_float(v[8 * u + 1]));
              o.y = pack2<T>(__uint_as_float(v[8 * u + 2]), __uint_as_float(v[8 * u + 3]));
              o.z = pack2<T>(__uint_as_float(v[8 * u + 4]), __uint_as_float(v[8 * u + 5]));
              o.w = pack2<T>(__uint_as_float(v[8 * u + 6]), __uint_as_float(v[8 * u + 7]));
              *reinterpret_cast<uint4*>(stg + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) = o;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&omap, stg, n0 + c, (int)t0 + q * 32, 0);
              bulk_commit();
            }
          } else if (split > 1) {
            // [N side][M side], a lane's values 512 bytes apart
            float* ex = reinterpret_cast<float*>(smem) + c * 128 + q * 32 + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i) ex[i * 128] = __uint_as_float(v[i]) + bias;
          } else if (col < p.N) {
            T* out = static_cast<T*>(p.out) + (t0 + c) * p.ldo + col;
            const int left = (int)min(32LL, p.rows - (t0 + c));
            if (left == 32) {
#pragma unroll
              for (int i = 0; i < 32; ++i, out += p.ldo) *out = from_f32<T>(__uint_as_float(v[i]) + bias);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i, out += p.ldo)
                if (i < left) *out = from_f32<T>(__uint_as_float(v[i]) + bias);
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[buf]);
    }
    if (kRowsOnM && lane == 0) bulk_wait0();
  }

  if (split > 1) {
    // every CTA of the cluster adds up its share of the rows, in rank order
    __syncwarp();
    cluster_sync_all();
    const int tt = tile0 / pl.n_tiles, n0 = (tile0 - tt * pl.n_tiles) * C::kCols;
    const long long t0 = (long long)tt * C::kRows;
    const uint32_t base = smem_u32(smem);
    // 8 consecutive output columns of a row a thread, 16 such groups a row
    const int c0 = BT / 8 * rank / split * 8, c1 = BT / 8 * (rank + 1) / split * 8;
    for (int x = threadIdx.x; x < (c1 - c0) * 16; x += kThreadsA) {
      const int m = (x & 15) * 8, c = c0 + (x >> 4);
      const long long t = t0 + c;
      const int col = n0 + m;
      if (t >= p.rows || col >= p.N) continue;
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < split; ++k) {
        const uint32_t at = mapa_shared(base + (uint32_t)(c * 128 + m) * 4u, (uint32_t)k);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3])
                       : "r"(at + (uint32_t)i * 4u)
                       : "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += v[i];
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + t * p.ldo + col) =
          make_uint4(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]), pack2<T>(sum[4], sum[5]),
                     pack2<T>(sum[6], sum[7]));
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
  // The weights are the MMA's M side (128 of their rows) and up to 128 rows of x its N side
  // while such tiles fit the SMs in one wave, or one tile takes all rows.  More rows are the M side
  // and 256 weight rows the N side: half as many tiles, and a lane of the epilogue holds consecutive
  // output columns, which leave by TMA (weights on the M side: 2-byte stores).  Both sides, weights
  // on M / rows on M, K = N = 4096, rank 16: 512 rows (128 tiles) 22.7 / 26.3 us, 576 (160)
  // 31.9 / 30.6, 1536 53-55 / 56-58, 8192 282 / 243; K = 384, N = 1536: 1536 rows (144 tiles) 9.7 / 14.2,
  // 1600 (156) 11.1 / 10.6, 8192 22.7 / 19.9.
  const long long narrow = (long long)((rows + 127) / 128) * ((N + 127) / 128);
  pl.rows_on_m = rows > 128 && narrow > num_sms;
  pl.bt = rows <= 32 ? 32 : (rows <= 64 ? 64 : 128);
  pl.tiles = (rows + pl.bt - 1) / pl.bt;
  pl.n_tiles = pl.rows_on_m ? (N + 255) / 256 : (N + 127) / 128;
  pl.kblocks = (K + 63) / 64;
  pl.chunks = (rank + kSliceRows - 1) / kSliceRows;
  // first launch: at least 3 K steps of 64 a warp, up to three CTAs for each SM (above rank 16 two are
  // resident at a time)
  const int steps = (K + 63) / 64;
  pl.down_kw = 1;
  while (pl.down_kw < kDownWarps && pl.down_kw * 2 * 3 <= steps) pl.down_kw *= 2;
  const int rows_cta = 32 * (kDownWarps / pl.down_kw);
  pl.down_x = adapters ? (rows + rows_cta - 1) / rows_cta : 0;
  const int want = 3 * num_sms;
  pl.down_split = std::max(1, std::min({want / std::max(pl.down_x, 1), 8, steps / (pl.down_kw * 3)}));
  pl.down_y = std::max(1, std::min({want / std::max(pl.down_x * pl.down_split, 1), 32, adapters}));
  pl.down_nt = rank <= 8 ? 1 : (rank <= 16 ? 2 : (rank <= 32 ? 4 : 8));
  pl.split = 1;
  // Few tiles are split along K over a cluster, whose CTAs add their parts through distributed
  // shared memory, so that a CTA keeps at least 16 steps: K steps of 64 and slices, as many as the tile
  // may have.  Below that the exchange (1 to 4 us) costs more than it saves: 32 rows of K = N = 1024,
  // rank 16, one adapter 7.8 us whole, 9.1 in two, 9.9 in eight; 128 rows with 64 adapters 25.7, 23.8,
  // 21.4.  K = 4096, N = 1536, 32 rows with one adapter 15.0, 12.4, 14.0; with 32 21.9, 22.9, 19.4.
  // Clusters of 4 or 8 take up to half the SMs only, since not all of those can hold one: 33 clusters
  // of 4 and 15 of 8 fit at a time (36 of 4 took 27.5 us where 36 of 2 took 16.1; K = 4096, N = 1536).
  // 132 SMs would do for the clusters of 4, and the rule is not the best everywhere: it takes 2 for
  // (whole / 2 / 4) K = N = 4096, 32 rows with 16 adapters 18.6 / 19.9 / 19.4, with 32 22.4 / 23.9 / 22.8, 128
  // rows with 16 28.3 / 24.1 / 22.8, with 64 42.1 / 35.2 / 31.6; N = 1536, 256 rows with 16 28.1 / 26.0 / 24.9.
  // Rows on the M side are never split: their tiles are more than half the SMs.
  const long long tiles = (long long)pl.tiles * pl.n_tiles;
  const int most = pl.kblocks + std::min(pl.bt, adapters) * pl.chunks;
  for (int s = 2; !pl.rows_on_m && s <= 8 && s <= pl.kblocks && most >= 16 * s; s *= 2)
    if (tiles * s <= (s == 2 ? num_sms : num_sms / 2)) pl.split = s;
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
  cudaError_t e = ensure_smem_limit(adapter_down_kernel<T, NT>, kDownSmem, configured);
  if (e != cudaSuccess) return e;
  const double m = p.rows, k = p.K, r = p.rank;
  LaunchScope scope("adapter_down", 2.0 * m * r * k, 2.0 * (m * k + p.adapters * r * k) + 4.0 * m * r, s);
  adapter_down_kernel<T, NT><<<dim3(pl.down_x + pl.tiles, pl.down_y, pl.down_split), 32 * kDownWarps, kDownSmem, s>>>(p, pl);
  return cudaGetLastError();
}

template <typename T, int BT, bool kRowsOnM>
cudaError_t launch_bt(const AdapterGemmParams& p, const Plan& pl, int num_sms, cudaStream_t s) {
  using C = GemmCfgA<BT, kRowsOnM>;
  static std::atomic<unsigned long long> configured;
  cudaError_t e = ensure_smem_limit(adapter_gemm_kernel<T, BT, kRowsOnM>, (int)C::kSmem, configured);
  if (e != cudaSuccess) return e;
  const double m = p.rows, k = p.K, n = p.N, r = p.rank;
  const CUtensorMap mx = map_2d(p.x, (uint64_t)p.rows, (uint64_t)p.K, (uint64_t)p.ldx, (uint32_t)pl.x_box);
  const CUtensorMap mw = map_2d(p.w, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)p.K, (uint32_t)C::kCols);
  // without adapters no row has one and the map is not read
  const CUtensorMap mb = p.adapters ? map_3d(p.lora_b, (uint64_t)p.rank, (uint64_t)p.N, (uint64_t)p.adapters,
                                             kSliceRows, (uint32_t)C::kCols, CU_TENSOR_MAP_SWIZZLE_32B)
                                    : mx;
  const CUtensorMap mo = kRowsOnM ? map_out_2d(p.out, false, (uint64_t)p.rows, (uint64_t)p.N, (uint64_t)p.ldo) : mx;
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
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)pl.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = pl.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, adapter_gemm_kernel<T, BT, kRowsOnM>, mx, mw, mb, mo, p, pl);
}

template <typename T>
cudaError_t launch_t(const AdapterGemmParams& p, int num_sms, cudaStream_t s) {
  if (p.rows == 0) return cudaSuccess;
  const Plan pl = make_plan(p.rows, p.K, p.N, p.adapters, p.rank, num_sms);
  if (pl.rows_on_m) return launch_bt<T, 256, true>(p, pl, num_sms, s);
  return pl.bt == 32   ? launch_bt<T, 32, false>(p, pl, num_sms, s)
         : pl.bt == 64 ? launch_bt<T, 64, false>(p, pl, num_sms, s)
                       : launch_bt<T, 128, false>(p, pl, num_sms, s);
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
