// cross_token.cu — cross attention of a few query rows (one new token, or a short chunk
// with few heads a group): up to 16 rows a key head.  See cross_attn.cu for the operator.
//
// Bound: reading K and V once.  The group's rows fill one m16 tile of mma.sync
// m16n8k16, whose fragments come straight from 128-byte swizzled TMA tiles by ldmatrix
// (an M of 128 rows on the tcgen05 path holds each K/V tile in shared memory for the length
// of a full tile's chain and leaves too little of it for loads in flight: 62.9 us against
// 42.9 for 16 sequences of up to 4096 keys, 32/8 heads of 128).  That call is 43 us, 41 of them
// this kernel's alone (206 MB, 5.1 TB/s); one sequence of 131072 keys, 8 heads of 64, 56 to 58 us.
//
// CTA = 288 threads: warp 8 brings tiles of 64 keys into a ring as deep as shared memory
// allows; warps 0-3 take the even tiles of the CTA's run and warps 4-7 the odd ones (the
// number of stages is even, so a stage is always the same four warps'), 16 keys a warp,
// each with its own running maximum, sum and O (fp32); they are joined once an
// item.  Runs of units, partial results and the joining launch are cross_attn.cu's.
#include <algorithm>

#include "attn_steps.cuh"
#include "common.cuh"
#include "cross_attn.cuh"
#include "operators.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kKeys = 64;
constexpr int kMaxStages = 12;
constexpr uint32_t kBox = kKeys * 128;  // 64 keys x 64 columns
// 16-byte piece `chunk` (8 columns) of key `row` in a 128B-swizzled tile of 64-column boxes
__device__ __forceinline__ uint32_t piece(uint32_t tile, int row, int chunk) {
  return tile + (uint32_t)((chunk >> 3) * kBox + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

template <typename T, int DP, bool kMask>
__global__ void __launch_bounds__(kThreads, 1)
    cross_token_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ CrossAttnParams p, const __grid_constant__ Geom g, int stages,
                       int rows) {
  constexpr int kHalves = DP / 64;
  constexpr uint32_t kStage = 2 * kHalves * kBox;  // K, then V
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ Spot s_spot;
  __shared__ long long s_count;
  __shared__ int s_abort, s_stop;
  __shared__ float s_m[kWarps][16], s_l[kWarps][16];
  volatile int* abort_flag = &s_abort;
  float* s_o = reinterpret_cast<float*>(smem + (size_t)stages * kStage);  // [warps][rows][DP]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  if (warp == kWarps) {
    const long long U = total_units(p, g, lane);
    const long long u0 = U * blockIdx.x / gridDim.x, u1 = U * (blockIdx.x + 1) / gridDim.x;
    const Spot s = find_spot(p, g, u0, lane);
    if (lane == 0) {
      s_spot = s;
      s_count = u1 - u0;
    }
  }
  __syncthreads();
  dependents_may_start();
  Walk k(s_spot, s_count);

  if (warp == kWarps) {
    if (lane == 0) {
      int st = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && k.next(p, g)) {
        const int kh = k.s.hk * g.k_headed, kb = k.s.b * g.k_batched;
        const int vh = k.s.hk * g.v_headed, vb = k.s.b * g.v_batched;
        for (int j = k.j0; j < k.j1; ++j) {
          if (!mbar_wait<false>(&empty[st], phase ^ 1, kErrTimeoutAttnKV, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[st], kStage);
          uint8_t* dst = smem + (size_t)st * kStage;
          for (int h = 0; h < kHalves; ++h) {
            tma_load_4d(dst + h * kBox, &kmap, &full[st], h * 64, j * kKeys, kh, kb);
            tma_load_4d(dst + (kHalves + h) * kBox, &vmap, &full[st], h * 64, j * kKeys, vh, vb);
          }
          if (++st == stages) st = 0, phase ^= 1;
        }
      }
      mbar_drain_ring(full, stages, st, phase);
    }
    return;
  }

  const int set = warp >> 2, wk = warp & 3;  // tiles of this parity; 16 keys of each
  const int qr = lane >> 2, qc = lane & 3;   // fragment row (and row + 8) and column pair
  const float c = p.scale_log2;
  const uint32_t base = smem_u32(smem);
  // ldmatrix row addresses: K wants (keys 0-7, 8 columns), (keys 0-7, next 8), (keys 8-15, ..) x 2;
  // V (transposed) wants (keys 0-7), (keys 8-15) of 8 columns, then of the next 8
  const int krow = wk * 16 + (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;
  const int vrow = wk * 16 + (lane & 15), vchunk = lane >> 4;
  int st = 0;
  uint32_t phase = 0;
  bool ok = true;
  while (ok && k.next(p, g)) {
    const int first = k.j0 + ((st & 1) != set);  // this set's first tile of the item
    // Q fragments of the rows r = n * group + head of the group, from global memory
    uint32_t qa[DP / 16][4];
    {
      const T* qp = static_cast<const T*>(p.q.data) + (long long)k.s.b * p.q.batch_stride +
                    (long long)k.s.hk * g.group * p.q.head_stride;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = qr + 8 * half, n = r / g.group, h = r - n * g.group;
        const T* row = qp + (long long)n * p.q.seq_stride + (long long)h * p.q.head_stride;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          const int c0 = s * 16 + qc * 2;
          qa[s][half] = r < rows && c0 < p.head_dim ? *reinterpret_cast<const uint32_t*>(row + c0) : 0u;
          qa[s][2 + half] = r < rows && c0 + 8 < p.head_dim ? *reinterpret_cast<const uint32_t*>(row + c0 + 8) : 0u;
        }
      }
    }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const unsigned char* mask = kMask ? p.key_mask + (size_t)k.s.b * p.k_len : nullptr;
    // the kept ones of this lane's four keys of tile j (pairs qc * 2 and qc * 2 + 8)
    auto kept = [&](int j) {
      const int k0 = j * kKeys + wk * 16 + qc * 2;
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = k0 + (i >> 1) * 8 + (i & 1);
        if (key < k.keys && (!kMask || mask[key])) bits |= 1u << i;
      }
      return bits;
    };
    uint32_t bits = kMask && first < k.j1 ? kept(first) : 0u;
    for (int jj = k.j0; jj < k.j1; ++jj) {
      const int stage = st;
      const uint32_t par = phase;
      if (++st == stages) st = 0, phase ^= 1;
      if ((stage & 1) != set) continue;
      if (!mbar_wait_warp<false>(&full[stage], par, kErrTimeoutAttnKV, abort_flag)) {
        ok = false;
        break;
      }
      const uint32_t kt = base + (uint32_t)stage * kStage, vt = kt + kHalves * kBox;
      // S: two column tiles of 8 keys; even and odd k-steps in accumulators of their own
      float sc[2][2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) (&sc[0][0][0])[i] = 0.f;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        uint32_t b[4];
        ldmatrix4(piece(kt, krow, 2 * s + kchunk), b);
        mma16816<T>(sc[s & 1][0], qa[s], b[0], b[1]);
        mma16816<T>(sc[s & 1][1], qa[s], b[2], b[3]);
      }
      const uint32_t now = bits;
      if (kMask && jj + 2 < k.j1) bits = kept(jj + 2);  // in flight during this tile
      const bool all = kMask ? __all_sync(0xffffffffu, now == 15u) : (jj + 1) * kKeys <= k.keys;
      const uint32_t keep = kMask ? now : (all ? 15u : kept(jj));
      float e[2][4];
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // i: row half * 2 + key of the pair
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float x = (sc[0][t][i] + sc[1][t][i]) * c;
          e[t][i] = all || (keep >> (2 * t + (i & 1)) & 1) ? x : -INFINITY;
          mx[i >> 1] = fmaxf(mx[i >> 1], e[t][i]);
        }
      }
      float alpha[2], ref[2];
      bool moved = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float mn = fmaxf(m[h], mx[h]);
        ref[h] = mn == -INFINITY ? 0.f : mn;  // no kept key yet: exponentials of -inf stay 0
        alpha[h] = fast_exp2(m[h] - ref[h]);
        moved |= mn > m[h];
        m[h] = mn;
      }
      uint32_t pa[4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[t][i] = fast_exp2(e[t][i] - (ref[i >> 1] - kLift<T>));
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) l[h] *= alpha[h];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[0];
          o[i][2] *= alpha[1];
          o[i][3] *= alpha[1];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) l[h] += (e[0][2 * h] + e[0][2 * h + 1]) + (e[1][2 * h] + e[1][2 * h + 1]);
      pa[0] = pack2<T>(e[0][0], e[0][1]);
      pa[1] = pack2<T>(e[0][2], e[0][3]);
      pa[2] = pack2<T>(e[1][0], e[1][1]);
      pa[3] = pack2<T>(e[1][2], e[1][3]);
      // keys that are not kept: their V is taken as zero (0 * NaN would reach the sum)
      const uint32_t v0 = (keep & 1 ? 0xffffu : 0u) | (keep & 2 ? 0xffff0000u : 0u);
      const uint32_t v1 = (keep & 4 ? 0xffffu : 0u) | (keep & 8 ? 0xffff0000u : 0u);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t b[4];
        ldmatrix4_trans(piece(vt, vrow, 2 * i + vchunk), b);
        if (!all) {
          b[0] &= v0;
          b[1] &= v1;
          b[2] &= v0;
          b[3] &= v1;
        }
        // a tile's products in accumulators of their own, added in fp32: an MMA cuts each product off
        // against what its accumulator holds, which lost weights of 2^-25 of a running sum (one of
        // 131072 keys, 8 heads of 64: 55.8 us, summed by the MMAs 54.9)
        float d[2][4] = {};
        mma16816<T>(d[0], pa, b[0], b[1]);
        mma16816<T>(d[1], pa, b[2], b[3]);
#pragma unroll
        for (int x = 0; x < 8; ++x) o[2 * i + (x >> 2)][x & 3] += d[x >> 2][x & 3];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
    if (!ok) *abort_flag = 1;
    // join the eight warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int r = qr + 8 * h;
      if (r < rows) {
        if (qc == 0) {
          s_m[warp][r] = m[h];
          s_l[warp][r] = l[h];
        }
        float* so = s_o + ((size_t)warp * rows + r) * DP + qc * 2;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          *reinterpret_cast<float2*>(so + i * 8) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    // one reading for all: the producer may set the flag while they read it
    if (threadIdx.x == 0) s_stop = *abort_flag;
    const bool whole = k.whole();
    for (int x = threadIdx.x; x < rows * (p.head_dim / 4); x += 256) {
      const int r = x / (p.head_dim / 4), col = (x - r * (p.head_dim / 4)) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
      float ls = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (s_l[w][r] == 0.f) continue;
        const float f = fast_exp2(s_m[w][r] - mm);
        const float4 v = *reinterpret_cast<const float4*>(s_o + ((size_t)w * rows + r) * DP + col);
        ls += s_l[w][r] * f;
        sum = make_float4(sum.x + v.x * f, sum.y + v.y * f, sum.z + v.z * f, sum.w + v.w * f);
      }
      if (whole) {
        const float inv = ls > 0.f ? 1.f / ls : (ls == 0.f ? 0.f : ls);
        const int n = r / g.group, h = k.s.hk * g.group + r - n * g.group;
        T* out = static_cast<T*>(p.out.data) + (long long)k.s.b * p.out.batch_stride +
                 (long long)n * p.out.seq_stride + (long long)h * p.out.head_stride + col;
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
      } else {
        float* po = p.ws + ((size_t)(2 * blockIdx.x + (k.seg > 0)) * g.slot_rows + r) * part_ld(p.head_dim);
        *reinterpret_cast<float4*>(po + col) = sum;
        if (col == 0) *reinterpret_cast<float2*>(po + p.head_dim) = make_float2(mm, ls);
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    ok = s_stop == 0;  // not written again before all have been at the next item's first barrier
  }
}

template <typename T, int DP, bool kMask>
cudaError_t launch_k(const CrossAttnParams& p, Geom g, cudaStream_t s) {
  static std::atomic<unsigned long long> configured;
  constexpr uint32_t stage = 2 * (DP / 64) * kBox;
  constexpr int most = 227 * 1024 - 2048;
  cudaError_t e = ensure_smem_limit(cross_token_kernel<T, DP, kMask>, most, configured);
  if (e != cudaSuccess) return e;
  const int rows = g.group * p.q_len;
  const size_t join = (size_t)kWarps * rows * DP * sizeof(float);
  const int stages = std::min<int>(kMaxStages, (int)((most - join) / stage)) & ~1;
  const CUtensorMap mk = cross_kv_map(p.k, p.batch, p.k_len, p.head_dim, kKeys, g.k_batched, g.k_headed);
  const CUtensorMap mv = cross_kv_map(p.v, p.batch, p.k_len, p.head_dim, kKeys, g.v_batched, g.v_headed);
  const double qrows = (double)p.batch * p.q_len * p.q.heads, keys = (double)p.batch * p.k_len * p.k.heads;
  LaunchScope scope("cross_token", 4.0 * qrows * p.k_len * p.head_dim, 4.0 * (qrows + keys) * p.head_dim, s);
  cross_token_kernel<T, DP, kMask>
      <<<g.contribs, kThreads, (size_t)stages * stage + join, s>>>(mk, mv, p, g, stages, rows);
  return cudaGetLastError();
}

}  // namespace

template <typename T>
cudaError_t launch_cross_token(const CrossAttnParams& p, Geom g, cudaStream_t s) {
  if (p.head_dim <= 64) return p.key_mask ? launch_k<T, 64, true>(p, g, s) : launch_k<T, 64, false>(p, g, s);
  return p.key_mask ? launch_k<T, 128, true>(p, g, s) : launch_k<T, 128, false>(p, g, s);
}
template cudaError_t launch_cross_token<__half>(const CrossAttnParams&, Geom, cudaStream_t);
template cudaError_t launch_cross_token<__nv_bfloat16>(const CrossAttnParams&, Geom, cudaStream_t);

MSST_DEFINE_ERROR_ACCESSOR(cross_token_device_error)

}  // namespace msst
