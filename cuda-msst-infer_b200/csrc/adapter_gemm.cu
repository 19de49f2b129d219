// adapter_gemm.cu — a shared projection with the low-rank adapters of many
// requests beside it.
#include "common.cuh"
#include "operators.cuh"
#include "runtime.h"

namespace msst {

namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// u[t, r] = s_a (A_a x[t])_r, one warp per value.
template <typename T>
__global__ void __launch_bounds__(256) adapter_down_simple_kernel(const __grid_constant__ AdapterGemmParams p) {
  const long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= (long long)p.rows * p.rank) return;
  const int t = (int)(i / p.rank), r = (int)(i - (long long)t * p.rank);
  const int a = __ldg(p.row_adapter + t);
  float s = 0.f;
  if (a >= 0 && a < p.adapters) {
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    const T* w = static_cast<const T*>(p.lora_a) + ((size_t)a * p.rank + r) * p.K;
    for (int k = lane; k < p.K; k += 32) s += to_f32(x[k]) * to_f32(w[k]);
    s = warp_sum(s) * (p.scales ? __ldg(p.scales + a) : 1.f);
  }
  if (lane == 0) p.u[i] = s;
}

// y[t, n], 16 x 16 outputs per block, x and W through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) adapter_gemm_simple_kernel(const __grid_constant__ AdapterGemmParams p) {
  __shared__ float sx[16][33], sw[16][33];
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const long long t0 = (long long)blockIdx.y * 16;
  const int n0 = blockIdx.x * 16;
  const long long t = t0 + ty;
  const int n = n0 + tx;
  float acc = 0.f;
  for (int k0 = 0; k0 < p.K; k0 += 32) {
    for (int i = threadIdx.x; i < 512; i += 256) {
      const int rr = i >> 5, kk = i & 31;
      const bool in = k0 + kk < p.K;
      sx[rr][kk] = in && t0 + rr < p.rows ? to_f32(static_cast<const T*>(p.x)[(t0 + rr) * p.ldx + k0 + kk]) : 0.f;
      sw[rr][kk] = in && n0 + rr < p.N ? to_f32(static_cast<const T*>(p.w)[(size_t)(n0 + rr) * p.K + k0 + kk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 32; ++kk) acc += sx[ty][kk] * sw[tx][kk];
    __syncthreads();
  }
  if (t >= p.rows || n >= p.N) return;
  if (p.bias) acc += __ldg(p.bias + n);
  const int a = __ldg(p.row_adapter + t);
  if (a >= 0 && a < p.adapters) {
    const T* bw = static_cast<const T*>(p.lora_b) + ((size_t)a * p.N + n) * p.rank;
    for (int r = 0; r < p.rank; ++r) acc += p.u[(size_t)t * p.rank + r] * to_f32(bw[r]);
  } else if (a != -1 && n == 0) {
    record_error(kErrAdapter);
  }
  static_cast<T*>(p.out)[t * p.ldo + n] = from_f32<T>(acc);
}

template <typename T>
cudaError_t launch_t(const AdapterGemmParams& p, cudaStream_t s) {
  if (p.rows == 0) return cudaSuccess;
  const double m = p.rows, k = p.K, n = p.N, r = p.rank;
  {
    LaunchScope scope("adapter_down", 2.0 * m * r * k, 2.0 * (m * k + p.adapters * r * k) + 4.0 * m * r, s);
    adapter_down_simple_kernel<T><<<(unsigned)(((long long)p.rows * p.rank + 7) / 8), 256, 0, s>>>(p);
  }
  LaunchScope scope("adapter_gemm", 2.0 * m * n * (k + r), 2.0 * (m * k + n * k + m * n + p.adapters * r * n), s);
  adapter_gemm_simple_kernel<T>
      <<<dim3((unsigned)((p.N + 15) / 16), (unsigned)((p.rows + 15) / 16)), 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_adapter_gemm(const AdapterGemmParams& p, int bf16, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, stream) : launch_t<__half>(p, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(adapter_gemm_device_error)

}  // namespace msst
