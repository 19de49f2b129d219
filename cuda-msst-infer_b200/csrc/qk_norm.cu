// qk_norm.cu — norms of queries and keys for each head with the position rotation
// in the same pass.
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

// The table row of a token, or -1 (and a recorded error) outside the tables: such
// a token is normed but not rotated.
__device__ __forceinline__ int table_row(const QkNormParams& p, long long token, int n) {
  const int pos = p.positions ? __ldg(p.positions + token) : n;
  if (pos >= 0 && pos < p.num_pos) return pos;
  record_error(kErrPosition);
  return -1;
}

// One warp per head vector, a pair of columns per lane and step.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_any_kernel(const __grid_constant__ QkNormParams p) {
  const int heads = p.x[0].heads + p.x[1].heads;
  const long long vec = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (vec >= (long long)p.batch * p.seq * heads) return;
  const int lane = threadIdx.x & 31;
  const long long token = vec / heads;
  int h = (int)(vec - token * heads);
  const int which = h >= p.x[0].heads;
  if (which) h -= p.x[0].heads;
  const int b = (int)(token / p.seq), n = (int)(token - (long long)b * p.seq);
  const HeadsView& in = p.x[which];
  const HeadsView& to = p.out[which];
  const T* src = static_cast<const T*>(in.data) + b * in.batch_stride + n * in.seq_stride + h * in.head_stride;
  T* dst = static_cast<T*>(to.data) + b * to.batch_stride + n * to.seq_stride + h * to.head_stride;
  const float* gamma = p.gamma[which];
  const int half = p.rot_dim >> 1, pairs = p.head_dim >> 1;
  auto columns = [&](int i, int& c0, int& c1) {
    if (i < half && p.halves) {
      c0 = i;
      c1 = i + half;
    } else {
      c0 = 2 * i;
      c1 = c0 + 1;
    }
  };
  float a[4], c[4], ss = 0.f;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int i = lane + 32 * s;
    a[s] = c[s] = 0.f;
    if (i < pairs) {
      int c0, c1;
      columns(i, c0, c1);
      a[s] = to_f32(src[c0]);
      c[s] = to_f32(src[c1]);
      ss += a[s] * a[s] + c[s] * c[s];
    }
  }
  const float r = rsqrtf(warp_sum(ss) / p.head_dim + p.eps);
  const int row = half > 0 ? table_row(p, token, n) : -1;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int i = lane + 32 * s;
    if (i < pairs) {
      int c0, c1;
      columns(i, c0, c1);
      float x = a[s] * r * (gamma ? __ldg(gamma + c0) : 1.f), y = c[s] * r * (gamma ? __ldg(gamma + c1) : 1.f);
      if (i < half && row >= 0) {
        const float co = __ldg(p.cos_tab + (size_t)row * half + i), si = __ldg(p.sin_tab + (size_t)row * half + i);
        const float t = x * co - y * si;
        y = y * co + x * si;
        x = t;
      }
      dst[c0] = from_f32<T>(x);
      dst[c1] = from_f32<T>(y);
    }
  }
}

template <typename T>
cudaError_t launch_t(const QkNormParams& p, cudaStream_t s) {
  const long long vecs = (long long)p.batch * p.seq * (p.x[0].heads + p.x[1].heads);
  if (vecs == 0) return cudaSuccess;
  const double values = (double)vecs * p.head_dim;
  LaunchScope scope("qk_norm_rope", 7.0 * values, 4.0 * values + 4.0 * (double)p.batch * p.seq, s);
  qk_norm_any_kernel<T><<<(unsigned)((vecs + 7) / 8), 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_qk_norm(const QkNormParams& p, int bf16, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, stream) : launch_t<__half>(p, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(qk_norm_device_error)

}  // namespace msst
