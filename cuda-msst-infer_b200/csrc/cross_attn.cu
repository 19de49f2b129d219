// cross_attn.cu — cross attention to an encoder's states of another length.
#include "common.cuh"
#include "operators.cuh"
#include "runtime.h"

namespace msst {

namespace {

// One warp per query row and head: 32 keys at a time, one score per lane, running
// maximum and sum; each lane owns head_dim / 32 columns of the output.
template <typename T>
__global__ void __launch_bounds__(128) cross_attention_simple_kernel(const __grid_constant__ CrossAttnParams p) {
  __shared__ float sq[4][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long rows = (long long)p.batch * p.q_len * p.q.heads;
  const long long r = (long long)blockIdx.x * 4 + warp;
  if (r >= rows) return;
  const int h = (int)(r % p.q.heads);
  const long long bn = r / p.q.heads;
  const int b = (int)(bn / p.q_len), n = (int)(bn - (long long)b * p.q_len);
  const int hk = h / (p.q.heads / p.k.heads);
  const int d = p.head_dim;
  const T* q = static_cast<const T*>(p.q.data) + b * p.q.batch_stride + n * p.q.seq_stride + h * p.q.head_stride;
  const T* k = static_cast<const T*>(p.k.data) + b * p.k.batch_stride + hk * p.k.head_stride;
  const T* v = static_cast<const T*>(p.v.data) + b * p.v.batch_stride + hk * p.v.head_stride;
  T* out = static_cast<T*>(p.out.data) + b * p.out.batch_stride + n * p.out.seq_stride + h * p.out.head_stride;
  for (int i = lane; i < d; i += 32) sq[warp][i] = to_f32(q[i]);
  __syncwarp();
  int len = p.k_len;
  if (p.key_lens) len = min(max(__ldg(p.key_lens + b), 0), len);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    const bool keep = j < len && (!p.key_mask || p.key_mask[(size_t)b * p.k_len + j]);
    float s = -INFINITY;
    if (keep) {
      s = 0.f;
      for (int i = 0; i < d; ++i) s += sq[warp][i] * to_f32(k[(long long)j * p.k.seq_stride + i]);
      s *= p.scale_log2;
    }
    float mx = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    if (mx == -INFINITY) continue;
    const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float e = keep ? exp2f(s - mn) : 0.f;
    float sum = e;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * alpha + sum;
    m = mn;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= alpha;
    for (int t = 0; t < 32; ++t) {
      const float pt = __shfl_sync(0xffffffffu, e, t);
      if (!__shfl_sync(0xffffffffu, (int)keep, t)) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < d) o[c] += pt * to_f32(v[(long long)(j0 + t) * p.v.seq_stride + lane + 32 * c]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < d) out[lane + 32 * c] = from_f32<T>(o[c] * inv);
}

template <typename T>
cudaError_t launch_t(const CrossAttnParams& p, cudaStream_t s) {
  const long long rows = (long long)p.batch * p.q_len * p.q.heads;
  if (rows == 0) return cudaSuccess;
  const double d = p.head_dim, keys = (double)p.batch * p.k_len;
  LaunchScope scope("cross_attention", 4.0 * rows * p.k_len * d, 4.0 * rows * d + 4.0 * keys * p.k.heads * d, s);
  cross_attention_simple_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cross_attention(const CrossAttnParams& p, int bf16, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, stream) : launch_t<__half>(p, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(cross_attn_device_error)

}  // namespace msst
