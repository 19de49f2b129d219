// prefix_attn.cu — attention of a batch's new tokens to a prefix that all requests share and to
// each request's own tokens in the pages of a cache, causal among the new ones.
#include "cache_ops.cuh"
#include "common.cuh"
#include "runtime.h"

namespace msst {

namespace {

__device__ __forceinline__ int own_len(const PrefixAttnParams& p, int r) {
  const long long most = (long long)p.blocks << p.page_shift;
  return (int)min((long long)max(__ldg(p.lens + r), 0), most);
}
__device__ __forceinline__ int first_row(const PrefixAttnParams& p, int r) {
  return p.q_starts ? min(max(__ldg(p.q_starts + r), 0), p.tokens) : r;
}

// One query row by one warp, key by key, 4 columns a lane.
template <typename T>
__device__ void attend_row(const PrefixAttnParams& p, int r, int token, int head, int limit, int lane) {
  const int hk = head / (p.q.heads / p.k_cache.heads);
  const bool active = 4 * lane < p.head_dim;
  auto load4 = [&](const T* x, float (&v)[4]) {
    v[0] = v[1] = v[2] = v[3] = 0.f;
    if (!active) return;
    const uint2 w = *reinterpret_cast<const uint2*>(x + 4 * lane);
    unpack2<T>(w.x, v[0], v[1]);
    unpack2<T>(w.y, v[2], v[3]);
  };
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load4(static_cast<const T*>(p.q.data) + token * p.q.seq_stride + head * p.q.head_stride, q);
  for (long long j = 0; j < (long long)p.prefix + limit; ++j) {
    const HeadsView& kv = j < p.prefix ? p.prefix_k : p.k_cache;
    const HeadsView& vv = j < p.prefix ? p.prefix_v : p.v_cache;
    long long ko, vo;
    if (j < p.prefix) {
      ko = j * kv.seq_stride;
      vo = j * vv.seq_stride;
    } else {
      const int i = (int)(j - p.prefix), page = __ldg(p.table + r * p.table_stride + (i >> p.page_shift));
      if ((unsigned)page >= (unsigned)p.pages) {
        record_error(kErrPage);
        continue;
      }
      const int at = i & ((1 << p.page_shift) - 1);
      ko = page * kv.batch_stride + at * kv.seq_stride;
      vo = page * vv.batch_stride + at * vv.seq_stride;
    }
    float k[4], v[4];
    load4(static_cast<const T*>(kv.data) + ko + hk * kv.head_stride, k);
    load4(static_cast<const T*>(vv.data) + vo + hk * vv.head_stride, v);
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float a = fast_exp2(m - base), e = fast_exp2(s - base);
    m = mn;
    l = l * a + e;
#pragma unroll
    for (int x = 0; x < 4; ++x) o[x] = o[x] * a + e * v[x];
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (!active) return;
  T* out = static_cast<T*>(p.out.data) + token * p.out.seq_stride + head * p.out.head_stride + 4 * lane;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
}

// The request of a token, or -1.
__device__ __forceinline__ int request_of(const PrefixAttnParams& p, int token) {
  if (!p.q_starts) return token;
  int lo = 0;
  for (int len = p.requests + 1; len > 1;) {
    const int half = len >> 1;
    if (first_row(p, lo + half) <= token) lo += half;
    len -= half;
  }
  return lo < p.requests && first_row(p, lo) <= token ? lo : -1;
}

template <typename T>
__global__ void __launch_bounds__(256) prefix_rows_kernel(const __grid_constant__ PrefixAttnParams p) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (long long)p.tokens * p.q.heads) return;
  const int token = (int)(row / p.q.heads), head = (int)(row - (long long)token * p.q.heads);
  const int r = request_of(p, token);
  if (r < 0) return;
  const int len = own_len(p, r), n = first_row(p, r + 1) - first_row(p, r), i = token - first_row(p, r);
  attend_row<T>(p, r, token, head, min(max(len - (p.q_starts ? n : 1) + i + 1, 0), len), threadIdx.x & 31);
}

template <typename T>
cudaError_t launch_t(const PrefixAttnParams& p, int num_sms, cudaStream_t s) {
  const long long rows = (long long)p.tokens * p.q.heads;
  LaunchScope scope("prefix_rows", 4.0 * rows * p.prefix * p.head_dim, 4.0 * rows * p.head_dim, s);
  prefix_rows_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

long long prefix_attention_workspace(int tokens, int requests, int prefix, int q_heads, int kv_heads, int head_dim,
                                     int num_sms) {
  return 0;
}

cudaError_t launch_prefix_attention(const PrefixAttnParams& p, int bf16, int num_sms, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, num_sms, stream) : launch_t<__half>(p, num_sms, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(prefix_attn_device_error)

}  // namespace msst
