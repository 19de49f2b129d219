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

template <bool kStream, typename V>
__device__ __forceinline__ V load(const V* p) {
  return kStream ? __ldcs(p) : *p;
}
template <bool kStream, typename V>
__device__ __forceinline__ void store(V* p, const V& v) {
  if constexpr (kStream)
    __stcs(p, v);
  else
    *p = v;
}

// The table row of a token, or -1 (and a recorded error) outside the tables: such
// a token is normed but not rotated.
__device__ __forceinline__ int table_row(const QkNormParams& p, long long token, int n) {
  const int pos = p.positions ? __ldg(p.positions + token) : n;
  if (pos >= 0 && pos < p.num_pos) return pos;
  record_error(kErrPosition);
  return -1;
}

// 8 columns a lane: LPV lanes (the power of two that covers head_dim / 8) hold a head
// vector, so the sum of squares takes log2(LPV) shuffles.  A group of LPV lanes takes
// kHeads heads of one token: their loads are all in flight before the first is used
// (64 bytes a thread, enough to cover HBM's latency at half occupancy), and the
// position's cos / sin row and gamma are fetched once for all of them.  Pairs stay
// inside a lane: with kHalves a lane of the rotated part takes columns
// [4l, 4l + 4) and [rot/2 + 4l, rot/2 + 4l + 4), two 8-byte loads instead of one of
// 16 bytes, which costs issue slots that this kernel has to spare (shuffling the
// partner's 8 values would cost more of them).
// Bound: HBM.  338 MB (4 x 4096 tokens, 32 + 8 heads of 128) take 64 us (5.3 TB/s), 197 MB of packed
// rows 36 us (5.5 TB/s).  kStream marks loads and stores as read and written once: 63.9 -> 59.5 us
// for one set of buffers of the first, no difference below L2's size, where the results should stay for the
// attention that reads them.  Two heads a group took 75 us, eight 77, 256 threads a
// block 67.
constexpr int kHeads = 4;

template <typename T, int LPV, bool kHalves, bool kStream>
__global__ void __launch_bounds__(128) qk_norm_kernel(const __grid_constant__ QkNormParams p, unsigned items,
                                                      int chunks_q, int chunks) {
  const unsigned item = qk_norm_item(blockIdx.x, threadIdx.x, LPV);
  const int l = threadIdx.x % LPV;
  if (item >= items) return;  // whole groups: the shuffles below stay inside a group
  const unsigned token = item / (unsigned)chunks;
  int chunk = (int)(item - token * (unsigned)chunks);
  const int which = chunk >= chunks_q;
  if (which) chunk -= chunks_q;
  const int b = (int)(token / (unsigned)p.seq), n = (int)(token - (unsigned)b * (unsigned)p.seq);
  const HeadsView& in = p.x[which];
  const HeadsView& to = p.out[which];
  const int h0 = chunk * kHeads, left = in.heads - h0;
  const bool active = 8 * l < p.head_dim;
  const int half = p.rot_dim >> 1;
  const bool turned = 8 * l < p.rot_dim;
  const int c0 = kHalves && turned ? 4 * l : 8 * l, c1 = kHalves && turned ? half + 4 * l : 8 * l + 4;
  const T* src = static_cast<const T*>(in.data) + b * in.batch_stride + n * in.seq_stride + h0 * in.head_stride;
  T* dst = static_cast<T*>(to.data) + b * to.batch_stride + n * to.seq_stride + h0 * to.head_stride;

  uint2 raw[kHeads][2];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    raw[u][0] = raw[u][1] = make_uint2(0u, 0u);
    if (active && u < left) {
      const T* s = src + u * in.head_stride;
      if constexpr (kHalves) {
        raw[u][0] = load<kStream>(reinterpret_cast<const uint2*>(s + c0));
        raw[u][1] = load<kStream>(reinterpret_cast<const uint2*>(s + c1));
      } else {
        const uint4 v = load<kStream>(reinterpret_cast<const uint4*>(s + c0));
        raw[u][0] = make_uint2(v.x, v.y);
        raw[u][1] = make_uint2(v.z, v.w);
      }
    }
  }
  float g[8], co[4], si[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = 1.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) co[i] = 1.f, si[i] = 0.f;
  const float* gamma = p.gamma[which];
  if (active && gamma) {
    *reinterpret_cast<float4*>(g) = __ldg(reinterpret_cast<const float4*>(gamma + c0));
    *reinterpret_cast<float4*>(g + 4) = __ldg(reinterpret_cast<const float4*>(gamma + c1));
  }
  const int row = half > 0 ? table_row(p, token, n) : -1;
  const bool rotate = turned && row >= 0;
  if (rotate) {
    const size_t at = (size_t)row * half + 4 * l;  // pairs 4l .. 4l + 3 with either pairing
    *reinterpret_cast<float4*>(co) = __ldg(reinterpret_cast<const float4*>(p.cos_tab + at));
    *reinterpret_cast<float4*>(si) = __ldg(reinterpret_cast<const float4*>(p.sin_tab + at));
  }
  const unsigned group = LPV == 32 ? 0xffffffffu : ((1u << LPV) - 1u) << ((threadIdx.x & 31) / LPV * LPV);
  const float inv_d = 1.f / (float)p.head_dim;
  // kAsk: pairs that are not rotated (a tail, a position outside the tables) keep their values, which
  // (1, 0) as a rotation would not do for an infinity's neighbour (0 * inf).  Interleaved groups whose
  // pairs all turn do not ask: 35.8 us for 60 x 801 tokens, 8 + 8 heads of 64, asking 36.1, a branch
  // in each head 36.9.  With halves the second form costs more than the question: 65.9 us for
  // 4 x 4096 tokens, 32 + 8 heads of 128, 64.4 always asking.
  auto heads = [&](auto ask) {
    constexpr bool kAsk = decltype(ask)::value;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (u >= left) break;
      float x[8];
      unpack2<T>(raw[u][0].x, x[0], x[1]);
      unpack2<T>(raw[u][0].y, x[2], x[3]);
      unpack2<T>(raw[u][1].x, x[4], x[5]);
      unpack2<T>(raw[u][1].y, x[6], x[7]);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int o = LPV / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
      const float r = rsqrtf(ss * inv_d + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= r * g[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // kHalves: (x[i], x[4 + i]); interleaved: (x[2i], x[2i + 1])
        float& a = kHalves ? x[i] : x[2 * i];
        float& c = kHalves ? x[4 + i] : x[2 * i + 1];
        if (kHalves && !turned) break;  // the unrotated tail of a vector
        const float t = a * co[i] - c * si[i], w = c * co[i] + a * si[i];
        a = !kAsk || rotate ? t : a;
        c = !kAsk || rotate ? w : c;
      }
      const uint2 y0 = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
      const uint2 y1 = make_uint2(pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
      if (active) {
        T* t = dst + u * to.head_stride;
        if constexpr (kHalves) {
          store<kStream>(reinterpret_cast<uint2*>(t + c0), y0);
          store<kStream>(reinterpret_cast<uint2*>(t + c1), y1);
        } else {
          store<kStream>(reinterpret_cast<uint4*>(t + c0), make_uint4(y0.x, y0.y, y1.x, y1.y));
        }
      }
    }
  };
  if (!kHalves && row >= 0 && p.rot_dim == p.head_dim)
    heads(std::false_type{});
  else
    heads(std::true_type{});
}

// Any even head_dim, stride and alignment: one warp per head vector, a pair of
// columns per lane and step.
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

// Whether the 8-column kernel can walk the call's tensors: 16-byte rows and tables,
// and no group of columns that is rotated in part.
bool wide_ok(const QkNormParams& p) {
  auto a16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if (p.head_dim % 8 != 0 || p.rot_dim % 8 != 0) return false;
  if (!a16(p.cos_tab) || !a16(p.sin_tab) || !a16(p.gamma[0]) || !a16(p.gamma[1])) return false;
  for (const HeadsView* v : {&p.x[0], &p.x[1], &p.out[0], &p.out[1]})
    if (v->heads && (!a16(v->data) || v->batch_stride % 8 || v->seq_stride % 8 || v->head_stride % 8)) return false;
  return true;
}

template <typename T, int LPV>
void launch_wide(const QkNormParams& p, cudaStream_t s) {
  const int cq = (p.x[0].heads + kHeads - 1) / kHeads, ck = (p.x[1].heads + kHeads - 1) / kHeads;
  const unsigned items = (unsigned)((long long)p.batch * p.seq * (cq + ck));
  const unsigned grid = (unsigned)(((long long)items * LPV + 127) / 128);
  // more than L2 (126 MB) holds is streamed
  const bool stream = 4.0 * p.batch * p.seq * (p.x[0].heads + p.x[1].heads) * p.head_dim > 126e6;
  auto go = [&](auto kernel) { kernel<<<grid, 128, 0, s>>>(p, items, cq, cq + ck); };
  if (p.halves)
    stream ? go(qk_norm_kernel<T, LPV, true, true>) : go(qk_norm_kernel<T, LPV, true, false>);
  else
    stream ? go(qk_norm_kernel<T, LPV, false, true>) : go(qk_norm_kernel<T, LPV, false, false>);
}

template <typename T>
cudaError_t launch_t(const QkNormParams& p, cudaStream_t s) {
  const long long vecs = (long long)p.batch * p.seq * (p.x[0].heads + p.x[1].heads);
  if (vecs == 0) return cudaSuccess;
  const double values = (double)vecs * p.head_dim;
  LaunchScope scope("qk_norm_rope", 7.0 * values, 4.0 * values + 4.0 * (double)p.batch * p.seq, s);
  if (!wide_ok(p))
    qk_norm_any_kernel<T><<<(unsigned)((vecs + 7) / 8), 256, 0, s>>>(p);
  else if (p.head_dim <= 8)
    launch_wide<T, 1>(p, s);
  else if (p.head_dim <= 16)
    launch_wide<T, 2>(p, s);
  else if (p.head_dim <= 32)
    launch_wide<T, 4>(p, s);
  else if (p.head_dim <= 64)
    launch_wide<T, 8>(p, s);
  else if (p.head_dim <= 128)
    launch_wide<T, 16>(p, s);
  else
    launch_wide<T, 32>(p, s);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_qk_norm(const QkNormParams& p, int bf16, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, stream) : launch_t<__half>(p, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(qk_norm_device_error)

}  // namespace msst
