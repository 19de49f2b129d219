// rope_append.cu — the position rotation of queries and keys, whose keys go to the pages
// of a cache with their values.
//
// A pair (a, b) becomes amplitude (a cos - b sin, b cos + a sin) of the angle position * freq:
// turns = position * freq / 2 pi and its distance from the next whole number in 64 bits, since fp32
// positions of a million would leave 0.06 radians of the fastest pair; sine and cosine of what is
// left (at most half a turn) in fp32.  Frequencies scaled for long contexts are just other ones, so
// there is no table to fetch, and one of 2^20 positions would be 512 MB.
//
// 8 columns a lane, a group of lanes (the power of two that covers head_dim / 8) takes four heads of a
// token, so a lane's four angles serve four heads.
// Bound: HBM: 403 MB (16384 tokens, 32 + 8 + 8 heads of 128) in 62 us, 6.5 TB/s, with loads and stores marked as streaming
// above L2's size; 5685 tokens of 8 + 8 + 8 heads of 48 6.6 us (4.0 TB/s), one token of 64 requests 2.7 us.
#include "cache_ops.cuh"
#include "common.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr int kHeads = 4;
constexpr int kThreads = 128;

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

template <typename T, int LPV, bool kHalves, bool kStream>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const __grid_constant__ RopeAppendParams p, unsigned items,
                                                               int chunks_q, int chunks_k) {
  const unsigned item = qk_norm_item(blockIdx.x, threadIdx.x, LPV);
  const int l = threadIdx.x % LPV;
  if (item >= items || 8 * l >= p.head_dim) return;
  const unsigned chunks = chunks_q + 2 * chunks_k;
  const unsigned token = item / chunks;
  int chunk = (int)(item - token * chunks);
  const int which = chunk < chunks_q ? 0 : (chunk < chunks_q + chunks_k ? 1 : 2);
  if (which) chunk -= which == 1 ? chunks_q : chunks_q + chunks_k;
  const HeadsView& in = which == 0 ? p.q : (which == 1 ? p.k : p.v);
  const HeadsView& to = which == 0 ? p.out_q : (which == 1 ? p.k_cache : p.v_cache);
  const int h0 = chunk * kHeads, left = in.heads - h0;
  T* dst = static_cast<T*>(to.data) + h0 * to.head_stride;
  if (which == 0) {
    dst += token * to.seq_stride;
  } else {
    const int slot = __ldg(p.slots + token);
    if (slot < 0) return;
    if (slot >= p.num_slots) {
      record_error(kErrSlot);
      return;
    }
    dst += (slot >> p.page_shift) * to.batch_stride + (slot & ((1 << p.page_shift) - 1)) * to.seq_stride;
  }
  const int half = p.rot_dim >> 1;
  const bool turned = which < 2 && 8 * l < p.rot_dim;
  const int c0 = kHalves && turned ? 4 * l : 8 * l, c1 = kHalves && turned ? half + 4 * l : 8 * l + 4;
  const T* src = static_cast<const T*>(in.data) + token * in.seq_stride + h0 * in.head_stride;

  uint2 raw[kHeads][2];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    raw[u][0] = raw[u][1] = make_uint2(0u, 0u);
    if (u < left) {
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
  float co[4], si[4];
  if (turned) {
    const double at = (double)__ldg(p.positions + token);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      double turns = at * (__ldg(p.freq + 4 * l + i) * 0.15915494309189535);  // 1 / 2 pi
      turns -= rint(turns);
      sincospif((float)(2.0 * turns), &si[i], &co[i]);
      si[i] *= p.amplitude;
      co[i] *= p.amplitude;
    }
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    if (u >= left) break;
    if (turned) {
      float x[8];
      unpack2<T>(raw[u][0].x, x[0], x[1]);
      unpack2<T>(raw[u][0].y, x[2], x[3]);
      unpack2<T>(raw[u][1].x, x[4], x[5]);
      unpack2<T>(raw[u][1].y, x[6], x[7]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // kHalves: (x[i], x[4 + i]); interleaved: (x[2i], x[2i + 1])
        float& a = kHalves ? x[i] : x[2 * i];
        float& b = kHalves ? x[4 + i] : x[2 * i + 1];
        const float t = a * co[i] - b * si[i];
        b = b * co[i] + a * si[i];
        a = t;
      }
      raw[u][0] = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
      raw[u][1] = make_uint2(pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
    T* t = dst + u * to.head_stride;
    if constexpr (kHalves) {
      store<kStream>(reinterpret_cast<uint2*>(t + c0), raw[u][0]);
      store<kStream>(reinterpret_cast<uint2*>(t + c1), raw[u][1]);
    } else {
      store<kStream>(reinterpret_cast<uint4*>(t + c0), make_uint4(raw[u][0].x, raw[u][0].y, raw[u][1].x, raw[u][1].y));
    }
  }
}

template <typename T, int LPV>
void launch_lpv(const RopeAppendParams& p, cudaStream_t s) {
  const int cq = (p.q.heads + kHeads - 1) / kHeads, ck = (p.k.heads + kHeads - 1) / kHeads;
  const unsigned items = (unsigned)((long long)p.tokens * (cq + 2 * ck));
  const unsigned grid = (unsigned)(((long long)items * LPV + kThreads - 1) / kThreads);
  // more than L2 (126 MB) holds is streamed
  const bool stream = 4.0 * p.tokens * (p.q.heads + 2 * p.k.heads) * p.head_dim > 126e6;
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(p, items, cq, ck); };
  if (p.halves)
    stream ? go(rope_append_kernel<T, LPV, true, true>) : go(rope_append_kernel<T, LPV, true, false>);
  else
    stream ? go(rope_append_kernel<T, LPV, false, true>) : go(rope_append_kernel<T, LPV, false, false>);
}

template <typename T>
cudaError_t launch_t(const RopeAppendParams& p, cudaStream_t s) {
  const double values = (double)p.tokens * (p.q.heads + 2 * p.k.heads) * p.head_dim;
  LaunchScope scope("rope_append", 3.0 * values, 4.0 * values + 8.0 * p.tokens, s);
  if (p.head_dim <= 32)
    launch_lpv<T, 4>(p, s);
  else if (p.head_dim <= 64)
    launch_lpv<T, 8>(p, s);
  else if (p.head_dim <= 128)
    launch_lpv<T, 16>(p, s);
  else
    launch_lpv<T, 32>(p, s);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope_append(const RopeAppendParams& p, int bf16, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, stream) : launch_t<__half>(p, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(rope_append_device_error)

}  // namespace msst
