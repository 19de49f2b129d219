// cache_plan.cu — block tables and slots of a paged cache from request lengths.
//
// Free pages are a stack.  Requests that have ended push their pages, in order of
// requests; then requests that grow pop theirs, in the same order, so the result is a
// function of the arguments alone: with the sums back(r) and need(r) over the requests before r,
//   free[count + back(r) + b] = table[r][b]              of an ended request,
//   table[r][have(r) + b] = free[top - 1 - need(r) - b]  of one that grows.
// Every CTA of a cluster scans all requests for itself (a few KB), so that a page or a
// token can be placed by any thread; lengths and count, which may be updated in place, are written only past the
// cluster's barrier.
//
// Bound: latency (two scans and a chain of three loads): 64 requests of one token 3.8 us, 1024 requests 7.6, prompts of
// 48060 tokens (384 KB written) on eight CTAs 9.8.  With three scans of 1024 threads for whatever sizes: 8.5, 11.0, 12.4.
#include <algorithm>

#include "cache_ops.cuh"
#include "common.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr int kMostThreads = 1024, kCtas = 8;

// Exclusive sums over the block's threads of N values at once, and the totals.
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long (*s_warp)[2], long long (&total)[N]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  long long incl[N];
#pragma unroll
  for (int i = 0; i < N; ++i) incl[i] = v[i];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const long long x = __shfl_up_sync(0xffffffffu, incl[i], o);
      if (lane >= o) incl[i] += x;
    }
  }
  if (lane == 31) {
#pragma unroll
    for (int i = 0; i < N; ++i) s_warp[warp][i] = incl[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // the warps' sums, one a lane, summed by every warp for itself
    long long x = lane < warps ? s_warp[lane][i] : 0;
    const long long own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    total[i] = __shfl_sync(0xffffffffu, x, 31);
    v[i] = incl[i] - v[i] + __shfl_sync(0xffffffffu, x - own, warp);
  }
}

// The last i of [0, n) with a[i] <= x (a[0] <= x).
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0;
  for (int len = n; len > 1;) {
    const int half = len >> 1;
    if (a[lo + half] <= x) lo += half;
    len -= half;
  }
  return lo;
}

__device__ __forceinline__ int clamp_int(long long v) { return (int)min(v, 0x7fffffffLL); }

__global__ void __launch_bounds__(kMostThreads) cache_plan_kernel(const __grid_constant__ CachePlanParams p) {
  extern __shared__ int s_mem[];
  const int R = p.requests, page = 1 << p.page_shift;
  int* s_start = s_mem;             // [R + 1] first row
  int* s_back = s_start + R + 1;    // [R + 1] pages given back before
  int* s_need = s_back + R + 1;     // [R + 1] pages taken before
  int* s_kept = s_need + R + 1;     // [R] tokens there already, negative (~) where the request is refused
  __shared__ long long s_warp[2][32][2];
  __shared__ int s_got, s_refused;
  const int tid = threadIdx.x, per = (R + blockDim.x - 1) / blockDim.x;
  const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
  const unsigned rank = cluster_ctarank(), stride = gridDim.x * blockDim.x, first = rank * blockDim.x + tid;
  const int most = (int)min((long long)p.blocks << p.page_shift, 0x7fffffffLL);
  if (tid == 0) s_got = s_refused = 0;

  const int count = min(max(*p.free_count, 0), p.pages);
  long long sums[2] = {0, 0};  // pages given back, new rows
  for (int r = r0; r < r1; ++r) {
    const int n = p.new_tokens[r], len = min(max(p.lens[r], 0), most);
    s_kept[r] = n < 0 ? 0 : len;
    s_back[r] = n < 0 ? (int)(((long long)len + page - 1) >> p.page_shift) : 0;
    s_start[r] = max(n, 0);
    sums[0] += s_back[r];
    sums[1] += max(n, 0);
  }
  long long all[2], need[1] = {0}, all_need[1];
  block_scan<2>(sums, s_warp[0], all);
  for (int r = r0; r < r1; ++r) {
    const int n = s_start[r], kept = s_kept[r], b = s_back[r];
    const long long after = (long long)kept + n;
    const bool wide = after > most || sums[1] + n > p.tokens;
    s_need[r] = wide ? -1 : (int)(((after + page - 1) >> p.page_shift) - (((long long)kept + page - 1) >> p.page_shift));
    need[0] += max(s_need[r], 0);
    s_start[r] = (int)min(sums[1], (long long)p.tokens);
    s_back[r] = clamp_int(sums[0]);
    sums[1] += n;
    sums[0] += b;
  }
  const long long all_back = all[0];
  if (tid == 0) {
    s_start[R] = (int)min(all[1], (long long)p.tokens);
    s_back[R] = clamp_int(all_back);
  }
  block_scan<1>(need, s_warp[1], all_need);
  const int top = (int)min(count + all_back, (long long)p.pages);
  for (int r = r0; r < r1; ++r) {
    const int n = s_need[r];
    const bool fits = n == 0 || (n > 0 && need[0] + n <= top);
    s_need[r] = clamp_int(need[0]);
    need[0] += max(n, 0);
    if (!fits) {
      s_kept[r] = ~s_kept[r];
      s_refused = 1;
    } else if (n > 0) {
      atomicMax(&s_got, (int)need[0]);
    }
  }
  if (tid == 0) s_need[R] = clamp_int(all_need[0]);
  __syncthreads();
  // pages of ended requests go on top of the stack
  for (long long i = first; i < s_back[R] && count + i < p.pages; i += stride) {
    const int r = last_at_most(s_back, R + 1, (int)i);
    p.free_pages[count + i] = p.table[r * p.table_stride + (i - s_back[r])];
  }
  // Every CTA has read the old lengths and count, and the stack is whole.
  cluster_sync_all();
  if (first == 0) {
    *p.out_count = top - s_got;
    p.q_starts[R] = s_start[R];
    if (s_refused) record_error(kErrCacheFull);
  }
  for (unsigned r = first; r < R; r += stride) {
    const int kept = s_kept[r], n = max(p.new_tokens[r], 0);
    p.out_lens[r] = kept < 0 ? ~kept : kept + n;
    p.q_starts[r] = s_start[r];
  }
  // pages come off its top
  for (long long x = first; x < s_got; x += stride) {
    const int i = (int)x, r = last_at_most(s_need, R + 1, i);
    const long long have = ((long long)s_kept[r] + page - 1) >> p.page_shift;
    p.table[r * p.table_stride + have + (i - s_need[r])] = __ldcg(p.free_pages + top - 1 - i);
  }
  for (long long x = first; x < p.tokens; x += stride) {
    const int t = (int)x;
    int slot = -1, position = 0;
    if (t < s_start[R]) {
      const int r = last_at_most(s_start, R + 1, t);
      const int kept = s_kept[r];
      // (a refused request's rows may pass what the host has checked the sum of start and a row of the table for)
      const long long place = (long long)(kept < 0 ? ~kept : kept) + (t - s_start[r]);
      position = clamp_int(p.start + place);
      if (kept >= 0) {
        const int at = (int)place;
        const int have = (int)(((long long)kept + page - 1) >> p.page_shift), b = at >> p.page_shift;
        const int at_page = b < have ? p.table[r * p.table_stride + b]
                                     : __ldcg(p.free_pages + top - 1 - (s_need[r] + b - have));
        slot = (int)(((unsigned)at_page << p.page_shift) + (unsigned)(at & (page - 1)));
      }
    }
    p.slots[t] = slot;
    p.positions[t] = position;
  }
}

}  // namespace

cudaError_t launch_cache_plan(const CachePlanParams& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured;
  constexpr int most = (4 * kMostPlanRequests + 3) * (int)sizeof(int);
  cudaError_t e = ensure_smem_limit(cache_plan_kernel, most, configured);
  if (e != cudaSuccess) return e;
  // a thread a request or row, while there are few; one CTA's barrier is the cheaper one
  const int ctas = p.tokens > 4096 ? kCtas : 1;
  const int wanted = std::max(p.requests, std::min(p.tokens / ctas, kMostThreads));
  const int threads = std::min(kMostThreads, std::max(128, (wanted + 31) & ~31));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = ctas;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = (4 * p.requests + 3) * sizeof(int);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)ctas, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  LaunchScope scope("cache_plan", 0.0, 20.0 * p.requests + 8.0 * p.tokens, stream);
  return cudaLaunchKernelEx(&cfg, cache_plan_kernel, p);
}

MSST_DEFINE_ERROR_ACCESSOR(cache_plan_device_error)

}  // namespace msst
