// prefix_attn.cu — attention of a batch's new tokens to a prefix that all requests share and to
// each request's own tokens in the pages of a cache, causal among the new ones.
//
// With the keys of row i split in the prefix's and the request's own, softmax(s) v is the joined
// result of two attentions with a running reference and sum each.  So the prefix's part takes the
// rows of ALL requests at once: the group's query heads of every token are packed into 128-row
// tiles and each K/V tile of the prefix is read for 256 rows, not for a request's few.  The own
// part has an item for each request and key head.
//
// One launch does both, with one CTA an SM.  Items are cut into units, in two sequences:
//   tile items   more than 16 rows a key head: tcgen05, pairs of 128-row tiles of one key head (tile_role, as
//                cross_attn.cu); a unit is a K/V tile of 128 keys for a pair, two for a lone tile
//   token items  up to 16 rows, a request's single token or a few: mma.sync (token_role), up to eight key heads at a
//                time; a unit is a K/V tile of 32 keys of these heads
// Every CTA sums the units of both from the lengths (find_runs), shares the CTAs out by what a unit of each
// costs and takes an equal contiguous run of its sequence.  The prefix's products and the reading of the
// requests' own pages so overlap, and the host knows nothing but the tensors' sizes (a captured call may be
// replayed with other lengths).  The parts of a row are joined by a second launch in a fixed order.
//
// A call whose requests have 256 rows of a key head and more on average (all that the host knows) takes prefix and own keys
// as one sequence instead: the rows of one request fill the tiles, and only the items that the runs cut are joined.
// Each request then reads the prefix for its own rows, a single token among the prompts too.
//
// What a row does not see is selected away; V rows past a request's last token are zeroed in shared memory
// before the product.  The V rows of new tokens cannot be, as later rows see them: where one of
// those holds infinities or NaN (0 * NaN would reach the rows before), these values alone are zeroed, and the joining
// launch adds them to the rows that see them (a weight is above 0, so that it does not matter to an infinity or NaN).
//
// Measured (one B200, both launches, in a CUDA graph) and what bounds it:
//   64 requests, one token each, 8192 keys of prefix, up to 1024 own, 32/8 heads of 128: 48 us.  Memory: 173 MB, most of
//     them at 6 TB/s; 8 us before the first tiles, then CTAs of equal runs end between 29 and 41 us, as the SMs do
//     not share the memory's rate equally (with the two kinds of CTA taking turns over the grid, 6 us more)
//   16 tokens, 131072 keys of prefix: 107 us, 555 MB at 5.2 TB/s
//   4096 tokens of six prompts, 4096 keys of prefix: 332 us back to back (power-capped), 303 after a pause, 1.06 PFLOP/s;
//     tensor and XU pipe 58 % busy each (the chain scores, softmax, product behind one buffer of scores a tile, as in
//     cross_attn.cu)
//   32 requests of 5 tokens, 3791 keys, 12/4 heads of 80: 25 to 28 us, all of it latency: 2.5 us to find the runs, 4 to the first
//     tile, three or four units, 2 to the second launch and 5 in it.  Code counts here: "no instruction" is the warps' first
//     stall, and forms that are written once and rolled up (the product's issue, the exact passes, barriers) are the faster ones
#include <algorithm>
#include <cstddef>

#include "attn_steps.cuh"
#include "cache_ops.cuh"
#include "common.cuh"
#include "cross_attn.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr int kThreads = 384;
constexpr int kSoftmaxWarp0 = 4;
constexpr int kFewRegs = 88, kSoftmaxRegs = 208;  // 128 x 88 + 256 x 208 = 384 x 168, as cross_attn.cu
constexpr uint32_t kHalfBytes = 128 * 64 * 2;     // 128 rows x 64 columns
constexpr int kTokenKeys = 32, kTokenShift = 5;   // a token item's K/V tile
constexpr uint32_t kTokenBox = kTokenKeys * 128;  // 32 keys x 64 columns
constexpr int kTokenWarps = 8;                    // that multiply; the other four bring tiles, one a team
constexpr int kMostTeams = 4, kMostEntries = 12;
// Steps of a row tile whose products add up in TMEM (a power of two).  The tensor core cuts what it adds off near 2^-26 of
// the sum so far, so that values of one sign lose 2^-27 of the sum with each key: 8e-4 of the result behind 131072 keys, 1.3 %
// behind 2 million.  After 16384 keys (fp16) or 65536 (bf16), 2^-13 and 2^-11, O goes to memory, where it is added
// in fp32, rounded to nearest.  (A prompt of 4096 tokens behind 131072 keys, bf16, 32/8 heads of 128: 8.6 ms without, 8.9
// so, 9.1 with every 8192 keys.  A step that puts O away takes the exact passes, whose wait it needs.)
template <typename T>
constexpr int kSumSteps = std::is_same<T, __half>::value ? 128 : 512;
constexpr int kLeftOut = -1;                       // less the worker's place: infinities and NaN are yet to be added

template <int DP>
struct PCfg {
  static constexpr int kHalves = DP / 64;
  static constexpr uint32_t kTile = kHalves * kHalfBytes;  // one Q, K or V tile
  static constexpr int kKSlots = DP == 128 ? 3 : 5, kVSlots = DP == 128 ? 2 : 5;
  static constexpr uint32_t kTiles = (2 + kKSlots + kVSlots) * kTile;
  static constexpr uint32_t kTail = 3 * 1024;  // segments, barriers and exchange of either role
  static constexpr size_t kSmem = kTiles + kTail;
  static_assert(kSmem <= 227 * 1024, "");
  static constexpr uint32_t kEntry = kHalves * kTokenBox;  // token role: K or V of one head and tile
  static constexpr int kBufs = DP == 128 ? 2 : 3;
  static constexpr uint32_t kColO = kBufs * 128;
};

// What the host knows of a launch.
struct PrefixGeom {
  int kv_heads, group;
  int gt, nt, g_tiles;        // heads and tokens of a row tile, tiles along the group
  int ksteps;
  int concat;                 // an item's keys are the prefix's and then its own (no items for the prefix alone)
  int prefix_tiles, prefix_tiles32;
  int prefix_token;           // all rows of a key head are at most 16: the prefix's item is a token item
  int n_tiles, full, lone;    // the prefix's tile items
  int box;                    // rows of a cache's TMA box
  int pk_headed, pv_headed, kc_headed, vc_headed;  // 0: key heads share one (stride 0)
  int heads, groups, teams;   // token items: key heads of an item, items of a request, teams of a CTA
  int entries, q_rows, q_slots;  // of a team: K or V tiles of all its heads, query rows a head, segments of those
  int tile_rows, token_rows, ld;  // rows of a partial result's slot (tile items, token items), floats of a row
  int tile_cost, token_cost;  // of a unit
  int tile_item, token_item;  // of an item's start and end, in units
  int* where;                 // [phase][tokens * q_heads] which partial results a row has
  float* tile_slots;          // [CTA][begins, ends][tile_rows][ld]
  float* token_slots;         // [CTA * teams][begins, ends][heads][token_rows][ld]
  float* whole;               // [phase][tokens * q_heads][ld] results of items that one worker had whole
  struct Segment* cuts;       // [CTA][teams] the item that the worker started and did not end (code 0: none)
  int* bad;                   // [CTA][teams] whether values have been left out of one of the worker's whole items
};

struct Request {
  int q0, n, own;  // first row, rows, own tokens
  // own tokens that row i sees
  __device__ __forceinline__ int limit(int i) const { return min(max(own - n + 1 + i, 0), own); }
};

__device__ __forceinline__ int first_row(const PrefixAttnParams& p, int r) {
  return p.q_starts ? min(max(__ldg(p.q_starts + r), 0), p.tokens) : r;
}
__device__ __forceinline__ Request load_request(const PrefixAttnParams& p, int r) {
  Request q;
  q.q0 = first_row(p, r);
  q.n = p.q_starts ? max(first_row(p, r + 1) - q.q0, 0) : 1;
  q.own = (int)min((long long)max(__ldg(p.lens + r), 0), (long long)p.blocks << p.page_shift);
  return q;
}
__device__ __forceinline__ bool is_token(const PrefixGeom& g, const Request& q) {
  return (long long)q.n * g.group <= kTokenRows;
}

// The items of one request (or, phase 0, of all rows against the prefix) for a key head.
struct Items {
  int n_tiles, full, lone;
  __device__ __forceinline__ Items() {}
  __device__ __forceinline__ Items(const PrefixGeom& g, const Request& q, bool token) {
    if (token) {
      n_tiles = full = 1, lone = 0;
    } else {
      n_tiles = (q.n + g.nt - 1) / g.nt;
      const int tiles = n_tiles * g.g_tiles;
      full = tiles >> 1, lone = tiles & 1;
    }
  }
  // K/V tiles of item t: `ptiles` of the prefix, then the own ones that its last row sees
  __device__ __forceinline__ int tiles(const PrefixGeom& g, const Request& q, bool token, int t, int ptiles) const {
    int end = q.n;
    if (!token) {
      const int a = 2 * t, b = t < full ? a + 1 : a;
      const int last = g.g_tiles == 1 ? b : max(a % n_tiles, b % n_tiles);  // (along the group the tokens start over)
      end = min((last + 1) * g.nt, q.n);
    }
    const int keys = q.own ? q.limit(end - 1) : 0, shift = token ? kTokenShift : 7;
    return max(1, ptiles + ((keys + (1 << shift) - 1) >> shift));
  }
  __device__ __forceinline__ int units(int t, int tiles) const { return t < full ? tiles : (tiles + 1) >> 1; }
  // What the item counts for in the sharing out: its units, and the start and end of an item in units
  __device__ __forceinline__ int weight(int t, int tiles, const PrefixGeom& g, bool token) const {
    return units(t, tiles) + (token ? g.token_item : g.tile_item);
  }
  __device__ __forceinline__ long long head_weight(const PrefixGeom& g, const Request& q, bool token, int ptiles) const {
    long long sum = 0;
    for (int t = 0; t < full + lone; ++t) sum += weight(t, tiles(g, q, token, t, ptiles), g, token);
    return sum;
  }
};

__device__ __forceinline__ int prefix_part(const PrefixGeom& g, bool token) {
  return token ? g.prefix_tiles32 : g.prefix_tiles;
}
// Weight of the prefix's own items in the sequence of token or tile items.
__device__ __forceinline__ long long prefix_weight(const PrefixGeom& g, bool token) {
  if (g.concat || (bool)g.prefix_token != token) return 0;
  if (token) return (long long)g.groups * (g.prefix_tiles32 + g.token_item);
  return (long long)g.kv_heads * ((long long)g.full * (g.prefix_tiles + g.tile_item) +
                                  g.lone * (((prefix_part(g, false) + 1) >> 1) + g.tile_item));
}

// The run of a worker, a CTA (tile items) or a team of its warps (token items): weights [u0, u0 + count) of the U of
// its sequence, worker `self` of `workers`; where it starts.
struct Run {
  long long u0, count, U;
  int token, self, workers, place;  // place: among the teams of all CTAs, the tile items' as team 0
  int phase, r, hk, t, j;
};

// Exclusive sums over the CTA's threads of two values, and the totals (s: two slots a warp).
struct Two {
  long long a, b;
};
__device__ __forceinline__ Two cta_scan(Two v, Two* s, Two& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Two incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl.a, o), y = __shfl_up_sync(0xffffffffu, incl.b, o);
    if (lane >= o) incl.a += x, incl.b += y;
  }
  if (lane == 31) s[warp] = incl;
  __syncthreads();
  Two before{0, 0};
  total = before;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const Two x = s[w];
    if (w < warp) before.a += x.a, before.b += x.b;
    total.a += x.a, total.b += x.b;
  }
  __syncthreads();
  return Two{before.a + incl.a - v.a, before.b + incl.b - v.b};
}

// a b / c; a 32-bit division (a fifth of the time) where the numbers allow one.
__host__ __device__ __forceinline__ long long mul_div(long long a, long long b, long long c) {
  const unsigned long long n = (unsigned long long)a * (unsigned long long)b;
  return (n | (unsigned long long)c) >> 32 ? (long long)(n / (unsigned long long)c)
                                           : (long long)((unsigned)n / (unsigned)c);
}

// All threads: the run of this CTA, or of each of its teams, from the lengths of all requests.
__device__ void find_runs(const PrefixAttnParams& p, const PrefixGeom& g, Run* runs, Two* scratch) {
  const int R = p.requests, tid = threadIdx.x;
  // weight of request r for a key head: .a as tile items, .b as a token item (for a group of heads)
  auto weights = [&](int r) -> Two {
    if (r >= R) return Two{0, 0};
    const Request q = load_request(p, r);
    if (q.n == 0) return Two{0, 0};
    const bool token = is_token(g, q);
    const long long u = Items(g, q, token).head_weight(g, q, token, g.concat ? prefix_part(g, token) : 0);
    return token ? Two{0, u} : Two{u, 0};
  };
  Two mine{0, 0}, total;
  for (int r = tid; r < R; r += kThreads) {
    const Two x = weights(r);
    mine.a += x.a, mine.b += x.b;
  }
  Two before = cta_scan(mine, scratch, total);
  const long long pre_a = prefix_weight(g, false), pre_b = prefix_weight(g, true);
  const long long total_a = total.a * g.kv_heads + pre_a, total_b = total.b * g.groups + pre_b;
  // CTAs of the tile items and of the token items, by what their units cost
  const int G = (int)gridDim.x;
  const float cost_a = (float)total_a * g.tile_cost, cost_b = (float)total_b * g.token_cost;
  int ca = cost_a + cost_b > 0.f ? (int)(G * (cost_a / (cost_a + cost_b)) + 0.5f) : 0;
  if (total_a > 0) ca = max(ca, 1);
  if (total_b > 0) ca = min(ca, G - 1);
  const bool token = (int)blockIdx.x >= ca;
  Run x{};
  x.token = token;
  x.U = token ? total_b : total_a;
  // as many workers as units at most, so that none between two others is without any
  x.workers = (int)min(x.U, (long long)(token ? (G - ca) * g.teams : ca));
  const int own_runs = token ? g.teams : 1, self0 = token ? (int)(blockIdx.x - ca) * g.teams : (int)blockIdx.x;
  const int items = token ? g.groups : g.kv_heads;  // of a request (for each pair of row tiles)
  const long long pre = token ? pre_b : pre_a;
  auto run_of = [&](int w) {  // the run without its start
    Run y = x;
    y.self = self0 + w;
    y.place = (int)blockIdx.x * g.teams + w;
    if (y.self < x.workers) {
      y.u0 = mul_div(x.U, y.self, x.workers);
      y.count = mul_div(x.U, y.self + 1, x.workers) - y.u0;
    }
    return y;
  };
  if (tid < own_runs) {
    Run y = run_of(tid);
    if (y.count > 0 && y.u0 < pre) {
      const long long head = pre / items;
      const int each = prefix_part(g, token) + (token ? g.token_item : g.tile_item);
      y.hk = (int)mul_div(y.u0, 1, head);
      const long long off = y.u0 - y.hk * head, pairs = token ? each : (long long)g.full * each;
      y.t = off < pairs ? (int)mul_div(off, 1, each) : g.full;
      y.j = (int)(off < pairs ? off - (long long)y.t * each : off - pairs);
    }
    runs[tid] = y;
  }
  __syncthreads();
  long long base = pre;
  for (int r0 = 0; r0 < R; r0 += kThreads) {
    if (R > kThreads) {  // (else this is what was summed above)
      mine = weights(r0 + tid);
      before = cta_scan(mine, scratch, total);
    }
    const long long head = token ? mine.b : mine.a, from = base + (token ? before.b : before.a) * items;
    for (int w = 0; head > 0 && w < own_runs; ++w) {
      const long long u0 = runs[w].u0;
      if (runs[w].count == 0 || u0 < from || u0 >= from + head * items) continue;
      const Request q = load_request(p, r0 + tid);
      const Items it(g, q, token);
      const int ptiles = g.concat ? prefix_part(g, token) : 0;
      Run y = runs[w];
      y.phase = 1;
      y.r = r0 + tid;
      y.hk = (int)mul_div(u0 - from, 1, head);
      long long off = u0 - from - y.hk * head;
      for (y.t = 0;; ++y.t) {
        const int u = it.weight(y.t, it.tiles(g, q, token, y.t, ptiles), g, token);
        if (off < u) break;
        off -= u;
      }
      y.j = (int)off;
      runs[w] = y;
    }
    base += (token ? total.b : total.a) * items;
  }
  __syncthreads();
}

// The worker that weight u falls to.
__device__ __forceinline__ int worker_of(long long u, const Run& run) {
  return (int)(((u + 1) * run.workers - 1) / run.U);
}

// One segment of a run: an item, or the part [j0, j1) of its units.
struct Segment {
  int q0, n, own;             // the request's first row, rows, own tokens (phase 0: all rows, none)
  int r, hk, phase;           // (token items: hk the group of key heads)
  int ptiles, tiles, units;   // K/V tiles of the prefix, K/V tiles and units in all
  int j0, j1;
  int lone, tile0, n_tiles;   // tile items: row tile(s) tile0, tile0 + 1 of n_tiles along the tokens
  int last;                   // 1: no segment, the run's end
  int code;                   // see below
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == units; }
  // own tokens that row i sees
  __device__ __forceinline__ int limit(int i) const { return Request{q0, n, own}.limit(i); }
  // tile items: K/V tile of row tile w in unit j, and whether it has one
  __device__ __forceinline__ int kv_tile(int w, int j) const { return lone ? 2 * j + w : j; }
  __device__ __forceinline__ bool uses(int w, int j) const { return kv_tile(w, j) < tiles; }
  // first token (of the item's rows) and head of row tile w
  __device__ __forceinline__ void origin(const PrefixGeom& g, int w, int& n0, int& g0) const {
    const int tile = tile0 + (lone ? 0 : w), gi = tile / n_tiles;
    n0 = (tile - gi * n_tiles) * g.nt;
    g0 = gi * g.gt;
  }
  // A partial result's slot of this worker
  __device__ __forceinline__ float* tile_slot(const PrefixGeom& g, const Run& run) const {
    return g.tile_slots + (size_t)(2 * run.self + (j0 > 0)) * g.tile_rows * g.ld;
  }
  __device__ __forceinline__ float* token_slot(const PrefixGeom& g, const Run& run, int h) const {
    return g.token_slots + (size_t)((2 * run.self + (j0 > 0)) * g.heads + h) * g.token_rows * g.ld;
  }
};
static_assert(sizeof(Segment) == 64, "");

// Where the parts of an item are, written for each of its rows by the worker that starts it.  Bits: the row of a
// slot (added by the writer), << 8 the first worker (those of tile items from kTileWorkers on), << 20 how many
// workers follow it (0: one had it whole).
constexpr int kTileWorkers = 2048;

// Walks the segments of a run.
struct ItemWalk {
  const PrefixAttnParams& p;
  const PrefixGeom& g;
  const Run& run;
  int phase, r, hk, t, j, ptiles;
  long long at, end;
  Request q, ahead;  // this item's request, and the next one (asked for before it is needed)
  Items it;
  __device__ __forceinline__ ItemWalk(const PrefixAttnParams& p_, const PrefixGeom& g_, const Run& x)
      : p(p_), g(g_), run(x), phase(x.phase), r(x.r), hk(x.hk), t(x.t), j(x.j), at(x.u0), end(x.u0 + x.count) {
    if (at >= end) return;
    if (phase == 1) ask(r);
    set_request();
  }
  __device__ __forceinline__ void ask(int i) {
    if (i < p.requests) ahead = load_request(p, i);
  }
  __device__ __forceinline__ void set_request() {
    const bool token = run.token;
    if (phase == 0)
      q.q0 = 0, q.n = p.tokens, q.own = 0;
    else
      q = ahead;
    it = Items(g, q, token);
    ptiles = phase == 0 || g.concat ? prefix_part(g, token) : 0;
    ask(phase == 0 ? 0 : r + 1);
  }
  // The next segment (x.last: none)
  __device__ __forceinline__ void next(Segment& x) {
    const bool token = run.token;
    for (;;) {
      x.last = at >= end;
      if (x.last) return;
      x.q0 = q.q0, x.n = q.n, x.own = q.own;
      x.r = r, x.hk = hk, x.phase = phase;
      x.ptiles = ptiles;
      x.tiles = it.tiles(g, q, token, t, ptiles);
      x.units = it.units(t, x.tiles);
      x.j0 = j;
      x.j1 = (int)min((long long)x.units, j + (end - at));
      x.lone = t == it.full;
      x.tile0 = 2 * t;
      x.n_tiles = it.n_tiles;
      x.code = 0;
      if (j == 0 && x.j1 < x.units) {
        const int more = worker_of(at + x.units - 1, run) - run.self;
        x.code = (run.self + (token ? 0 : kTileWorkers)) << 8 | more << 20;
      }
      at += it.weight(t, x.tiles, g, token) - j;
      j = 0;
      if (at < end && ++t == it.full + it.lone) {
        t = 0;
        if (++hk == (token ? g.groups : g.kv_heads)) {
          hk = 0;
          if (phase == 0) phase = 1, r = -1;
          do {
            if (++r >= p.requests) {  // not reached: weights are left
              at = end;
              break;
            }
            set_request();
          } while (q.n == 0 || is_token(g, q) != token);
        }
      }
      if (x.j0 < x.units) return;  // (a run that starts past an item's units has none of it)
    }
  }
};

// Tile items: the segments of a CTA's run in a ring in shared memory: one lane walks the items for all roles (in
// registers of every role the walk spilled 470 bytes, and local memory has little L1 beside the tiles).
constexpr int kRing = 4;
constexpr unsigned long long kUnitLimitNs = 20000;  // ten times what a unit takes
struct SegmentRing {
  Segment at[kRing];
  uint64_t full[kRing], empty[kRing];
  __device__ __forceinline__ void init(int readers, int lane) {
    if (lane < 2 * kRing) mbar_init(&full[lane], lane < kRing ? 1 : readers);
  }
  // The s-th segment once it is there; a warp's lanes together, or one lane alone
  __device__ __forceinline__ bool wait_warp(int s, volatile int* abort_flag) {
    return mbar_wait_warp<false>(&full[s % kRing], s / kRing & 1, kErrTimeoutAttnQ, abort_flag);
  }
  __device__ __forceinline__ bool wait(int s, volatile int* abort_flag) {
    return mbar_wait<false>(&full[s % kRing], s / kRing & 1, kErrTimeoutAttnQ, abort_flag);
  }
  // One lane: walks the run
  __device__ void fill(const PrefixAttnParams& p, const PrefixGeom& g, const Run& run, volatile int* abort_flag) {
    ItemWalk walk(p, g, run);
    for (int s = 0;; ++s) {
      Segment x;
      walk.next(x);
      // The place is free when the segment kRing before has ended: no step of a chain but all of its units
      const Segment& before = at[s % kRing];
      const unsigned long long more = s < kRing ? 0 : (unsigned long long)(before.j1 - before.j0) * kUnitLimitNs;
      if (!mbar_wait<false>(&empty[s % kRing], (s / kRing & 1) ^ 1, kErrTimeoutAttnQ, abort_flag, kWaitLimitNs + more))
        return;
      at[s % kRing] = x;
      mbar_arrive(&full[s % kRing]);
      if (x.last) return;
      if (x.code) g.cuts[run.place] = x;
    }
  }
};

// The page that own token `key` of request r is in; one outside the cache reads as zeros (TMA fills
// what lies outside a tensor) and is reported.
__device__ __forceinline__ int checked_page(const PrefixAttnParams& p, int page) {
  if ((unsigned)page < (unsigned)p.pages) return page;
  record_error(kErrPage);
  return p.pages;
}

// Eight floats to 32-byte aligned memory.
__device__ __forceinline__ void store8(float* to, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// Infinities and NaN among 16-bit values: the largest magnitudes so far, for the even and the odd ones, as whole
// numbers; theirs are the largest of all.
struct Magnitude {
  uint32_t top = 0;
  __device__ __forceinline__ void add(const uint4& v) {
    top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu));
    top = __vmaxu2(top, v.w & 0x7fff7fffu);
  }
  template <typename T>
  __device__ __forceinline__ bool finite() const {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return (top & 0xffffu) < e && top >> 16 < e;
  }
};
// Those of eight values that are neither.
template <typename T>
__device__ __forceinline__ uint4 finite_ones(uint4 v) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  auto pair = [](uint32_t x) {
    return ((x & 0x7fffu) < e ? x & 0xffffu : 0u) | ((x >> 16 & 0x7fffu) < e ? x & 0xffff0000u : 0u);
  };
  return make_uint4(pair(v.x), pair(v.y), pair(v.z), pair(v.w));
}

// ------------------------------------------------------------------------------- tile items
// Rows [lo, hi) of a V tile: infinities and NaN become zeros.  (Rare: out of the loop's way, as clear_keys below.)
template <typename T, int kHalves>
__device__ __noinline__ void leave_out(uint8_t* tile, int lo, int hi, int lane) {
#pragma unroll 1
  for (int row = lo + lane; row < hi; row += 32) {
#pragma unroll 1
    for (int x = 0; x < 8 * kHalves; ++x) {
      uint4* piece = reinterpret_cast<uint4*>(tile + row * 128 + (x >> 3) * kHalfBytes + (((x + lane) & 7) << 4));
      *piece = finite_ones<T>(*piece);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// O of a row (mem null: none that counts) after kSumSteps<T> steps: stored in memory, or added to what is there times
// beta; kBack: what is there times beta added to O.  A warp's lanes together.  (Out of the loop's way, as clear_keys below.)
enum Away { kStore, kAdd, kBack };
__device__ __noinline__ void put_away(uint32_t o, float* mem, int d, Away how, float beta) {
  const bool scaled = __any_sync(0xffffffffu, mem && beta != 1.f);
#pragma unroll 1
  for (int c0 = 0; c0 < d; c0 += 32) {
    uint32_t r[32];
    tmem_ld32(o + c0, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int u = 0; u < 32; u += 4) {
      if (!mem || c0 + u >= d) break;
      float* at = mem + c0 + u;
      float4 v = make_float4(__uint_as_float(r[u]), __uint_as_float(r[u + 1]), __uint_as_float(r[u + 2]),
                             __uint_as_float(r[u + 3]));
      if (how == kAdd && !scaled) {  // (the row's thread alone adds here: in the order of its steps)
        asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                     : "memory");
        continue;
      }
      if (how != kStore) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(at));
        v.x += beta * x.x, v.y += beta * x.y, v.z += beta * x.z, v.w += beta * x.w;
      }
      if (how != kBack) __stcg(reinterpret_cast<float4*>(at), v);
      r[u] = __float_as_uint(v.x), r[u + 1] = __float_as_uint(v.y);
      r[u + 2] = __float_as_uint(v.z), r[u + 3] = __float_as_uint(v.w);
    }
    __syncwarp();
    if (how == kBack) tmem_st32(o + c0, r);
  }
  if (how == kBack) tmem_st_wait();
}

template <typename T, int DP>
__device__ void tile_role(uint8_t* smem, const CUtensorMap& qmap, const CUtensorMap& pkmap, const CUtensorMap& pvmap,
                          const CUtensorMap& kcmap, const CUtensorMap& vcmap, const PrefixAttnParams& p,
                          const PrefixGeom& g, const Run& run) {
  using C = PCfg<DP>;
  constexpr uint32_t kIsBf16 = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr int NB = C::kBufs;
  using KPos = RingPos<C::kKSlots>;
  using VPos = RingPos<C::kVSlots>;
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * C::kTile;
  uint8_t* sV = sK + C::kKSlots * C::kTile;
  SegmentRing* ring = reinterpret_cast<SegmentRing*>(smem + C::kTiles);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + 1);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* s_full = bars + 2;    // [NB buffers]
  uint64_t* p_full = bars + 6;    // [NB buffers]
  uint64_t* pv_done = bars + 10;  // [2 tiles], every step
  uint64_t* o_done = bars + 12;   // [2 tiles], every item
  uint64_t* meet = bars + 14;     // [4 lane quarters]: the two halves of a lone tile
  uint64_t* mma_end = bars + 18;
  uint64_t* k_full = bars + 19;
  uint64_t* k_empty = k_full + C::kKSlots;
  uint64_t* v_full = k_empty + C::kKSlots;  // landed
  uint64_t* v_ready = v_full + C::kVSlots;  // fit for the MMA
  uint64_t* v_empty = v_ready + C::kVSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + C::kVSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* s_bad = tmem_slot + 2;                 // a bit a segment (mod 32): see warp 2
  float* s_ml = reinterpret_cast<float*>(tmem_slot + 4);    // [2 halves][ref, l][128]
  static_assert(sizeof(SegmentRing) + (19 + 2 * C::kKSlots + 3 * C::kVSlots) * 8 + 16 + 2048 <= C::kTail, "");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    // a lane a barrier: softmax warps' 128 threads arrive at p_full, the two halves at meet, one thread elsewhere
    constexpr int kBars = 19 + 2 * C::kKSlots + 3 * C::kVSlots;
    for (int i = lane; i < kBars; i += 32) mbar_init(&bars[i], i >= 6 && i < 10 ? 128 : (i >= 14 && i < 18 ? 2 : 1));
    ring->init(8, lane);  // the softmax warps are the last to need a segment
    if (lane == 0) {
      *abort_flag = 0;
      *s_bad = 0;
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int s = 0;  // every role walks the segments of the run

  if (warp < kSoftmaxWarp0) {
    warpgroup_reg_dec<kFewRegs>();
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        KPos kp;
        VPos vp;
        uint32_t q_phase = 0;
        bool ok = true;
        // K/V tile `tile` of the current item: whole boxes of the prefix (its end is filled with zeros), of
        // the own tokens the boxes that hold any
        auto load_tile = [&](const CUtensorMap& pre, int pre_headed, const CUtensorMap& cache, int cache_headed, uint8_t* dst,
                             uint64_t* bar, const Segment& k, int tile) {
          if (tile < k.ptiles) {
            mbar_arrive_expect_tx(bar, C::kTile);
            for (int h = 0; h < C::kHalves; ++h)
              for (int b = 0; b < 128 / kTokenKeys; ++b)
                tma_load_4d(dst + h * kHalfBytes + b * kTokenBox, &pre, bar, h * 64, tile * 128 + b * kTokenKeys,
                            k.hk * pre_headed, 0);
            return;
          }
          const int key0 = (tile - k.ptiles) * 128, boxes = min(128 / g.box, max(0, (k.own - key0 + g.box - 1) / g.box));
          mbar_arrive_expect_tx(bar, (uint32_t)(boxes * g.box) * 128u * C::kHalves);
          const int* row = p.table + k.r * p.table_stride;
          for (int b0 = 0; b0 < boxes; b0 += 4) {
            int page[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              page[i] = b0 + i < boxes ? __ldg(row + ((key0 + (b0 + i) * g.box) >> p.page_shift)) : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (b0 + i >= boxes) break;
              const int at = (key0 + (b0 + i) * g.box) & ((1 << p.page_shift) - 1), id = checked_page(p, page[i]);
              for (int h = 0; h < C::kHalves; ++h)
                tma_load_4d(dst + h * kHalfBytes + (b0 + i) * g.box * 128, &cache, bar, h * 64, at, k.hk * cache_headed, id);
            }
          }
        };
        for (; ok; ++s) {
          if (!(ok = ring->wait(s, abort_flag))) break;
          const Segment k = ring->at[s % kRing];
          if (k.last) break;
          if (!(ok = mbar_wait<false>(q_empty, q_phase ^ 1, kErrTimeoutAttnQ, abort_flag))) break;
          q_phase ^= 1;
          const int nq = k.lone ? 1 : 2;
          mbar_arrive_expect_tx(q_full, nq * C::kHalves * (uint32_t)(g.gt * g.nt) * 128u);
          for (int w = 0; w < nq; ++w) {
            int n0, g0;
            k.origin(g, w, n0, g0);
            for (int h = 0; h < C::kHalves; ++h)
              tma_load_4d(sQ + w * C::kTile + h * kHalfBytes, &qmap, q_full, h * 64, g0, k.q0 + n0, k.hk);
          }
          const int streams = k.lone ? 2 : 1;  // K/V tiles of a unit
          // with three buffers S runs ahead of PV by up to two units, so K goes first
          constexpr int kLead = NB == 3 ? 1 : 0;
          for (int i = k.j0; ok && i < k.j1 + kLead; ++i) {
            for (int w = 0; w < streams && i < k.j1 && k.uses(w, i); ++w) {
              if (!(ok = mbar_wait<false>(&k_empty[kp.slot], kp.phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
              load_tile(pkmap, g.pk_headed, kcmap, g.kc_headed, sK + kp.slot * C::kTile, &k_full[kp.slot], k,
                        k.kv_tile(w, i));
              kp = kp.plus(1);
            }
            const int v = i - kLead;
            for (int w = 0; ok && w < streams && v >= k.j0 && k.uses(w, v); ++w) {
              if (!(ok = mbar_wait<false>(&v_empty[vp.slot], vp.phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
              load_tile(pvmap, g.pv_headed, vcmap, g.vc_headed, sV + vp.slot * C::kTile, &v_full[vp.slot], k,
                        k.kv_tile(w, v));
              vp = vp.plus(1);
            }
          }
        }
        mbar_drain(q_full, q_phase ^ 1);
        mbar_drain_ring(k_full, C::kKSlots, kp.slot, kp.phase);
        mbar_drain_ring(v_full, C::kVSlots, vp.slot, vp.phase);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        const uint32_t idesc_s = umma_idesc_f16(kIsBf16, 128, 0);
        const uint32_t idesc_o = umma_idesc_f16(kIsBf16, (uint32_t)g.ksteps * 16, 1);
        const uint64_t dq0 = sw128_desc(smem_u32(sQ), 16, 1024);
        const uint64_t dk0 = sw128_desc(smem_u32(sK), 16, 1024);
        const uint64_t dv0 = sw128_desc(smem_u32(sV), kHalfBytes, 1024);
        constexpr uint32_t kTileDesc = C::kTile >> 4;
        const int ksteps = g.ksteps;
        KPos kp;  // next K and V slots to wait for
        VPos vp;
        uint32_t kslot = 0, vslot = 0, turns = 0;  // slots in use; parity of each tile's steps (two buffers)
        uint32_t seq = 0;  // position in the sequence of the segment's first step
        bool ok = true;
        for (; ok; ++s) {
          if (!(ok = ring->wait(s, abort_flag))) break;
          const Segment k = ring->at[s % kRing];
          if (k.last) break;
          if (!(ok = mbar_wait<false>(q_full, s & 1, kErrTimeoutAttnQ, abort_flag))) break;
          tc_fence_after();
          const int steps = k.j1 - k.j0;
          // steps of the second tile: all, but for a lone tile's last unit without a K/V tile for it
          const int steps1 = k.uses(1, k.j1 - 1) ? steps : steps - 1;
          const bool lone = k.lone;
          // Step n of the segment is step n / 2 of tile n % 2.  PV(n), and S(n + NB) behind it: NB scores ahead.
          // (One copy of either, as all of this is fetched while the first tile waits.)
#pragma unroll 1
          for (int n = -NB; n < 2 * steps; ++n) {
            if (n >= 0 && (n >> 1) < (n & 1 ? steps1 : steps)) {
              const int w = n & 1, t = n >> 1;
              if (w == 0 || lone) {
                if (!(ok = mbar_wait<false>(&v_ready[vp.slot], vp.phase, kErrTimeoutAttnKV, abort_flag))) break;
                vslot = vp.slot;
                vp = vp.plus(1);
              }
              const StepBuf<NB> b(w, turns >> w, seq + n);
              turns ^= 1u << w;
              if (!(ok = mbar_wait<false>(&p_full[b.buf], b.parity, kErrTimeoutAttnP, abort_flag))) break;
              tc_fence_after();
              const uint64_t dv = dv0 + (uint64_t)(vslot * kTileDesc);
              const uint32_t pa = tmem + b.buf * 128, dO = tmem + C::kColO + (uint32_t)(w * DP);
              umma_f16_ts(dO, pa, dv, idesc_o, (t & (kSumSteps<T> - 1)) != 0);
#pragma unroll
              for (int kk = 1; kk < 8; ++kk) umma_f16_ts(dO, pa + (uint32_t)(kk * 8), dv + 128 * kk, idesc_o, 1u);
              umma_commit(&pv_done[w]);
              if (w == 1 || lone) umma_commit(&v_empty[vslot]);
            }
            if (n == 2 * steps - 2) umma_commit(&o_done[0]);
            const int n2 = n + NB, w = n2 & 1;
            if ((n2 >> 1) < (w ? steps1 : steps)) {
              if (w == 0 || lone) {
                if (!(ok = mbar_wait<false>(&k_full[kp.slot], kp.phase, kErrTimeoutAttnKV, abort_flag))) break;
                kslot = kp.slot;
                kp = kp.plus(1);
                tc_fence_after();
              }
              const uint32_t dS = tmem + StepBuf<NB>(w, 0, seq + n2).buf * 128;
              const uint64_t dq = dq0 + (uint64_t)((lone ? 0 : w) * kTileDesc);
              const uint64_t dk = dk0 + (uint64_t)(kslot * kTileDesc);
#pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk) {
                if (kk >= ksteps) break;
                const uint64_t off = (uint64_t)((kk >> 2) * (kHalfBytes >> 4) + (kk & 3) * 2);
                umma_f16_ss(dS, dq + off, dk + off, idesc_s, kk != 0);
              }
              umma_commit(&s_full[StepBuf<NB>(w, 0, seq + n2).buf]);
              if (w == 1 || lone) umma_commit(&k_empty[kslot]);
            }
            if (n2 == 2 * steps - 1) umma_commit(q_empty);  // every S has been issued
          }
          if (ok) umma_commit(&o_done[1]);
          seq += (uint32_t)(steps + steps1);
        }
        umma_commit(mma_end);  // TMEM and the tiles are not given up under an MMA
        mbar_drain(mma_end, 0);
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------ rows that nobody sees, or not all
      VPos vp;
      bool ok = true;
      for (; ok; ++s) {
        if (!(ok = ring->wait_warp(s, abort_flag))) break;
        const Segment k = ring->at[s % kRing];
        if (k.last) break;
        const int streams = k.lone ? 2 : 1;
        uint32_t bad = 0;
        int n0, g0;
        k.origin(g, 0, n0, g0);
        // own tokens that every row of the item sees (along the group's tiles the tokens start over)
        const int common = k.limit(g.g_tiles > 1 ? 0 : n0);
        if (lane == 0) *s_bad = *s_bad & ~(1u << ((s + 16) & 31));  // read by all long ago
        for (int j = k.j0; ok && j < k.j1; ++j) {
          for (int w = 0; w < streams && k.uses(w, j); ++w) {
            if (!(ok = mbar_wait_warp<false>(&v_full[vp.slot], vp.phase, kErrTimeoutAttnKV, abort_flag))) break;
            const int tile = k.kv_tile(w, j);
            const bool pre = tile < k.ptiles;
            const int key0 = (pre ? tile : tile - k.ptiles) * 128;
            const int khi = (pre ? p.prefix : k.own) - key0, klo = pre ? khi : common - key0;
            uint8_t* tile_at = sV + vp.slot * C::kTile;
            if (khi < 128) {
              // a lane's row, its pieces in an order that keeps the lanes on different banks
              for (int row = max(khi, 0) + lane; row < 128; row += 32) {
#pragma unroll
                for (int x = 0; x < 8 * C::kHalves; ++x)
                  *reinterpret_cast<uint4*>(tile_at + row * 128 + (x >> 3) * kHalfBytes + (((x + lane) & 7) << 4)) =
                      make_uint4(0u, 0u, 0u, 0u);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
            if (klo < min(khi, 128)) {
              // rows that some see and others do not: 0 * NaN would reach the others
              Magnitude seen;
              for (int row = max(klo, 0) + lane; row < min(khi, 128); row += 32) {
#pragma unroll
                for (int x = 0; x < 8 * C::kHalves; ++x) {
                  seen.add(*reinterpret_cast<const uint4*>(tile_at + row * 128 + (x >> 3) * kHalfBytes +
                                                           (((x + lane) & 7) << 4)));
                }
              }
              if (__any_sync(0xffffffffu, !seen.finite<T>())) {
                if (!bad && lane == 0) *s_bad = *s_bad | 1u << (s & 31);
                bad = 1;
                leave_out<T, C::kHalves>(tile_at, max(klo, 0), min(khi, 128), lane);
              }
            }
            if (lane == 0) mbar_arrive(&v_ready[vp.slot]);
            vp = vp.plus(1);
          }
        }
      }
    } else if (lane == 0) {
      ring->fill(p, g, run, abort_flag);
    }
  } else {
    warpgroup_reg_inc<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax + epilogue
    const int w = (warp - kSoftmaxWarp0) >> 2, q = warp & 3;
    const int row = q * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t oAddr = tmem + lane_off + C::kColO + (uint32_t)(w * DP);
    const float c = p.scale_log2;
    uint32_t mine = 0, seq = 0;  // this tile's steps so far; sequence position of the segment
    uint32_t meets = 0;
    bool ok = true;
    for (;; ++s) {
      if (!ring->wait_warp(s, abort_flag)) break;
      const Segment& k = ring->at[s % kRing];
      if (k.last) break;
      int n0, g0;
      k.origin(g, w, n0, g0);
      const int rn = row / g.gt, n = n0 + rn, head = g0 + row - rn * g.gt;
      const bool valid = rn < g.nt && n < k.n && head < g.group;
      const bool warp_active = __any_sync(0xffffffffu, valid);
      const int limit = valid ? k.limit(n) : k.own;  // own tokens that the row sees
      float ref = 0.f, l = 0.f;
      bool have = false;  // the reference is set
      const int all_steps = k.j1 - k.j0, steps1 = k.uses(1, k.j1 - 1) ? all_steps : all_steps - 1;
      const int steps = w ? steps1 : all_steps;
      float away_ref = 0.f;  // reference of what has been put away, in the worker's slot
      float* const away = valid ? k.tile_slot(g, run) + (size_t)(w * 128 + row) * g.ld : nullptr;
      for (int t = 0; t < steps; ++t, ++mine) {
        const StepBuf<NB> b(w, mine, seq + 2 * t + w);
        const uint32_t sAddr = tmem + lane_off + b.buf * 128;
        const int tile = k.kv_tile(w, k.j0 + t);
        const int khi = tile < k.ptiles ? p.prefix - tile * 128 : limit - (tile - k.ptiles) * 128;
        const bool put = t > 0 && (t & (kSumSteps<T> - 1)) == 0;  // O is put away, and starts anew
        const bool all = __all_sync(0xffffffffu, khi >= 128) && !put;
        if (!mbar_wait_warp<false>(&s_full[b.buf], b.parity, kErrTimeoutAttnS, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_active) {
          bool done = false;
          if (all) {
            // every key is seen: one pass without a maximum, against the reference (at first that of 32 scores)
            constexpr uint32_t kAllWords[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
            if (!have) {
              uint32_t r[32];
              tmem_ld32(sAddr, r);
              tmem_ld_wait(r);
              // (-inf where these scores are: sums against it are not finite)
              ref = chunk_max(r, 0xffffffffu, c) - kRefShift<T>;
              have = true;
            }
            uint32_t pk[64];
            const float sum = row_exp<T, true>(sAddr, kAllWords, c, ref, pk);
            done = __all_sync(0xffffffffu, !valid || sum <= kSumLimit<T>);
            if (done) {
              l += sum;
              tmem_st32(sAddr, *reinterpret_cast<const uint32_t(*)[32]>(pk));
              tmem_st32(sAddr + 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
            }
          }
          if (!done) {
            // Some keys are not seen, or a sum has grown too large or is not finite, or O is put away: the reference moves
            // to the row's maximum where that is above it, O and l with it, in two passes chunk by chunk.  (Rolled up, with
            // one form for all masks: code that a short run meets once is fetched while it waits.  P in 16 bits as in
            // chunk_exp.)
            float m = -INFINITY;
#pragma unroll 1
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t r[32];
              tmem_ld32(sAddr + ch * 32, r);
              tmem_ld_wait(r);
              m = fmaxf(m, chunk_max(r, len_word(khi, ch), c));
            }
            if (!have) ref = -INFINITY;
            have = true;
            const float moved = fmaxf(ref, m - kRefShift<T>), base = moved == -INFINITY ? 0.f : moved;
            const float alpha = fast_exp2(ref - base);
            if (put || (t > 0 && __any_sync(0xffffffffu, moved > ref))) {
              // O holds the previous steps once the last PV is through (the one before it was
              // when this step's S was issued, so the parity is the right phase's)
              if (!mbar_wait_warp<false>(&pv_done[w], (mine - 1) & 1, kErrTimeoutAttnO, abort_flag)) {
                ok = false;
                break;
              }
              tc_fence_after();
              if (put) {
                put_away(oAddr, away, p.head_dim, t == kSumSteps<T> ? kStore : kAdd,
                         away_ref == ref ? 1.f : fast_exp2(away_ref - ref));
                away_ref = ref;
              } else {
#pragma unroll 1
                for (int h = 0; h < DP / 32; ++h) {
                  uint32_t r[32];
                  tmem_ld32(oAddr + h * 32, r);
                  tmem_ld_wait(r);
#pragma unroll
                  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                  tmem_st32(oAddr + h * 32, r);
                }
              }
              tmem_st_wait();
            }
            l *= moved > ref ? alpha : 1.f;
            ref = moved;
            // P of chunk ch goes over scores of chunks that have been read
#pragma unroll 1
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t r[32], pk[16];
              tmem_ld32(sAddr + ch * 32, r);
              tmem_ld_wait(r);
              const uint32_t word = len_word(khi, ch);
              float sum = 0.f;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float e0 = word >> (2 * i) & 1 ? fast_exp2(__uint_as_float(r[2 * i]) * c - base) : 0.f;
                const float e1 = word >> (2 * i + 1) & 1 ? fast_exp2(__uint_as_float(r[2 * i + 1]) * c - base) : 0.f;
                sum += e0 + e1;
                pk[i] = pack2<T>(e0, e1);
              }
              l += sum;
              tmem_st16(sAddr + ch * 16, pk);
            }
          }
          tmem_st_wait();
        }
        // (a barrier a buffer: the tile's other warps may be a step ahead)
        tc_fence_before();
        mbar_arrive(&p_full[b.buf]);
      }
      if (!ok) break;
      seq += (uint32_t)(all_steps + steps1);
      if (!mbar_wait_warp<false>(&o_done[w], s & 1, kErrTimeoutAttnO, abort_flag)) break;
      tc_fence_after();
      if (steps > kSumSteps<T> && warp_active)
        put_away(oAddr, away, p.head_dim, kBack, away_ref == ref ? 1.f : fast_exp2(away_ref - ref));
      // a lone tile: the two halves meet, weigh each other in and write half the columns each
      float a0 = 1.f, a1 = 0.f;
      int c_lo = 0, c_hi = p.head_dim;
      uint32_t src0 = oAddr, src1 = oAddr;
      if (k.lone) {
        float* ml = s_ml;
        ml[w * 256 + row] = ref;
        ml[w * 256 + 128 + row] = steps > 0 ? l : -1.f;  // -1: no O
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet[q]);
        if (!mbar_wait_warp<false>(&meet[q], meets & 1, kErrTimeoutAttnO, abort_flag)) break;
        ++meets;
        tc_fence_after();
        const float r0 = ml[row], r1 = ml[256 + row], l0 = ml[128 + row], l1 = ml[256 + 128 + row];
        const bool has1 = l1 != -1.f;
        if (has1) {
          // a half without a kept key has l = 0 and no reference of its own
          ref = l0 == 0.f ? r1 : (l1 == 0.f ? r0 : fmaxf(r0, r1));
          a0 = l0 == 0.f ? 0.f : fast_exp2(r0 - ref);
          a1 = l1 == 0.f ? 0.f : fast_exp2(r1 - ref);
          l = l0 * a0 + l1 * a1;
        } else {
          ref = r0;
          l = l0;
        }
        src0 = tmem + lane_off + C::kColO;
        src1 = has1 ? src0 + DP : src0;
        // 16-column pieces, the first half of them to w = 0
        const int mid = ((p.head_dim + 31) >> 5) * 16;
        if (w == 0)
          c_hi = min(mid, p.head_dim);
        else
          c_lo = min(mid, p.head_dim);
      }
      // (past the meeting: a lone tile's other half may have multiplied the last V tile)
      const bool bad = *s_bad >> (s & 31) & 1;
      const bool whole = k.whole(), finish = whole && g.concat;
      const float inv = finish ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
      const float f0 = a0 * inv, f1 = a1 * inv;
      if (warp_active) {
        const size_t grow = (size_t)(k.q0 + n) * p.q.heads + (size_t)(k.hk * g.group + head);
        const size_t plane = (size_t)p.tokens * p.q.heads * k.phase;
        T* out = static_cast<T*>(p.out.data) + (k.q0 + n) * p.out.seq_stride +
                 (long long)(k.hk * g.group + head) * p.out.head_stride;
        const int at = (k.lone ? 0 : w * 128) + row;
        float* po = whole ? g.whole + (plane + grow) * g.ld : k.tile_slot(g, run) + (size_t)at * g.ld;
        for (int c0 = c_lo; c0 < c_hi; c0 += 16) {
          uint32_t r0[16], r1[16];
          tmem_ld16(src0 + c0, r0);
          tmem_ld16(src1 + c0, r1);
          tmem_ld_wait(r0, r1);
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = f0 != 0.f ? __uint_as_float(r0[i]) * f0 : 0.f;
            if (f1 != 0.f) v[i] += __uint_as_float(r1[i]) * f1;
          }
          if (valid) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (c0 + 8 * u >= c_hi) break;
              if (finish) {
                *reinterpret_cast<uint4*>(out + c0 + 8 * u) =
                    make_uint4(pack2<T>(v[8 * u], v[8 * u + 1]), pack2<T>(v[8 * u + 2], v[8 * u + 3]),
                               pack2<T>(v[8 * u + 4], v[8 * u + 5]), pack2<T>(v[8 * u + 6], v[8 * u + 7]));
              } else {
                store8(po + c0 + 8 * u, v + 8 * u);
              }
            }
          }
        }
        if (valid && (!k.lone || w == 0)) {
          if (!finish) *reinterpret_cast<float4*>(po + p.head_dim) = make_float4(ref, l, bad ? 1.f : 0.f, 0.f);
          if (finish && bad) g.bad[run.place] = 1;
          if (k.j0 == 0) g.where[plane + grow] = finish && bad ? kLeftOut - run.place : k.code | at;
        }
      }
      tc_fence_before();
      if (k.lone) {
        // neither half may go on (and overwrite O or the exchange) before both have read
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet[q]);
        if (!mbar_wait_warp<false>(&meet[q], meets & 1, kErrTimeoutAttnO, abort_flag)) break;
        ++meets;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[s % kRing]);
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------- token items
// A team takes up to 8 key heads of a request as one item, a warp a head: K and V of 32 keys of all its heads
// come by one TMA box (64 columns x 32 keys x heads), so that what lies side by side in the cache is read together,
// and each warp multiplies them by its head's 16 rows and writes its parts from its registers; no warp waits for
// another.  With fewer key heads a CTA has up to four teams with runs of their own.  A warp a team
// brings the tiles, K and V in turn through one ring.
// Bound: memory, 64 requests of up to 1024 own tokens, 8 key heads of 128, without a prefix: 135 MB in 31 us.  On the way
// to it: tiles of one head shared out over eight warps that met at each item's end, 37 us; a run for
// each warp, which asked for its own tiles, 57 (its warps stood still while the TMA unit was busy, and the parts of a
// cache line were asked for at different times).
// 16-byte piece `chunk` (8 columns) of row `row` in a 128B-swizzled tile of 64-column boxes of `box` bytes
__device__ __forceinline__ uint32_t token_piece(uint32_t tile, uint32_t box, int row, int chunk) {
  return tile + (uint32_t)(chunk >> 3) * box + (uint32_t)(row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// The V rows of a tile that not all rows see, a lane a key: zeroed from key khi on, which is not there (0 * NaN would
// reach the sum); of the others from klo on, which some see and others do not, infinities and NaN alone, and whether there
// were any.
// (Out of the loop's way: its instructions are fetched again and again, and masks on every fragment were a third of them.)
template <typename T, int kHalves>
__device__ __noinline__ bool clear_keys(uint8_t* tile, uint32_t half_bytes, int row0, int row16, int klo, int khi, int lane) {
  uint8_t* row = tile + (lane < 16 ? row0 + lane : row0 + row16 + lane - 16) * 128;
  Magnitude seen;
  if (lane >= klo) {
#pragma unroll 1
    for (int x = 0; x < 8 * kHalves; ++x) {
      uint4* piece = reinterpret_cast<uint4*>(row + (x >> 3) * half_bytes + (((x + lane) & 7) << 4));
      if (lane >= khi) {
        *piece = make_uint4(0u, 0u, 0u, 0u);
      } else {
        seen.add(*piece);
      }
    }
    if (!seen.finite<T>()) {
#pragma unroll 1
      for (int x = 0; x < 8 * kHalves; ++x) {
        uint4* piece = reinterpret_cast<uint4*>(row + (x >> 3) * half_bytes + (((x + lane) & 7) << 4));
        *piece = finite_ones<T>(*piece);
      }
    }
  }
  fence_proxy_async_smem();  // the tile's place is given back to TMA after these writes
  __syncwarp();
  return !seen.finite<T>();
}

struct Team {  // in shared memory
  Segment seg[2];
  uint64_t seg_full[2], seg_empty[2], full[kMostEntries], empty[kMostEntries], q_full[2], q_empty[2];
  int abort, pad;
};

template <typename T, int DP>
__device__ void token_role(uint8_t* smem, const CUtensorMap& qmap, const CUtensorMap& pkmap, const CUtensorMap& pvmap,
                           const CUtensorMap& kcmap, const CUtensorMap& vcmap, const PrefixAttnParams& p,
                           const PrefixGeom& g, const Run* runs) {
  using C = PCfg<DP>;
  constexpr int kHalves = C::kHalves;
  static_assert(kMostTeams * sizeof(Team) <= C::kTail, "");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = warp < kTokenWarps ? warp / g.heads : warp - kTokenWarps, h = warp - team * g.heads;
  Team* tm = reinterpret_cast<Team*>(smem + C::kTiles) + team;
  volatile int* abort_flag = &tm->abort;
  Run run{};
  if (team < g.teams) run = runs[team];
  __syncthreads();  // the runs have been read
  if (warp < g.teams) {  // a lane a barrier: the team's warps arrive where something is given back
    Team* x = reinterpret_cast<Team*>(smem + C::kTiles) + warp;
    static_assert(offsetof(Team, abort) - offsetof(Team, seg_full) == 32 * sizeof(uint64_t), "");
    const bool given_back = (lane >= 2 && lane < 4) || (lane >= 16 && lane < 28) || lane >= 30;
    mbar_init(&x->seg_full[lane], given_back ? g.heads : 1);
    if (lane == 0) x->abort = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (team >= g.teams || run.count == 0) return;
  const uint32_t entry_bytes = (uint32_t)g.heads * C::kEntry, half_bytes = (uint32_t)g.heads * kTokenBox;
  const uint32_t q_half = (uint32_t)(g.heads * g.q_rows) * 128u;
  uint8_t* tiles = smem + (size_t)team * g.entries * entry_bytes;
  uint8_t* sQ = smem + (size_t)g.teams * g.entries * entry_bytes + (size_t)team * g.q_slots * kHalves * q_half;

  if (warp >= kTokenWarps) {
    // ------------------------------------------------------------ the team's tiles
    ItemWalk walk(p, g, run);
    int s = 0, e = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (;; ++s) {
      Segment x;
      walk.next(x);
      if (!(ok = mbar_wait_warp<false>(&tm->seg_empty[s & 1], (s >> 1 & 1) ^ 1, kErrTimeoutAttnQ, abort_flag))) break;
      if (lane == 0) {
        tm->seg[s & 1] = x;
        mbar_arrive(&tm->seg_full[s & 1]);
        if (!x.last && x.code) g.cuts[run.place] = tm->seg[s & 1];
      }
      if (x.last) break;
      const int head0 = x.hk * g.heads, qs = s % g.q_slots, q_use = s / g.q_slots;
      if (!(ok = mbar_wait_warp<false>(&tm->q_empty[qs], (q_use & 1) ^ 1, kErrTimeoutAttnQ, abort_flag))) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&tm->q_full[qs], (uint32_t)(g.heads * (g.q_rows / g.group) * g.group) * 128u * kHalves);
        for (int i = 0; i < kHalves; ++i)
          tma_load_4d(sQ + (qs * kHalves + i) * q_half, &qmap, &tm->q_full[qs], i * 64, 0, x.q0, head0);
      }
      int table0 = -32, pages = 0;  // of the request's block table: entries [table0, table0 + 32), a lane each
      for (int j = x.j0; ok && j < x.j1; ++j) {
        int first = 0, second = 0, boxes = 1, at = 0;
        if (j >= x.ptiles) {
          const int key0 = (j - x.ptiles) * kTokenKeys, left = x.own - key0, block = key0 >> p.page_shift;
          if (block + (kTokenKeys >> 4) > table0 + 32) {
            table0 = block;
            pages = block + lane < p.blocks ? __ldg(p.table + x.r * p.table_stride + block + lane) : 0;
          }
          first = __shfl_sync(0xffffffffu, pages, block - table0);
          second = __shfl_sync(0xffffffffu, pages, block + 1 - table0);  // (of a tile of two pages)
          boxes = left <= 0 ? 0 : (left > g.box ? kTokenKeys / g.box : 1);
          at = key0 & ((1 << p.page_shift) - 1);
        }
        for (int v = 0; v < 2; ++v) {
          if (!(ok = mbar_wait_warp<false>(&tm->empty[e], phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
          if (lane == 0) {
            uint64_t* bar = &tm->full[e];
            uint8_t* dst = tiles + e * entry_bytes;
            if (j < x.ptiles) {
              mbar_arrive_expect_tx(bar, entry_bytes);
              for (int i = 0; i < kHalves; ++i)
                tma_load_4d(dst + i * half_bytes, v ? &pvmap : &pkmap, bar, i * 64, j * kTokenKeys,
                            head0 * (v ? g.pv_headed : g.pk_headed), 0);
            } else if (boxes == 0) {
              mbar_arrive(bar);
            } else {
              // (a page of 16 keys is a box of its own, heads side by side in each: see the row that a key has)
              mbar_arrive_expect_tx(bar, (uint32_t)(boxes * g.box * g.heads) * 128u * kHalves);
              for (int b = 0; b < boxes; ++b) {
                const int id = checked_page(p, b ? second : first);
                for (int i = 0; i < kHalves; ++i)
                  tma_load_4d(dst + i * half_bytes + b * g.box * g.heads * 128, v ? &vcmap : &kcmap, bar, i * 64, at,
                              head0 * (v ? g.vc_headed : g.kc_headed), id);
              }
            }
          }
          __syncwarp();
          if (++e == g.entries) e = 0, phase ^= 1;
        }
      }
      if (!ok) break;
    }
    if (!ok && lane == 0) {  // nothing is given up under copies in flight
      mbar_drain_ring(tm->full, g.entries, e, phase);
      mbar_drain_ring(tm->q_full, g.q_slots, s % g.q_slots, s / g.q_slots & 1);
    }
    return;
  }

  const int qr = lane >> 2, qc = lane & 3;  // fragment row (and row + 8) and column pair
  const float c = p.scale_log2;
  const uint32_t base = smem_u32(tiles), base_q = smem_u32(sQ);
  // ldmatrix row addresses: Q wants (rows 0-7, 8 columns), (rows 8-15, ..), then the next 8 columns of both; K
  // (keys 0-7, 8 columns), (keys 0-7, next 8), (keys 8-15, ..) x 2; V (transposed) (keys 0-7), (keys 8-15)
  // of 8 columns, then of the next 8
  const int krow = (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;
  const int vrow = lane & 15, vchunk = lane >> 4;
  const int q_box = g.q_rows / g.group * g.group;  // rows of a head
  int at = 0;  // the entry to wait for and the parity of its use
  uint32_t phase = 0;
  bool ok = true;
  for (int s = 0; ok; ++s) {
    if (!mbar_wait_warp<false>(&tm->seg_full[s & 1], s >> 1 & 1, kErrTimeoutAttnQ, abort_flag)) break;
    const Segment& k = tm->seg[s & 1];
    if (k.last) break;
    uint32_t qa[DP / 16][4];
    const int qs = s % g.q_slots;
    if (!mbar_wait_warp<false>(&tm->q_full[qs], s / g.q_slots & 1, kErrTimeoutAttnQ, abort_flag)) break;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)  // (rows past the head's are another's, whose results nobody reads)
      ldmatrix4(token_piece(base_q + qs * kHalves * q_half, q_half, h * q_box + (vrow & (g.q_rows - 1)), 2 * i + vchunk), qa[i]);
    __syncwarp();
    if (lane == 0) mbar_arrive(&tm->q_empty[qs]);
    const int rows = k.n * g.group, j1 = k.j1, ptiles = k.ptiles, own = k.own;
    // own tokens that the fragment's two rows see, and that every row sees
    const int limit[2] = {qr < rows ? k.limit(qr / g.group) : own, qr + 8 < rows ? k.limit((qr + 8) / g.group) : own};
    const int common = k.limit(0);
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool bad = false;
    for (int jj = k.j0; jj < j1; ++jj) {
      if (!(ok = mbar_wait_warp<false>(&tm->full[at], phase, kErrTimeoutAttnKV, abort_flag))) break;
      const bool pre = jj < ptiles;
      // Where a key's row is: in a box of 32 keys, head by head, or (16 keys a page) in two of 16, head by head in each
      const bool split = !pre && g.box < kTokenKeys;
      const int row0 = split ? h * 16 : h * 32, row16 = split ? g.heads * 16 : 16;
      const uint32_t kt = base + at * entry_bytes;
      float sc[4][4];  // four column tiles of 8 keys
#pragma unroll
      for (int i = 0; i < 16; ++i) (&sc[0][0])[i] = 0.f;
#pragma unroll
      for (int x = 0; x < DP / 16; ++x) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t b[4];
          ldmatrix4(token_piece(kt, half_bytes, row0 + y * row16 + krow, 2 * x + kchunk), b);
          mma16816<T>(sc[2 * y], qa[x], b[0], b[1]);
          mma16816<T>(sc[2 * y + 1], qa[x], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&tm->empty[at]);
      if (++at == g.entries) at = 0, phase ^= 1;
      // of the tile's 32 keys: the first khi are there, the first klo are seen by every row
      const int key0 = (pre ? jj : jj - ptiles) * kTokenKeys;
      const int khi = (pre ? p.prefix : own) - key0, klo = pre ? khi : common - key0;
      const bool all = klo >= kTokenKeys;
      float mx[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) (&sc[0][0])[i] *= c;
      if (!all) {
        const int lim[2] = {(pre ? khi : limit[0] - key0) - qc * 2, (pre ? khi : limit[1] - key0) - qc * 2};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)  // i: row half * 2 + key of the pair
            if (8 * t + (i & 1) >= lim[i >> 1]) sc[t][i] = -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmax3(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]),
                      fmax3(sc[2][2 * h], sc[2][2 * h + 1], fmaxf(sc[3][2 * h], sc[3][2 * h + 1])));
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
        ref[h] -= kLift<T>;
        moved |= mn > m[h];
        m[h] = mn;
      }
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
      // weights in the operands' 16 bits, which the product with V takes (l adds them up unrounded, in fp32)
      uint32_t pa[2][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][i] = fast_exp2(sc[t][i] - ref[i >> 1]);
        pa[t >> 1][2 * (t & 1)] = pack2<T>(sc[t][0], sc[t][1]);
        pa[t >> 1][2 * (t & 1) + 1] = pack2<T>(sc[t][2], sc[t][3]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        l[h] += ((sc[0][2 * h] + sc[0][2 * h + 1]) + (sc[1][2 * h] + sc[1][2 * h + 1])) +
                ((sc[2][2 * h] + sc[2][2 * h + 1]) + (sc[3][2 * h] + sc[3][2 * h + 1]));
      if (!(ok = mbar_wait_warp<false>(&tm->full[at], phase, kErrTimeoutAttnKV, abort_flag))) break;
      const uint32_t vt = base + at * entry_bytes;
      if (!all) bad |= clear_keys<T, kHalves>(tiles + at * entry_bytes, half_bytes, row0, row16, klo, khi, lane);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        // a tile's products in accumulators of their own, added in fp32 (see cross_token.cu)
        float d[2][4] = {};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t b[4];
          ldmatrix4_trans(token_piece(vt, half_bytes, row0 + y * row16 + vrow, 2 * i + vchunk), b);
          mma16816<T>(d[0], pa[y], b[0], b[1]);
          mma16816<T>(d[1], pa[y], b[2], b[3]);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) o[2 * i + (x >> 2)][x & 3] += d[x >> 2][x & 3];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&tm->empty[at]);
      if (++at == g.entries) at = 0, phase ^= 1;
    }
    if (!ok) break;
    bad = __any_sync(0xffffffffu, bad);
    const bool whole = k.j0 == 0 && j1 == k.units, finish = whole && g.concat;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
      const int r = qr + 8 * half;
      if (r >= rows) continue;
      const int n = r / g.group, head = (k.hk * g.heads + h) * g.group + r - n * g.group;
      const size_t grow = (size_t)p.tokens * p.q.heads * k.phase + (size_t)(k.q0 + n) * p.q.heads + head;
      if (finish) {
        const float inv = l[half] > 0.f ? 1.f / l[half] : (l[half] == 0.f ? 0.f : l[half]);
        T* out = static_cast<T*>(p.out.data) + (k.q0 + n) * p.out.seq_stride + (long long)head * p.out.head_stride + qc * 2;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          if (8 * i < p.head_dim) *reinterpret_cast<uint32_t*>(out + 8 * i) = pack2<T>(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
      } else {
        float* po = whole ? g.whole + grow * g.ld : k.token_slot(g, run, h) + (size_t)r * g.ld;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          if (8 * i < p.head_dim) *reinterpret_cast<float2*>(po + 8 * i + qc * 2) = make_float2(o[i][2 * half], o[i][2 * half + 1]);
        // the sums are taken against the maximum less kLift
        if (qc == 0)
          *reinterpret_cast<float4*>(po + p.head_dim) = make_float4(m[half] - kLift<T>, l[half], bad ? 1.f : 0.f, 0.f);
      }
      if (qc == 0 && finish && bad) g.bad[run.place] = 1;
      if (qc == 0 && k.j0 == 0) g.where[grow] = finish && bad ? kLeftOut - run.place : k.code | r;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&tm->seg_empty[s & 1]);
  }
}

// Tensor maps: of the tile items' query rows, K and V of one head; of the token items', of a team's heads.
struct Maps {
  CUtensorMap q, pk, pv, kc, vc;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_attention_kernel(const __grid_constant__ Maps tile, const __grid_constant__ Maps token,
                            const __grid_constant__ PrefixAttnParams p, const __grid_constant__ PrefixGeom g) {
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzled tiles start on 1024 bytes
  // the runs are found in memory that the roles take over
  Two* scratch = reinterpret_cast<Two*>(smem);
  Run* runs = reinterpret_cast<Run*>(smem + 1024);
  if (threadIdx.x < 10) {
    const Maps& m = threadIdx.x < 5 ? tile : token;
    tma_prefetch_desc(&m.q + threadIdx.x % 5);  // (the members in their order)
  }
  if (threadIdx.x < g.teams) {
    const int place = (int)blockIdx.x * g.teams + threadIdx.x;
    g.cuts[place].code = 0;
    g.bad[place] = 0;
  }
  find_runs(p, g, runs, scratch);
  dependents_may_start();
  if (runs[0].token) {
    token_role<T, DP>(smem, token.q, token.pk, token.pv, token.kc, token.vc, p, g, runs);
  } else {
    const Run run = runs[0];
    __syncthreads();
    if (run.count > 0) tile_role<T, DP>(smem, tile.q, tile.pk, tile.pv, tile.kc, tile.vc, p, g, run);
  }
}

// ------------------------------------------------------------------------------- joining
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

// Adds the infinities and NaN of the V rows that a query row sees and that its item left out of the product, 4 columns
// a lane.  Left out are those of keys that not all of the item's rows see (see `common`), of tokens no further back than a
// pair of row tiles reaches; where others had their part in the product, they are in v already and change nothing.
template <typename T>
__device__ void add_left_out(const PrefixAttnParams& p, const PrefixGeom& g, int token, int head, int lane, float (&v)[4]) {
  const int r = request_of(p, token);
  if (r < 0) return;
  const Request q = load_request(p, r);
  const int limit = q.limit(token - q.q0), from = g.g_tiles == 1 ? max(limit - 2 * g.nt, 0) : min(q.limit(0), limit);
  const T* x = static_cast<const T*>(p.v_cache.data) + (head / g.group) * p.v_cache.head_stride + 4 * lane;
  const int* row = p.table + r * p.table_stride;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = from; i < limit; ++i) {
    const int page = checked_page(p, __ldg(row + (i >> p.page_shift)));
    if (4 * lane >= p.head_dim || page >= p.pages) continue;
    const uint2 w = *reinterpret_cast<const uint2*>(x + page * p.v_cache.batch_stride +
                                                    (i & ((1 << p.page_shift) - 1)) * p.v_cache.seq_stride);
    float f[4];
    unpack2<T>(w.x, f[0], f[1]);
    unpack2<T>(w.y, f[2], f[3]);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (!isfinite(f[c])) sum[c] += f[c];
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (!isfinite(sum[c])) v[c] += sum[c];
}

// What a row's parts have added up to: reference, sum and 4 columns a lane.
struct Sum {
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float pm, float pl, const float4& x) {
    if (pl == 0.f) return;  // no key of that part is seen
    const float mn = fmaxf(m, pm), a = fast_exp2(m - mn), e = fast_exp2(pm - mn);
    l = l * a + pl * e;
    m = mn;
    o[0] = o[0] * a + x.x * e;
    o[1] = o[1] * a + x.y * e;
    o[2] = o[2] * a + x.z * e;
    o[3] = o[3] * a + x.w * e;
  }
};

// The parts of a row for one phase: their number, where the first one is and how far apart the others.
struct Parts {
  const float* base = nullptr;
  size_t stride = 0;
  int count = 0;
  __device__ __forceinline__ void find(const PrefixGeom& g, int code, int place_in_slot, const float* whole, int ctas) {
    const int c0 = code >> 8 & 0xfff, more = code >> 20;
    const bool tile = c0 >= kTileWorkers;
    const int first = tile ? c0 - kTileWorkers : c0, last = tile ? ctas - 1 : ctas * g.teams - 1;
    const size_t slot = (size_t)(tile ? g.tile_rows : g.heads * g.token_rows) * g.ld;
    // the first part ends its worker's run, the others begin theirs
    base = more == 0 ? whole
                     : (tile ? g.tile_slots : g.token_slots) + 2 * min(first, last) * slot + (size_t)place_in_slot * g.ld;
    stride = 2 * slot;
    count = 1 + min(more, max(last - first, 0));
  }
  __device__ __forceinline__ const float* at(int i) const { return base + i * stride + (i > 0 ? stride >> 1 : 0); }
};

// Parts first, first + step, ... of two lists one behind the other (kAhead in flight) into the sum.
template <int kAhead>
__device__ __forceinline__ void add_parts(const Parts& a, const Parts& b, int first, int step, int d, int col, Sum& sum,
                                          bool& again) {
  const int n = a.count + b.count;
  for (int i0 = first; i0 < n; i0 += kAhead * step) {
    float4 h[kAhead], v[kAhead];
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      h[y] = v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
      const int i = i0 + y * step;
      if (i >= n) continue;
      const float* f = i < a.count ? a.at(i) : b.at(i - a.count);
      h[y] = __ldcg(reinterpret_cast<const float4*>(f + d));
      if (col < d) v[y] = __ldcg(reinterpret_cast<const float4*>(f + col));
    }
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      again |= h[y].z != 0.f;
      sum.add(h[y].x, h[y].y, v[y]);
    }
  }
}

// Writes a row; again: its item has left values out.
template <typename T>
__device__ __forceinline__ void finish_row(const PrefixAttnParams& p, const PrefixGeom& g, int token, int head, const Sum& sum,
                                           bool again, int lane) {
  const float inv = sum.l > 0.f ? 1.f / sum.l : (sum.l == 0.f ? 0.f : sum.l);
  float v[4] = {sum.o[0] * inv, sum.o[1] * inv, sum.o[2] * inv, sum.o[3] * inv};
  if (again) add_left_out<T>(p, g, token, head, lane, v);
  if (4 * lane >= p.head_dim) return;
  T* out = static_cast<T*>(p.out.data) + token * p.out.seq_stride + head * p.out.head_stride + 4 * lane;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

// The same for a row that has been written without them.
template <typename T>
__device__ __forceinline__ void complete_row(const PrefixAttnParams& p, const PrefixGeom& g, int token, int head, int lane) {
  T* out = static_cast<T*>(p.out.data) + token * p.out.seq_stride + head * p.out.head_stride + 4 * lane;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const bool active = 4 * lane < p.head_dim;
  if (active) {
    const uint2 w = *reinterpret_cast<const uint2*>(out);
    unpack2<T>(w.x, v[0], v[1]);
    unpack2<T>(w.y, v[2], v[3]);
  }
  add_left_out<T>(p, g, token, head, lane, v);
  if (active) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

// Adds up the parts of each row, in a fixed order: the prefix's and the own ones, or, of one sequence of both,
// those of the rows that a run cut (the others are done).  4 columns a lane; a warp a row, kWide (few rows, whose
// parts may be many): a block a row, its warps taking parts in turn.
// Bound: latency, three loads one behind the other.
template <typename T, bool kWide>
__global__ void __launch_bounds__(256, 2)
    prefix_join_kernel(const __grid_constant__ PrefixAttnParams p, const __grid_constant__ PrefixGeom g, int ctas) {
  __shared__ float4 s_o[kWide ? 8 : 1][32];
  __shared__ float s_m[8], s_l[8];
  __shared__ int s_again[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = p.head_dim;
  const long long rows = (long long)p.tokens * p.q.heads, row = kWide ? blockIdx.x : (long long)blockIdx.x * 8 + warp;
  if (row >= rows) return;
  const int token = (int)(row / p.q.heads), head = (int)(row - (long long)token * p.q.heads);
  wait_for_previous();
  const bool of_a_request = !p.q_starts || (token >= first_row(p, 0) && token < first_row(p, p.requests));
  const int code0 = g.concat ? 0 : g.where[row], code1 = g.where[rows + row];
  if (!of_a_request) {
    if (p.zero_rest) finish_row<T>(p, g, token, head, Sum(), false, lane);
    return;
  }
  if (code0 < 0 || code1 < 0) {
    if (!kWide || warp == 0) complete_row<T>(p, g, token, head, lane);
    return;
  }
  if (g.concat && code1 >> 20 == 0) return;
  bool again = false;
  Sum sum;
  {
    const int h = head / g.group % g.heads;
    auto place = [&](int code) {  // (of a team's slot: its head's rows)
      const int at = code & 255;
      return (code >> 8 & 0xfff) >= kTileWorkers ? at : h * g.token_rows + min(at, g.token_rows - 1);
    };
    Parts a, b;
    if (!g.concat) a.find(g, code0, place(code0), g.whole + (size_t)row * g.ld, ctas);
    b.find(g, code1, place(code1), g.whole + (size_t)(rows + row) * g.ld, ctas);
    add_parts<8>(a, b, kWide ? warp : 0, kWide ? 8 : 1, d, lane * 4, sum, again);
  }
  if constexpr (kWide) {
    s_o[warp][lane] = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
    if (lane == 0) {
      s_m[warp] = sum.m;
      s_l[warp] = sum.l;
      s_again[warp] = again;
    }
    __syncthreads();
    if (warp > 0) return;
    sum = Sum();
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      sum.add(s_m[w], s_l[w], s_o[w][lane]);
      again |= s_again[w] != 0;
    }
  }
  finish_row<T>(p, g, token, head, sum, again, lane);
}

// The same for many rows of one sequence of prefix and own keys, most of which are done: block (x, y) takes rows
// [8 y, 8 y + 8) of both tiles of the item that worker x started and did not end, a warp one of each, whose parts come
// together.  (4096 tokens of 32 heads, 37,000 rows of them cut: 9 us; a row a warp, 15; looking through all rows, 26.)
template <typename T>
__global__ void __launch_bounds__(256, 4)
    prefix_join_cuts_kernel(const __grid_constant__ PrefixAttnParams p, const __grid_constant__ PrefixGeom g, int ctas) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, x = blockIdx.y * 8 + warp;
  wait_for_previous();
  const Segment k = g.cuts[blockIdx.x];
  if (k.code > 0) {
    int n[2], head[2];
    bool valid[2];
    if ((k.code >> 8 & 0xfff) >= kTileWorkers) {
      const int rn = x / g.gt;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        int n0, g0;
        k.origin(g, u, n0, g0);
        n[u] = n0 + rn;
        head[u] = g0 + x - rn * g.gt;
        valid[u] = rn < g.nt && n[u] < k.n && head[u] < g.group && !(k.lone && u);
        head[u] += k.hk * g.group;
      }
    } else {  // (up to 128 rows)
      const int h = x / g.token_rows, r = x - h * g.token_rows;
      n[0] = r / g.group;
      head[0] = (k.hk * g.heads + h) * g.group + r - n[0] * g.group;
      valid[0] = h < g.heads && n[0] < k.n;
      n[1] = head[1] = 0;
      valid[1] = false;
    }
    Parts parts;
    parts.find(g, k.code, x, nullptr, ctas);
    const int d = p.head_dim, col = lane * 4;
    Sum sum[2];
    bool again[2] = {false, false};
    for (int i0 = 0; i0 < parts.count; i0 += 2) {
      float4 h[2][2], v[2][2];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          h[y][u] = v[y][u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i0 + y >= parts.count || !valid[u]) continue;
          const float* f = parts.at(i0 + y) + (size_t)u * 128 * g.ld;
          h[y][u] = __ldcg(reinterpret_cast<const float4*>(f + d));
          if (col < d) v[y][u] = __ldcg(reinterpret_cast<const float4*>(f + col));
        }
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          again[u] |= h[y][u].z != 0.f;
          sum[u].add(h[y][u].x, h[y][u].y, v[y][u]);
        }
    }
#pragma unroll 1
    for (int u = 0; u < 2; ++u)
      if (u ? valid[1] : valid[0])
        finish_row<T>(p, g, k.q0 + (u ? n[1] : n[0]), u ? head[1] : head[0], u ? sum[1] : sum[0], u ? again[1] : again[0], lane);
  }
  if (p.zero_rest && p.q_starts) {
    const int before = first_row(p, 0), behind = first_row(p, p.requests);
    const long long rest = ((long long)before + max(p.tokens - behind, 0)) * p.q.heads;
    for (long long i = (long long)blockIdx.x * gridDim.y * 8 + x; i < rest; i += (long long)gridDim.x * gridDim.y * 8) {
      const int token = (int)(i / p.q.heads);
      finish_row<T>(p, g, token < before ? token : behind + token - before, (int)(i % p.q.heads), Sum(), false, lane);
    }
  }
  if (g.bad[blockIdx.x]) {  // whole items that have left values out
    const long long rows = (long long)p.tokens * p.q.heads;
    for (long long row0 = 32LL * x; row0 < rows; row0 += 32LL * gridDim.y * 8) {
      const bool hit = row0 + lane < rows && g.where[rows + row0 + lane] == kLeftOut - (int)blockIdx.x;
      for (uint32_t some = __ballot_sync(0xffffffffu, hit); some; some &= some - 1) {
        const long long row = row0 + __ffs(some) - 1;
        complete_row<T>(p, g, (int)(row / p.q.heads), (int)(row % p.q.heads), lane);
      }
    }
  }
}

// Without a request every row is one of nobody: zeroed, 8 columns a thread.
__global__ void __launch_bounds__(256) prefix_zero_kernel(const __grid_constant__ PrefixAttnParams p) {
  const unsigned pieces = (unsigned)p.head_dim >> 3;
  const long long all = (long long)p.tokens * p.out.heads * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
    const long long row = i / pieces, token = row / p.out.heads;
    // (16-bit values of either type)
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out.data) + token * p.out.seq_stride +
                              (row - token * p.out.heads) * p.out.head_stride + 8 * (i - row * pieces)) =
        make_uint4(0u, 0u, 0u, 0u);
  }
}

// ------------------------------------------------------------------------------- host
// Bytes of a workspace that it may take to reach the next multiple of 32 (see store8).
constexpr int kSpare = 16;

// Sizes of a launch, and where the parts of its workspace lie (bytes).
struct Layout {
  PrefixGeom g;
  long long where, cuts, tile_slots, token_slots, whole, bytes;
};

Layout make_layout(int tokens, int requests, int prefix, int q_heads, int kv_heads, int head_dim, int num_sms) {
  Layout x{};
  PrefixGeom& g = x.g;
  g.kv_heads = kv_heads;
  g.group = q_heads / kv_heads;
  g.gt = std::min(g.group, 128);
  g.nt = 128 / g.gt;
  g.g_tiles = (g.group + g.gt - 1) / g.gt;
  g.ksteps = (head_dim + 15) / 16;
  const long long rows = (long long)tokens * g.group;  // of a key head
  // Rows of one request that fill a pair of tiles gain nothing from the others', and their parts need no joining
  g.concat = prefix == 0 || rows >= 256LL * requests;
  g.prefix_token = rows <= kTokenRows;
  g.prefix_tiles = (int)(((long long)prefix + 127) >> 7);
  g.prefix_tiles32 = (int)(((long long)prefix + kTokenKeys - 1) >> kTokenShift);
  g.n_tiles = (tokens + g.nt - 1) / g.nt;
  const int tiles = g.n_tiles * g.g_tiles;
  g.full = tiles / 2;
  g.lone = tiles & 1;
  for (g.heads = std::min(kv_heads, kTokenWarps); kv_heads % g.heads; --g.heads) {
  }
  g.groups = kv_heads / g.heads;
  g.teams = std::min(kMostTeams, kTokenWarps / g.heads);
  g.tile_rows = g.prefix_token ? 0 : 256;
  g.token_rows = (int)std::min<long long>(rows, kTokenRows);
  g.ld = head_dim + 8;
  const long long n = (long long)tokens * q_heads;
  auto up = [](long long b) { return (b + 255) & ~255LL; };
  x.cuts = up(2 * n * 4);
  x.tile_slots = up(x.cuts + (long long)num_sms * kMostTeams * (sizeof(Segment) + sizeof(int)));
  x.token_slots = up(x.tile_slots + 2LL * num_sms * g.tile_rows * g.ld * 4);
  x.whole = up(x.token_slots + 2LL * num_sms * g.teams * g.heads * g.token_rows * g.ld * 4);
  x.bytes = x.whole + (g.concat ? 0 : 2 * n * g.ld * 4);
  return x;
}

// {d, group, tokens, key heads} in boxes of 64 x group_box x tokens x heads; a stride that is never walked only has
// to be a legal one
uint64_t legal(long long stride) { return (uint64_t)(stride ? stride * 2 : 16); }
CUtensorMap prefix_query_map(const PrefixAttnParams& p, const PrefixGeom& g, int group_box, int tokens, int heads) {
  const uint64_t dims[4] = {(uint64_t)p.head_dim, (uint64_t)g.group, (uint64_t)p.tokens, (uint64_t)g.kv_heads};
  const uint64_t str[3] = {legal(p.q.head_stride), legal(p.q.seq_stride), legal(p.q.head_stride * g.group)};
  const uint32_t box[4] = {64, (uint32_t)group_box, (uint32_t)tokens, (uint32_t)heads};
  return make_tensor_map(p.q.data, 4, dims, str, box);
}
// {d, keys, key heads, pages} in boxes of 64 x rows x heads; heads with stride 0 are one
CUtensorMap prefix_kv_map(const HeadsView& v, int pages, int keys, int d, int rows, int heads) {
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)keys, v.head_stride ? (uint64_t)v.heads : 1, (uint64_t)pages};
  const uint64_t str[3] = {legal(v.seq_stride), legal(v.head_stride), legal(v.batch_stride)};
  const uint32_t box[4] = {64, (uint32_t)rows, (uint32_t)heads, 1};
  return make_tensor_map(v.data, 4, dims, str, box);
}

template <typename T, int DP>
cudaError_t launch_k(const PrefixAttnParams& p, PrefixGeom g, int num_sms, cudaStream_t s) {
  using C = PCfg<DP>;
  static std::atomic<unsigned long long> configured;
  cudaError_t e = ensure_smem_limit(prefix_attention_kernel<T, DP>, (int)C::kSmem, configured);
  if (e != cudaSuccess) return e;
  g.pk_headed = p.prefix_k.head_stride != 0;
  g.pv_headed = p.prefix_v.head_stride != 0;
  g.kc_headed = p.k_cache.head_stride != 0;
  g.vc_headed = p.v_cache.head_stride != 0;
  const bool token_prefix = p.prefix && (g.concat || g.prefix_token);  // token items have a part of the prefix
  if (g.kv_heads > 1 && !(g.kc_headed && g.vc_headed && (!token_prefix || (g.pk_headed && g.pv_headed)))) {
    // heads that share one have no box of several
    g.heads = 1;
    g.groups = g.kv_heads;
    g.teams = kMostTeams;
  }
  // a team's rings: query rows for one segment, for two where 8 rows a head are enough, tiles in the rest
  const long long most_rows = p.q_starts || (g.prefix_token && !g.concat) ? (long long)p.tokens * g.group : g.group;
  g.q_rows = most_rows <= 8 ? 8 : 16;
  g.q_slots = most_rows <= 8 ? 2 : 1;
  const int team_bytes = (int)C::kTiles / g.teams - g.q_slots * g.heads * g.q_rows * 128 * C::kHalves;
  g.entries = std::min(kMostEntries, team_bytes / (g.heads * (int)C::kEntry));
  // What a unit takes of an SM in units of 10 ns, as measured at head_dim 128 (and, token units, 64): a tile unit 2 us of the
  // chain; a token unit what its boxes take, whole ones of 64 columns whatever head_dim fills of them.  (They share the CTAs
  // out, and change no result but by the order of its sums; a sweep scatters by 2 %.)  An item's start and end is as long as
  // four tile units (its query rows, the first scores, the last product, the rows written).  When they were chosen, 64 single
  // tokens behind 8192 keys, 32/8 heads of 128, took 47.6 us (four inputs in turn); with tile units at 170, 190 and 245 50.3,
  // 48.5 and 48.2, with items of 3 and 5 tile units 48.6 and 47.1, with token items of 2 units 48.4; 60 requests of 8 tokens
  // 27.4, 26.6 with 3 and 27.5 with 5; a prompt of 4096 tokens was slowest with 2 and alike with 3 and 4.  Token units
  // at 18, 26 and 30, some steps before: 51, 53 and 55 us, 51 with 22.
  g.tile_cost = 215;
  g.token_cost = g.heads * (DP == 128 ? 22 : 16);
  g.tile_item = 4;
  g.token_item = 1;
  const int page = 1 << p.page_shift;
  g.box = std::min(page, kTokenKeys);
  // What a launch cannot come to needs no map (0.25 us each): without q_starts every request is of one kind, and the
  // prefix has items of one kind alone unless they are part of the requests'.
  const bool own_tile = p.q_starts || g.group > kTokenRows, own_token = g.group <= kTokenRows;
  Maps tile, token;
  tile.q = prefix_query_map(p, g, g.gt, g.nt, 1);
  token.q = own_token ? prefix_query_map(p, g, g.group, g.q_rows / g.group, g.heads) : tile.q;
  auto fill = [&](Maps& m, bool own, bool pre, int heads) {
    m.pk = m.pv = m.kc = m.vc = m.q;
    if (own) {
      m.kc = prefix_kv_map(p.k_cache, p.pages, page, p.head_dim, g.box, heads);
      m.vc = prefix_kv_map(p.v_cache, p.pages, page, p.head_dim, g.box, heads);
    }
    if (p.prefix && (g.concat ? own : pre)) {
      m.pk = prefix_kv_map(p.prefix_k, 1, p.prefix, p.head_dim, kTokenKeys, heads);
      m.pv = prefix_kv_map(p.prefix_v, 1, p.prefix, p.head_dim, kTokenKeys, heads);
    }
  };
  fill(tile, own_tile, !g.prefix_token, 1);
  fill(token, own_token, g.prefix_token, g.heads);
  const double values = (double)p.tokens * p.q.heads * p.head_dim;
  {
    // (the own tokens are counted on the GPU)
    LaunchScope scope("prefix_attention", 4.0 * values * p.prefix,
                      4.0 * values + 4.0 * p.prefix * g.kv_heads * p.head_dim, s);
    prefix_attention_kernel<T, DP><<<num_sms, kThreads, C::kSmem, s>>>(tile, token, p, g);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  const long long n = (long long)p.tokens * p.q.heads;
  LaunchScope scope("prefix_join", 0.0, 0.0, s);
  if (g.concat && n > 16384) {
    DependentLaunch l(dim3(num_sms * g.teams, 128 / 8), 256, 0, s);
    return cudaLaunchKernelEx(&l.cfg, prefix_join_cuts_kernel<T>, p, g, num_sms);
  }
  // so few rows that all warps of a block can share one, or a row a warp
  const bool wide = n <= 4LL * num_sms;
  DependentLaunch l(dim3((unsigned)(wide ? n : (n + 7) / 8)), 256, 0, s);
  return wide ? cudaLaunchKernelEx(&l.cfg, prefix_join_kernel<T, true>, p, g, num_sms)
              : cudaLaunchKernelEx(&l.cfg, prefix_join_kernel<T, false>, p, g, num_sms);
}

template <typename T>
cudaError_t launch_t(const PrefixAttnParams& p, int num_sms, cudaStream_t s) {
  Layout x = make_layout(p.tokens, p.requests, p.prefix, p.q.heads, p.k_cache.heads, p.head_dim, num_sms);
  // (the caller's workspace starts on 16 bytes, the parts are written 32 at a time)
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.ws) + kSpare + 15) & ~(uintptr_t)(kSpare + 15));
  x.g.where = reinterpret_cast<int*>(ws);
  x.g.cuts = reinterpret_cast<Segment*>(ws + x.cuts);
  x.g.bad = reinterpret_cast<int*>(x.g.cuts + num_sms * kMostTeams);
  x.g.tile_slots = reinterpret_cast<float*>(ws + x.tile_slots);
  x.g.token_slots = reinterpret_cast<float*>(ws + x.token_slots);
  x.g.whole = reinterpret_cast<float*>(ws + x.whole);
  return p.head_dim <= 64 ? launch_k<T, 64>(p, x.g, num_sms, s) : launch_k<T, 128>(p, x.g, num_sms, s);
}

// CTAs of a launch: one an SM, as many as a row's code can name.
int ctas_of(int num_sms) { return std::min(num_sms, kTileWorkers / kMostTeams); }

}  // namespace

long long prefix_attention_workspace(int tokens, int requests, int prefix, int q_heads, int kv_heads, int head_dim,
                                     int num_sms) {
  if (tokens == 0 || requests == 0) return 0;
  return make_layout(tokens, requests, prefix, q_heads, kv_heads, head_dim, ctas_of(num_sms)).bytes + kSpare;
}

cudaError_t launch_prefix_attention(const PrefixAttnParams& p, int bf16, int num_sms, cudaStream_t stream) {
  if (p.requests == 0) {
    const long long pieces = (long long)p.tokens * p.out.heads * (p.head_dim / 8);
    LaunchScope scope("prefix_zero", 0.0, 16.0 * pieces, stream);
    prefix_zero_kernel<<<(unsigned)std::min((pieces + 255) / 256, 8LL * num_sms), 256, 0, stream>>>(p);
    return cudaGetLastError();
  }
  return bf16 ? launch_t<__nv_bfloat16>(p, ctas_of(num_sms), stream) : launch_t<__half>(p, ctas_of(num_sms), stream);
}

MSST_DEFINE_ERROR_ACCESSOR(prefix_attn_device_error)

}  // namespace msst
