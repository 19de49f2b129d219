// prefix_attn.cu — attention of a batch's new tokens to a prefix that all requests share and to
// each request's own tokens in the pages of a cache, causal among the new ones.
//
// With the keys of row i split in the prefix's and the request's own, softmax(s) v is the joined
// result of two attentions with a running reference and sum each.  So the prefix's part takes the
// rows of ALL requests at once: the group's query heads of every token are packed into 128-row
// tiles and each K/V tile of the prefix is read for 256 rows, not for a request's few.  The own
// part has an item for each request and key head.
//
// One launch does both.  Items are cut into units (a K/V tile of 128 keys for a pair of row tiles, two
// for a lone one; 64 keys for up to 16 rows), in two sequences:
//   tile items   more than 16 rows: tcgen05, 128-row tiles (tile_role, as cross_attn.cu)
//   token items  up to 16 rows, a request's single token or a few: mma.sync (token_role, as
//                cross_token.cu), bound by reading K and V
// Every CTA sums the units of both from the lengths, shares the CTAs out by what a unit of each costs
// and takes an equal contiguous run of its sequence.  The prefix's products and the reading of the
// requests' own pages so overlap, and nothing is known on the host but the tensors' sizes.
// prefix_join_kernel adds up the parts of a row in a fixed order.
//
// Long prompts (256 rows a request and more) take prefix and own keys as one sequence instead: the rows of one
// request fill the tiles, and only items that a CTA's run cuts are joined.
//
// What a row does not see is selected away; V rows past a request's last token are zeroed in shared memory
// before the MMA.  The V rows of new tokens cannot be, as later rows see them: where one of
// those holds an infinity or NaN (0 * NaN would reach the rows before), the item's rows are computed again, key by
// key, by the joining kernel.
#include <algorithm>

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
constexpr int kTokenKeys = 64, kTokenWarps = 8;
constexpr uint32_t kTokenBox = kTokenKeys * 128;  // 64 keys x 64 columns
constexpr int kMaxStages = 12;
constexpr int kRecompute = -1;

template <int DP>
struct PCfg {
  static constexpr int kHalves = DP / 64;
  static constexpr uint32_t kTile = kHalves * kHalfBytes;  // one Q, K or V tile
  static constexpr int kKSlots = DP == 128 ? 3 : 5, kVSlots = DP == 128 ? 2 : 5;
  static constexpr uint32_t kTail = 2560;  // barriers and exchange of either role
  static constexpr size_t kSmem = (2 + kKSlots + kVSlots) * kTile + kTail;
  static_assert((19 + 2 * kKSlots + 3 * kVSlots) * 8 + 16 + 2048 <= kTail, "tile role");
  static_assert(2 * kMaxStages * 8 + 16 + 2 * kTokenWarps * 16 * 4 <= kTail, "token role");
  static constexpr int kBufs = DP == 128 ? 2 : 3;
  static constexpr uint32_t kColO = kBufs * 128;
  static constexpr uint32_t kStage = 2 * kHalves * kTokenBox;  // token role: K, then V
};

// What the host knows of a launch.
struct PrefixGeom {
  int kv_heads, group;
  int gt, nt, g_tiles;        // heads and tokens of a row tile, tiles along the group
  int ksteps;
  int concat;                 // an item's keys are the prefix's and then its own (no items for the prefix alone)
  int prefix_tiles, prefix_tiles64;
  int prefix_token;           // all rows of a key head are at most 16: the prefix's item is a token item
  int n_tiles, full, lone;    // the prefix's tile items
  int box;                    // rows of a cache's TMA box
  int pk_headed, pv_headed, kc_headed, vc_headed;
  int stages, slot_rows, ld;  // ring of the token role; rows and row length (floats) of a partial result
  int tile_cost, token_cost;  // of a unit
  int* where;                 // [phase][tokens * q_heads] which partial results a row has
  float* slots;               // [CTA][begins, ends][slot_rows][ld]
  float* whole;               // [phase][tokens * q_heads][ld] results of items that one CTA had whole
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
      end = min((max(a % n_tiles, b % n_tiles) + 1) * g.nt, q.n);
    }
    const int keys = q.own ? q.limit(end - 1) : 0, shift = token ? 6 : 7;
    return max(1, ptiles + ((keys + (1 << shift) - 1) >> shift));
  }
  __device__ __forceinline__ int units(int t, int tiles) const { return t < full ? tiles : (tiles + 1) >> 1; }
  __device__ __forceinline__ long long head_units(const PrefixGeom& g, const Request& q, bool token, int ptiles) const {
    long long sum = 0;
    for (int t = 0; t < full + lone; ++t) sum += units(t, tiles(g, q, token, t, ptiles));
    return sum;
  }
};

__device__ __forceinline__ int prefix_part(const PrefixGeom& g, bool token) {
  return token ? g.prefix_tiles64 : g.prefix_tiles;
}
// Units of the prefix's own items in the sequence of token or tile items.
__device__ __forceinline__ long long prefix_units(const PrefixGeom& g, bool token) {
  if (g.concat || (bool)g.prefix_token != token) return 0;
  if (token) return (long long)g.kv_heads * g.prefix_tiles64;
  return (long long)g.kv_heads * ((long long)g.full * g.prefix_tiles + g.lone * ((g.prefix_tiles + 1) >> 1));
}

// A CTA's run: units [u0, u0 + count) of the U of its sequence, CTAs [base, base + ctas); where it starts.
struct Run {
  long long u0, count, U;
  int token, base, ctas;
  int phase, r, hk, t, j;
};

// Exclusive sum over the CTA's threads and the total (s: a slot a warp).
__device__ __forceinline__ long long cta_scan(long long v, long long* s, long long& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) s[warp] = incl;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s[w];
    total += s[w];
  }
  __syncthreads();
  return before + incl - v;
}

// All threads: this CTA's run, from the lengths of all requests.
__device__ void find_run(const PrefixAttnParams& p, const PrefixGeom& g, Run* run, long long* scratch) {
  const int R = p.requests, tid = threadIdx.x;
  auto units_of = [&](int r, long long& a, long long& b) {
    a = b = 0;
    if (r >= R) return;
    const Request q = load_request(p, r);
    if (q.n == 0) return;
    const bool token = is_token(g, q);
    const long long u = Items(g, q, token).head_units(g, q, token, g.concat ? prefix_part(g, token) : 0) * g.kv_heads;
    (token ? b : a) = u;
  };
  long long a = 0, b = 0, mine_a, mine_b;
  for (int r = tid; r < R; r += kThreads) {
    units_of(r, mine_a, mine_b);
    a += mine_a;
    b += mine_b;
  }
  long long total_a, total_b;
  cta_scan(a, scratch, total_a);
  cta_scan(b, scratch, total_b);
  total_a += prefix_units(g, false);
  total_b += prefix_units(g, true);
  // CTAs of the tile items and of the token items
  const long long G = gridDim.x, cost_a = total_a * g.tile_cost, cost_b = total_b * g.token_cost;
  long long ca = cost_a + cost_b > 0 ? (G * cost_a + (cost_a + cost_b) / 2) / (cost_a + cost_b) : 0;
  if (total_a > 0) ca = max(ca, 1LL);
  if (total_b > 0) ca = min(ca, G - 1);
  const long long cb = min(G - ca, total_b);
  const bool token = blockIdx.x >= ca;
  ca = min(ca, total_a);
  Run x;
  x.token = token;
  x.U = token ? total_b : total_a;
  // the token items' CTAs are the grid's last ones
  x.base = token ? (int)(G - cb) : 0;
  x.ctas = (int)(token ? cb : ca);
  const long long c = (long long)blockIdx.x - x.base;
  if (c < 0 || c >= x.ctas) {
    x.u0 = x.count = 0;
  } else {
    x.u0 = x.U * c / x.ctas;
    x.count = x.U * (c + 1) / x.ctas - x.u0;
  }
  x.phase = x.r = x.hk = x.t = x.j = 0;
  if (x.count > 0) {
    const long long pre = prefix_units(g, token);
    if (x.u0 < pre) {
      if (tid == 0) {
        const long long head = pre / g.kv_heads, off = x.u0 % head;
        const int tiles = prefix_part(g, token);
        x.hk = (int)(x.u0 / head);
        const long long pairs = token ? tiles : (long long)g.full * tiles;
        x.t = off < pairs ? (int)(off / tiles) : g.full;
        x.j = (int)(off < pairs ? off % tiles : off - pairs);
        *run = x;
      }
    } else {
      long long target = x.u0 - pre;
      for (int r0 = 0; r0 < R; r0 += kThreads) {
        units_of(r0 + tid, mine_a, mine_b);
        const long long mine = token ? mine_b : mine_a;
        long long total;
        const long long before = cta_scan(mine, scratch, total);
        if (before <= target && target < before + mine) {
          const Request q = load_request(p, r0 + tid);
          const Items it(g, q, token);
          const int ptiles = g.concat ? prefix_part(g, token) : 0;
          long long off = target - before;
          x.phase = 1;
          x.r = r0 + tid;
          x.hk = (int)(off / (mine / g.kv_heads));
          off -= x.hk * (mine / g.kv_heads);
          for (;; ++x.t) {
            const int u = it.units(x.t, it.tiles(g, q, token, x.t, ptiles));
            if (off < u) break;
            off -= u;
          }
          x.j = (int)off;
          *run = x;
        }
        if (target < total) break;  // the same for all threads
        target -= total;
      }
    }
  } else if (tid == 0) {
    *run = x;
  }
  __syncthreads();
}

// Walks the segments (one item each) of a run.
struct PrefixWalk {
  const PrefixAttnParams& p;
  const PrefixGeom& g;
  bool token;
  int phase, r, hk, t;
  long long left, at;  // units left; the sequence's unit that the segment starts with
  Request q;
  Items it;
  int ptiles;
  int seg, tiles, units, j0, j1;
  bool lone;
  __device__ __forceinline__ PrefixWalk(const PrefixAttnParams& p_, const PrefixGeom& g_, const Run& x)
      : p(p_), g(g_), token(x.token), phase(x.phase), r(x.r), hk(x.hk), t(x.t), left(x.count), at(x.u0), seg(-1), j0(0), j1(x.j) {
    if (left > 0) set_request();
  }
  __device__ __forceinline__ void set_request() {
    if (phase == 0) {
      q.q0 = 0, q.n = p.tokens, q.own = 0;
    } else {
      q = load_request(p, r);
    }
    it = Items(g, q, token);
    ptiles = phase == 0 || g.concat ? prefix_part(g, token) : 0;
  }
  __device__ __forceinline__ bool next() {
    const int from = j0;
    j0 = seg < 0 ? j1 : 0;
    if (left <= 0) return false;
    if (seg >= 0) {
      at += j1 - from;
      if (++t == it.full + it.lone) {
        t = 0;
        if (++hk == g.kv_heads) {
          hk = 0;
          if (phase == 0) phase = 1, r = -1;
          for (;;) {
            if (++r >= p.requests) return false;  // not reached while units are left
            set_request();
            if (q.n > 0 && is_token(g, q) == token) break;
          }
        }
      }
    }
    ++seg;
    tiles = it.tiles(g, q, token, t, ptiles);
    lone = t == it.full;
    units = it.units(t, tiles);
    j1 = (int)min((long long)units, j0 + left);
    left -= j1 - j0;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == units; }
  // tile role: K/V tile of row tile w in unit j, and whether it has one
  __device__ __forceinline__ int kv_tile(int w, int j) const { return lone ? 2 * j + w : j; }
  __device__ __forceinline__ bool uses(int w, int j) const { return kv_tile(w, j) < tiles; }
  // first token (of the item's rows) and head of row tile w
  __device__ __forceinline__ void origin(int w, int& n0, int& g0) const {
    const int tile = lone ? 2 * it.full : 2 * t + w, gi = tile / it.n_tiles;
    n0 = (tile - gi * it.n_tiles) * g.nt;
    g0 = gi * g.gt;
  }
  // Where the parts of the segment's item are: the CTA that starts it writes this for each row.  Bits: the row of
  // a slot, the first CTA, how many CTAs follow it (0: one had it whole).
  __device__ __forceinline__ int code(const Run& x, int row) const {
    if (j1 == units) return row;
    const long long last = at + units - 1;
    const int c0 = (int)blockIdx.x, c1 = x.base + (int)(((last + 1) * x.ctas - 1) / x.U);
    return row | c0 << 8 | (c1 - c0) << 20;
  }
  // A part of the item: its slot in this CTA
  __device__ __forceinline__ float* slot(const PrefixGeom& gg) const {
    return gg.slots + (size_t)(2 * blockIdx.x + (j0 > 0)) * gg.slot_rows * gg.ld;
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

// Whether one of the 16-bit values in w is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool any_non_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w >> 16 & e) == e;
}

// ------------------------------------------------------------------------------- tile items
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
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + C::kVSlots * C::kTile);
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

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&pv_done[w], 1);
      mbar_init(&o_done[w], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&meet[i], 2);
    mbar_init(mma_end, 1);
    for (int i = 0; i < C::kKSlots; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < C::kVSlots; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ready[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    *abort_flag = 0;
    *s_bad = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  PrefixWalk k(p, g, run);

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
                             uint64_t* bar, int tile) {
          if (tile < k.ptiles) {
            mbar_arrive_expect_tx(bar, C::kTile);
            for (int h = 0; h < C::kHalves; ++h)
              for (int b = 0; b < 2; ++b)
                tma_load_4d(dst + h * kHalfBytes + b * 8192, &pre, bar, h * 64, tile * 128 + b * 64, k.hk * pre_headed, 0);
            return;
          }
          const int key0 = (tile - k.ptiles) * 128, boxes = min(128 / g.box, max(0, (k.q.own - key0 + g.box - 1) / g.box));
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
        while (ok && k.next()) {
          if (!(ok = mbar_wait<false>(q_empty, q_phase ^ 1, kErrTimeoutAttnQ, abort_flag))) break;
          q_phase ^= 1;
          const int nq = k.lone ? 1 : 2;
          mbar_arrive_expect_tx(q_full, nq * C::kHalves * (uint32_t)(g.gt * g.nt) * 128u);
          for (int w = 0; w < nq; ++w) {
            int n0, g0;
            k.origin(w, n0, g0);
            for (int h = 0; h < C::kHalves; ++h)
              tma_load_4d(sQ + w * C::kTile + h * kHalfBytes, &qmap, q_full, h * 64, g0, k.q.q0 + n0, k.hk);
          }
          const int streams = k.lone ? 2 : 1;  // K/V tiles of a unit
          // with three buffers S runs ahead of PV by up to two units, so K goes first
          constexpr int kLead = NB == 3 ? 1 : 0;
          for (int i = k.j0; ok && i < k.j1 + kLead; ++i) {
            for (int w = 0; w < streams && i < k.j1 && k.uses(w, i); ++w) {
              if (!(ok = mbar_wait<false>(&k_empty[kp.slot], kp.phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
              load_tile(pkmap, g.pk_headed, kcmap, g.kc_headed, sK + kp.slot * C::kTile, &k_full[kp.slot], k.kv_tile(w, i));
              kp = kp.plus(1);
            }
            const int v = i - kLead;
            for (int w = 0; ok && w < streams && v >= k.j0 && k.uses(w, v); ++w) {
              if (!(ok = mbar_wait<false>(&v_empty[vp.slot], vp.phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
              load_tile(pvmap, g.pv_headed, vcmap, g.vc_headed, sV + vp.slot * C::kTile, &v_full[vp.slot], k.kv_tile(w, v));
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
        KPos kp;                    // next K slot to wait for
        VPos vp;
        uint32_t kc[2] = {0, 0};    // slots in use
        uint32_t vc[2] = {0, 0};
        uint32_t mine[2] = {0, 0}, pmine[2] = {0, 0};  // S and PV issued so far, per tile
        uint32_t seq = 0;           // position in the sequence of the segment's first step
        bool ok = true;
        while (ok && k.next()) {
          if (!mbar_wait<false>(q_full, k.seg & 1, kErrTimeoutAttnQ, abort_flag)) break;
          tc_fence_after();
          const int steps = k.j1 - k.j0;
          // steps of the second tile: all, but for a lone tile's last unit without a K/V tile for it
          const int steps1 = k.uses(1, k.j1 - 1) ? steps : steps - 1;
          const bool lone = k.lone;
          // S of step t of tile w
          auto do_s = [&](const int w, const int t) -> bool {
            if (t >= (w ? steps1 : steps)) return true;
            if (w == 0 || lone) {
              if (!mbar_wait<false>(&k_full[kp.slot], kp.phase, kErrTimeoutAttnKV, abort_flag)) return false;
              kc[w] = kp.slot;
              kp = kp.plus(1);
              tc_fence_after();
            }
            const uint32_t slot = lone ? kc[w] : kc[0];
            const StepBuf<NB> b(w, mine[w]++, seq + 2 * t + w);
            const uint64_t dq = dq0 + (uint64_t)((lone ? 0 : w) * kTileDesc);
            const uint64_t dk = dk0 + (uint64_t)(slot * kTileDesc);
            const uint32_t dS = tmem + b.buf * 128;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
              if (kk >= ksteps) break;
              const uint64_t off = (uint64_t)((kk >> 2) * (kHalfBytes >> 4) + (kk & 3) * 2);
              umma_f16_ss(dS, dq + off, dk + off, idesc_s, kk != 0);
            }
            umma_commit(&s_full[b.buf]);
            if (w == 1 || lone) umma_commit(&k_empty[slot]);
            return true;
          };
          // PV of step t of tile w
          auto do_pv = [&](const int w, const int t) -> bool {
            if (t >= (w ? steps1 : steps)) return true;
            if (w == 0 || lone) {
              if (!mbar_wait<false>(&v_ready[vp.slot], vp.phase, kErrTimeoutAttnKV, abort_flag)) return false;
              vc[w] = vp.slot;
              vp = vp.plus(1);
            }
            const uint32_t slot = lone ? vc[w] : vc[0];
            const StepBuf<NB> b(w, pmine[w]++, seq + 2 * t + w);
            if (!mbar_wait<false>(&p_full[b.buf], b.parity, kErrTimeoutAttnP, abort_flag)) return false;
            tc_fence_after();
            const uint64_t dv = dv0 + (uint64_t)(slot * kTileDesc);
            const uint32_t pa = tmem + b.buf * 128, dO = tmem + C::kColO + (uint32_t)(w * DP);
            umma_f16_ts(dO, pa, dv, idesc_o, t > 0);
#pragma unroll
            for (int kk = 1; kk < 8; ++kk) umma_f16_ts(dO, pa + (uint32_t)(kk * 8), dv + 128 * kk, idesc_o, 1u);
            umma_commit(&pv_done[w]);
            if (w == 1 || lone) umma_commit(&v_empty[slot]);
            return true;
          };
          // S(s + NB) behind PV(s)
          if (!(ok = do_s(0, 0) && do_s(1, 0) && (NB == 2 || do_s(0, 1)))) break;
          for (int t = 0; t < steps; ++t) {
            if (!(ok = do_pv(0, t))) break;
            if (t == steps - 1) umma_commit(&o_done[0]);
            if (!(ok = NB == 3 ? do_s(1, t + 1) : do_s(0, t + 1))) break;
            if (!(ok = do_pv(1, t) && (NB == 3 ? do_s(0, t + 2) : do_s(1, t + 1)))) break;
            if (t == (steps > 1 ? steps - 2 : 0)) umma_commit(q_empty);  // every S has been issued
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
      while (ok && k.next()) {
        const int streams = k.lone ? 2 : 1;
        uint32_t bad = 0;
        int n0, g0;
        k.origin(0, n0, g0);
        // own tokens that every row of the item sees (along the group's tiles the tokens start over)
        const int common = k.q.limit(g.g_tiles > 1 ? 0 : n0);
        if (lane == 0) *s_bad = *s_bad & ~(1u << ((k.seg + 16) & 31));  // read by all long ago
        for (int j = k.j0; ok && j < k.j1; ++j) {
          for (int w = 0; w < streams && k.uses(w, j); ++w) {
            if (!(ok = mbar_wait_warp<false>(&v_full[vp.slot], vp.phase, kErrTimeoutAttnKV, abort_flag))) break;
            const int tile = k.kv_tile(w, j);
            const bool pre = tile < k.ptiles;
            const int key0 = (pre ? tile : tile - k.ptiles) * 128;
            const int khi = (pre ? p.prefix : k.q.own) - key0, klo = pre ? khi : common - key0;
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
              bool found = false;
              for (int row = max(klo, 0) + lane; row < min(khi, 128); row += 32) {
#pragma unroll
                for (int x = 0; x < 8 * C::kHalves; ++x) {
                  const uint4 v = *reinterpret_cast<const uint4*>(tile_at + row * 128 + (x >> 3) * kHalfBytes +
                                                                  (((x + lane) & 7) << 4));
                  found |= any_non_finite<T>(v.x) || any_non_finite<T>(v.y) || any_non_finite<T>(v.z) || any_non_finite<T>(v.w);
                }
              }
              if (__any_sync(0xffffffffu, found) && !bad) {
                bad = 1;
                if (lane == 0) *s_bad = *s_bad | 1u << (k.seg & 31);
              }
            }
            if (lane == 0) mbar_arrive(&v_ready[vp.slot]);
            vp = vp.plus(1);
          }
        }
      }
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
    while (ok && k.next()) {
      int n0, g0;
      k.origin(w, n0, g0);
      const int rn = row / g.gt, n = n0 + rn, head = g0 + row - rn * g.gt;
      const bool valid = rn < g.nt && n < k.q.n && head < g.group;
      const bool warp_active = __any_sync(0xffffffffu, valid);
      const int limit = valid ? k.q.limit(n) : k.q.own;  // own tokens that the row sees
      float ref = 0.f, l = 0.f;
      bool have = false;  // the reference is set
      const int all_steps = k.j1 - k.j0, steps1 = k.uses(1, k.j1 - 1) ? all_steps : all_steps - 1;
      const int steps = w ? steps1 : all_steps;
      for (int t = 0; t < steps; ++t, ++mine) {
        const StepBuf<NB> b(w, mine, seq + 2 * t + w);
        const uint32_t sAddr = tmem + lane_off + b.buf * 128;
        const int tile = k.kv_tile(w, k.j0 + t);
        const int khi = tile < k.ptiles ? p.prefix - tile * 128 : limit - (tile - k.ptiles) * 128;
        const bool all = __all_sync(0xffffffffu, khi >= 128), any = __any_sync(0xffffffffu, khi > 0);
        if (!mbar_wait_warp<false>(&s_full[b.buf], b.parity, kErrTimeoutAttnS, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_active) {
          uint32_t words[4];
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) words[ch] = len_word(khi, ch);
          uint32_t pk[64];
          if (any) {
            if (!have) {
              uint32_t r[32];
              tmem_ld32(sAddr, r);
              tmem_ld_wait(r);
              // -inf for a row that sees none of these keys or whose scores are -inf: no reference yet, and
              // sums against it are not finite, which sends every step through the exact passes until one finds a score
              ref = chunk_max(r, words[0], c) - kRefShift<T>;
              have = true;
            }
            float sum = all ? row_exp<T, true>(sAddr, words, c, ref, pk) : row_exp<T, false>(sAddr, words, c, ref, pk);
            if (__any_sync(0xffffffffu, valid && !(sum <= kSumLimit<T>))) {
              // exact passes: the reference moves to the row's maximum, O and l with it
              float m = -INFINITY;
#pragma unroll 1
              for (int ch = 0; ch < 4; ++ch) {
                uint32_t r[32], word = words[0];
#pragma unroll
                for (int i = 1; i < 4; ++i)
                  if (i == ch) word = words[i];
                tmem_ld32(sAddr + ch * 32, r);
                tmem_ld_wait(r);
                m = fmaxf(m, chunk_max(r, word, c));
              }
              const float moved = fmaxf(ref, m - kRefShift<T>), base = moved == -INFINITY ? 0.f : moved;
              const float alpha = fast_exp2(ref - base);
              if (t > 0) {
                // O holds the previous steps once the last PV is through (the one before it was
                // when this step's S was issued, so the parity is the right phase's)
                if (!mbar_wait_warp<false>(&pv_done[w], (mine - 1) & 1, kErrTimeoutAttnO, abort_flag)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
#pragma unroll 1
                for (int h = 0; h < DP / 32; ++h) {
                  uint32_t r[32];
                  tmem_ld32(oAddr + h * 32, r);
                  tmem_ld_wait(r);
#pragma unroll
                  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                  tmem_st32(oAddr + h * 32, r);
                }
                tmem_st_wait();
              }
              l *= alpha;
              ref = moved;
              sum = row_exp<T, false>(sAddr, words, c, base, pk);
            }
            l += sum;
          } else {
#pragma unroll
            for (int i = 0; i < 64; ++i) pk[i] = 0u;
          }
          tmem_st32(sAddr, *reinterpret_cast<const uint32_t(*)[32]>(pk));
          tmem_st32(sAddr + 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
          tmem_st_wait();
        }
        // (a barrier a buffer: the tile's other warps may be a step ahead)
        tc_fence_before();
        mbar_arrive(&p_full[b.buf]);
      }
      if (!ok) break;
      seq += (uint32_t)(all_steps + steps1);
      if (!mbar_wait_warp<false>(&o_done[w], k.seg & 1, kErrTimeoutAttnO, abort_flag)) break;
      tc_fence_after();
      const bool bad = *s_bad >> (k.seg & 31) & 1;
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
      const bool whole = k.whole(), finish = whole && g.concat;
      const float inv = finish ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
      const float f0 = a0 * inv, f1 = a1 * inv;
      if (warp_active) {
        const size_t grow = (size_t)(k.q.q0 + n) * p.q.heads + (size_t)(k.hk * g.group + head);
        const size_t plane = (size_t)p.tokens * p.q.heads * k.phase;
        T* out = static_cast<T*>(p.out.data) + (k.q.q0 + n) * p.out.seq_stride +
                 (long long)(k.hk * g.group + head) * p.out.head_stride;
        const int at = (k.lone ? 0 : w * 128) + row;
        float* po = whole ? g.whole + (plane + grow) * g.ld : k.slot(g) + (size_t)at * g.ld;
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
          if (k.j0 == 0) g.where[plane + grow] = finish && bad ? kRecompute : k.code(run, at);
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
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------- token items
// 16-byte piece `chunk` (8 columns) of key `row` in a 128B-swizzled tile of 64-column boxes
__device__ __forceinline__ uint32_t token_piece(uint32_t tile, int row, int chunk) {
  return tile + (uint32_t)((chunk >> 3) * kTokenBox + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

template <typename T, int DP>
__device__ void token_role(uint8_t* smem, const CUtensorMap& pkmap, const CUtensorMap& pvmap, const CUtensorMap& kcmap,
                           const CUtensorMap& vcmap, const PrefixAttnParams& p, const PrefixGeom& g, const Run& run) {
  using C = PCfg<DP>;
  constexpr int kHalves = C::kHalves;
  constexpr uint32_t kStage = C::kStage;
  const int stages = g.stages;
  float* s_o = reinterpret_cast<float*>(smem + (size_t)stages * kStage);  // [warps][rows][DP]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kSmem - C::kTail);
  uint64_t* empty = full + kMaxStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kMaxStages);
  int* s_stop = const_cast<int*>(abort_flag) + 1;
  volatile int* s_bad = abort_flag + 2;  // [2]: by the parity of the segment
  float(*s_m)[16] = reinterpret_cast<float(*)[16]>(const_cast<int*>(abort_flag) + 4);
  float(*s_l)[16] = s_m + kTokenWarps;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    s_bad[0] = s_bad[1] = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp > kTokenWarps) return;
  PrefixWalk k(p, g, run);

  if (warp == kTokenWarps) {
    if (lane == 0) {
      int st = 0;
      uint32_t phase = 0;
      bool ok = true;
      // pages of tile j's boxes, asked for a tile ahead
      auto pages_of = [&](int j, int (&page)[4]) {
        const int key0 = (j - k.ptiles) * kTokenKeys;
        const int* row = p.table + k.r * p.table_stride;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          page[i] = key0 >= 0 && i * g.box < kTokenKeys && key0 + i * g.box < k.q.own
                        ? __ldg(row + ((key0 + i * g.box) >> p.page_shift))
                        : 0;
      };
      while (ok && k.next()) {
        int page[4], ahead[4];
        pages_of(k.j0, page);
        for (int j = k.j0; j < k.j1; ++j) {
          pages_of(j + 1, ahead);
          if (!mbar_wait<false>(&empty[st], phase ^ 1, kErrTimeoutAttnKV, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + (size_t)st * kStage;
          if (j < k.ptiles) {
            mbar_arrive_expect_tx(&full[st], kStage);
            for (int h = 0; h < kHalves; ++h) {
              tma_load_4d(dst + h * kTokenBox, &pkmap, &full[st], h * 64, j * kTokenKeys, k.hk * g.pk_headed, 0);
              tma_load_4d(dst + (kHalves + h) * kTokenBox, &pvmap, &full[st], h * 64, j * kTokenKeys, k.hk * g.pv_headed, 0);
            }
          } else {
            const int key0 = (j - k.ptiles) * kTokenKeys;
            const int boxes = min(kTokenKeys / g.box, max(0, (k.q.own - key0 + g.box - 1) / g.box));
            mbar_arrive_expect_tx(&full[st], (uint32_t)(boxes * g.box) * 128u * 2 * kHalves);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i >= boxes) break;
              const int at = (key0 + i * g.box) & ((1 << p.page_shift) - 1), id = checked_page(p, page[i]);
              uint8_t* to = dst + i * g.box * 128;
              for (int h = 0; h < kHalves; ++h) {
                tma_load_4d(to + h * kTokenBox, &kcmap, &full[st], h * 64, at, k.hk * g.kc_headed, id);
                tma_load_4d(to + (kHalves + h) * kTokenBox, &vcmap, &full[st], h * 64, at, k.hk * g.vc_headed, id);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) page[i] = ahead[i];
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
  while (ok && k.next()) {
    const int rows = k.q.n * g.group;
    // Q fragments of the rows r = n * group + head of the group, from global memory
    uint32_t qa[DP / 16][4];
    int limit[2];  // own tokens that the fragment's two rows see
    {
      const T* qp = static_cast<const T*>(p.q.data) + k.q.q0 * p.q.seq_stride +
                    (long long)k.hk * g.group * p.q.head_stride;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = qr + 8 * half, n = r / g.group, h = r - n * g.group;
        const T* row = qp + (long long)n * p.q.seq_stride + (long long)h * p.q.head_stride;
        limit[half] = r < rows ? k.q.limit(n) : k.q.own;
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
    const int common = k.q.limit(0);
    bool bad = false;
    for (int jj = k.j0; jj < k.j1; ++jj) {
      const int stage = st;
      const uint32_t par = phase;
      if (++st == stages) st = 0, phase ^= 1;
      if ((stage & 1) != set) continue;
      if (!mbar_wait_warp<false>(&full[stage], par, kErrTimeoutAttnKV, abort_flag)) {
        ok = false;
        break;
      }
      const uint32_t kt = base + (uint32_t)stage * kStage, vt = kt + kHalves * kTokenBox;
      // S: two column tiles of 8 keys; even and odd k-steps in accumulators of their own
      float sc[2][2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) (&sc[0][0][0])[i] = 0.f;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        uint32_t b[4];
        ldmatrix4(token_piece(kt, krow, 2 * s + kchunk), b);
        mma16816<T>(sc[s & 1][0], qa[s], b[0], b[1]);
        mma16816<T>(sc[s & 1][1], qa[s], b[2], b[3]);
      }
      // of this warp's 16 keys: the first khi are there, the first klo are seen by every row
      const bool pre = jj < k.ptiles;
      const int key0 = (pre ? jj : jj - k.ptiles) * kTokenKeys + wk * 16;
      const int khi = (pre ? p.prefix : k.q.own) - key0, klo = pre ? khi : common - key0;
      const bool all = klo >= 16;
      const int lim[2] = {pre ? khi : limit[0] - key0, pre ? khi : limit[1] - key0};
      float e[2][4];
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // i: row half * 2 + key of the pair
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float x = (sc[0][t][i] + sc[1][t][i]) * c;
          e[t][i] = all || 8 * t + qc * 2 + (i & 1) < lim[i >> 1] ? x : -INFINITY;
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
      // keys that are not there: their V is taken as zero (0 * NaN would reach the sum)
      const int k0 = qc * 2;
      const uint32_t v0 = (k0 < khi ? 0xffffu : 0u) | (k0 + 1 < khi ? 0xffff0000u : 0u);
      const uint32_t v1 = (k0 + 8 < khi ? 0xffffu : 0u) | (k0 + 9 < khi ? 0xffff0000u : 0u);
      const bool ask = klo < min(khi, 16);  // keys that some rows see and others do not
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t b[4];
        ldmatrix4_trans(token_piece(vt, vrow, 2 * i + vchunk), b);
        if (!all) {
          b[0] &= v0;
          b[1] &= v1;
          b[2] &= v0;
          b[3] &= v1;
          if (ask)
            bad |= any_non_finite<T>(b[0]) || any_non_finite<T>(b[1]) || any_non_finite<T>(b[2]) || any_non_finite<T>(b[3]);
        }
        // a tile's products in accumulators of their own, added in fp32 (see cross_token.cu)
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
    if (bad) s_bad[k.seg & 1] = 1;
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
    if (threadIdx.x == 0) *s_stop = *abort_flag;
    const bool item_bad = s_bad[k.seg & 1] != 0;
    if (threadIdx.x == 0) s_bad[(k.seg + 1) & 1] = 0;
    const bool whole = k.whole(), finish = whole && g.concat;
    for (int x = threadIdx.x; x < rows * (p.head_dim / 4); x += 256) {
      const int r = x / (p.head_dim / 4), col = (x - r * (p.head_dim / 4)) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int i = 0; i < kTokenWarps; ++i) mm = fmaxf(mm, s_m[i][r]);
      float ls = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kTokenWarps; ++i) {
        if (s_l[i][r] == 0.f) continue;
        const float f = fast_exp2(s_m[i][r] - mm);
        const float4 v = *reinterpret_cast<const float4*>(s_o + ((size_t)i * rows + r) * DP + col);
        ls += s_l[i][r] * f;
        sum = make_float4(sum.x + v.x * f, sum.y + v.y * f, sum.z + v.z * f, sum.w + v.w * f);
      }
      const int n = r / g.group, h = k.hk * g.group + r - n * g.group;
      const size_t grow = (size_t)p.tokens * p.q.heads * k.phase + (size_t)(k.q.q0 + n) * p.q.heads + h;
      if (finish) {
        const float inv = ls > 0.f ? 1.f / ls : (ls == 0.f ? 0.f : ls);
        T* out = static_cast<T*>(p.out.data) + (k.q.q0 + n) * p.out.seq_stride + (long long)h * p.out.head_stride + col;
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
      } else {
        float* po = whole ? g.whole + grow * g.ld : k.slot(g) + (size_t)r * g.ld;
        *reinterpret_cast<float4*>(po + col) = sum;
        // the sums are taken against the maximum less kLift
        if (col == 0)
          *reinterpret_cast<float4*>(po + p.head_dim) = make_float4(mm - kLift<T>, ls, item_bad ? 1.f : 0.f, 0.f);
      }
      if (col == 0 && k.j0 == 0) g.where[grow] = finish && item_bad ? kRecompute : k.code(run, r);
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    ok = *s_stop == 0;  // not written again before all have been at the next item's first barrier
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap pkmap,
                            const __grid_constant__ CUtensorMap pvmap, const __grid_constant__ CUtensorMap kcmap,
                            const __grid_constant__ CUtensorMap vcmap, const __grid_constant__ PrefixAttnParams p,
                            const __grid_constant__ PrefixGeom g) {
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzled tiles start on 1024 bytes
  // the run is found in memory that the roles take over
  long long* scratch = reinterpret_cast<long long*>(smem);
  Run* s_run = reinterpret_cast<Run*>(smem + 1024);
  find_run(p, g, s_run, scratch);
  const Run run = *s_run;
  __syncthreads();
  dependents_may_start();
  if (run.count == 0) return;
  if (run.token)
    token_role<T, DP>(smem, pkmap, pvmap, kcmap, vcmap, p, g, run);
  else
    tile_role<T, DP>(smem, qmap, pkmap, pvmap, kcmap, vcmap, p, g, run);
}

// ------------------------------------------------------------------------------- joining
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
    float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    long long page = 0, at = j;
    if (j >= p.prefix) {
      const int i = (int)(j - p.prefix);
      page = checked_page(p, __ldg(p.table + r * p.table_stride + (i >> p.page_shift)));
      at = i & ((1 << p.page_shift) - 1);
    }
    if (page < p.pages) {
      load4(static_cast<const T*>(kv.data) + page * kv.batch_stride + at * kv.seq_stride + hk * kv.head_stride, k);
      load4(static_cast<const T*>(vv.data) + page * vv.batch_stride + at * vv.seq_stride + hk * vv.head_stride, v);
    }
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

// Adds up the parts of each row, in the order of its keys: the prefix's and the own ones (kRows = 1, a warp a
// row), or, of one sequence of both, those of the rows that a run cut (kRows = 32 rows a warp are looked
// through; the others are done).  4 columns a lane, up to kAhead parts in flight.
// Bound: latency.
constexpr int kAhead = 4;

template <typename T, int kRows>
__global__ void __launch_bounds__(256)
    prefix_join_kernel(const __grid_constant__ PrefixAttnParams p, const __grid_constant__ PrefixGeom g, int ctas) {
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)p.tokens * p.q.heads;
  const long long row0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kRows;
  if (row0 >= rows) return;
  wait_for_previous();
  uint32_t todo = 1;
  if (kRows > 1) {
    const long long row = row0 + lane;
    bool need = false;
    if (row < rows && request_of(p, (int)(row / p.q.heads)) >= 0) {
      const int code = g.where[rows + row];
      need = code < 0 || code >> 20;
    }
    todo = __ballot_sync(0xffffffffu, need);
  }
  while (todo) {
    const long long row = row0 + __ffs(todo) - 1;
    todo &= todo - 1;
    const int token = (int)(row / p.q.heads), head = (int)(row - (long long)token * p.q.heads);
    const int r = request_of(p, token);
    if (r < 0) continue;
    const int d = p.head_dim, col = lane * 4;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool again = false;
    for (int phase = kRows > 1 ? 1 : 0; phase < 2; ++phase) {
      const int code = g.where[rows * phase + row];
      if (code < 0) {
        again = true;
        break;
      }
      const int at = code & 255, c0 = code >> 8 & 0xfff, more = code >> 20;
      auto part = [&](int i) -> const float* {
        if (more == 0) return g.whole + (size_t)(rows * phase + row) * g.ld;
        return g.slots + ((size_t)(2 * min(c0 + i, ctas - 1) + (i > 0)) * g.slot_rows + at) * g.ld;
      };
      for (int i0 = 0; i0 <= more; i0 += kAhead) {
        float4 head4[kAhead], x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          head4[i] = x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i0 + i > more) continue;
          const float* f = part(i0 + i);
          head4[i] = __ldcg(reinterpret_cast<const float4*>(f + d));
          if (col < d) x[i] = __ldcg(reinterpret_cast<const float4*>(f + col));
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          again |= head4[i].z != 0.f;
          if (head4[i].y == 0.f) continue;  // no key of that part is seen
          const float mn = fmaxf(m, head4[i].x), a = fast_exp2(m - mn), e = fast_exp2(head4[i].x - mn);
          l = l * a + head4[i].y * e;
          m = mn;
          o[0] = o[0] * a + x[i].x * e;
          o[1] = o[1] * a + x[i].y * e;
          o[2] = o[2] * a + x[i].z * e;
          o[3] = o[3] * a + x[i].w * e;
        }
      }
    }
    if (again) {
      const Request q = load_request(p, r);
      attend_row<T>(p, r, token, head, q.limit(token - q.q0), lane);
    } else if (col < d) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      T* out = static_cast<T*>(p.out.data) + token * p.out.seq_stride + head * p.out.head_stride + col;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
    }
  }
}

// ------------------------------------------------------------------------------- host
// Sizes of a launch, and where the parts of its workspace lie (bytes).
struct Layout {
  PrefixGeom g;
  long long where, slots, whole, bytes;
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
  g.prefix_tiles64 = (int)(((long long)prefix + 63) >> 6);
  g.n_tiles = (tokens + g.nt - 1) / g.nt;
  const int tiles = g.n_tiles * g.g_tiles;
  g.full = tiles / 2;
  g.lone = tiles & 1;
  g.slot_rows = g.prefix_token ? kTokenRows : 256;
  g.ld = head_dim + 8;
  const long long n = (long long)tokens * q_heads;
  auto up = [](long long b) { return (b + 255) & ~255LL; };
  x.slots = up(2 * n * 4);
  x.whole = up(x.slots + 2LL * num_sms * g.slot_rows * g.ld * 4);
  x.bytes = x.whole + (g.concat ? 0 : 2 * n * g.ld * 4);
  return x;
}

CUtensorMap prefix_query_map(const PrefixAttnParams& p, const PrefixGeom& g) {
  // {d, group, tokens, key heads} in boxes of 64 x gt x nt; a stride that is never walked only has to be a legal one
  auto st = [](long long s) { return (uint64_t)(s ? s * 2 : 16); };
  const uint64_t dims[4] = {(uint64_t)p.head_dim, (uint64_t)g.group, (uint64_t)p.tokens, (uint64_t)g.kv_heads};
  const uint64_t str[3] = {st(p.q.head_stride), st(p.q.seq_stride), st(p.q.head_stride * g.group)};
  const uint32_t box[4] = {64, (uint32_t)g.gt, (uint32_t)g.nt, 1};
  return make_tensor_map(p.q.data, 4, dims, str, box);
}

template <typename T, int DP>
cudaError_t launch_k(const PrefixAttnParams& p, PrefixGeom g, int num_sms, cudaStream_t s) {
  using C = PCfg<DP>;
  static std::atomic<unsigned long long> configured;
  cudaError_t e = ensure_smem_limit(prefix_attention_kernel<T, DP>, (int)C::kSmem, configured);
  if (e != cudaSuccess) return e;
  // the ring of the token role: what the joined rows of its largest item leave
  const long long rows = (long long)p.tokens * g.group;
  const long long most = p.q_starts || (g.prefix_token && !g.concat) ? rows : g.group;
  const size_t join = (size_t)kTokenWarps * std::min<long long>(most, kTokenRows) * DP * sizeof(float);
  g.stages = std::min<int>(kMaxStages, (int)((C::kSmem - C::kTail - join) / C::kStage)) & ~1;
  g.tile_cost = 20;
  g.token_cost = DP == 128 ? 8 : 5;
  g.box = std::min(1 << p.page_shift, kTokenKeys);
  const CUtensorMap mq = prefix_query_map(p, g);
  int batched;
  const CUtensorMap mkc =
      cross_kv_map(p.k_cache, p.pages, 1 << p.page_shift, p.head_dim, g.box, batched, g.kc_headed);
  const CUtensorMap mvc =
      cross_kv_map(p.v_cache, p.pages, 1 << p.page_shift, p.head_dim, g.box, batched, g.vc_headed);
  const CUtensorMap mpk = p.prefix ? cross_kv_map(p.prefix_k, 1, p.prefix, p.head_dim, 64, batched, g.pk_headed) : mkc;
  const CUtensorMap mpv = p.prefix ? cross_kv_map(p.prefix_v, 1, p.prefix, p.head_dim, 64, batched, g.pv_headed) : mvc;
  const double values = (double)p.tokens * p.q.heads * p.head_dim;
  {
    // (the own tokens are counted on the GPU)
    LaunchScope scope("prefix_attention", 4.0 * values * p.prefix,
                      4.0 * values + 4.0 * p.prefix * g.kv_heads * p.head_dim, s);
    prefix_attention_kernel<T, DP><<<num_sms, kThreads, C::kSmem, s>>>(mq, mpk, mpv, mkc, mvc, p, g);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  const long long n = (long long)p.tokens * p.q.heads, a_block = 8 * (g.concat ? 32 : 1);
  LaunchScope scope("prefix_join", 0.0, 0.0, s);
  DependentLaunch l(dim3((unsigned)((n + a_block - 1) / a_block)), 256, 0, s);
  return g.concat ? cudaLaunchKernelEx(&l.cfg, prefix_join_kernel<T, 32>, p, g, num_sms)
                  : cudaLaunchKernelEx(&l.cfg, prefix_join_kernel<T, 1>, p, g, num_sms);
}

template <typename T>
cudaError_t launch_t(const PrefixAttnParams& p, int num_sms, cudaStream_t s) {
  Layout x = make_layout(p.tokens, p.requests, p.prefix, p.q.heads, p.k_cache.heads, p.head_dim, num_sms);
  char* ws = reinterpret_cast<char*>(p.ws);
  x.g.where = reinterpret_cast<int*>(ws);
  x.g.slots = reinterpret_cast<float*>(ws + x.slots);
  x.g.whole = reinterpret_cast<float*>(ws + x.whole);
  return p.head_dim <= 64 ? launch_k<T, 64>(p, x.g, num_sms, s) : launch_k<T, 128>(p, x.g, num_sms, s);
}

// CTAs of a launch: one an SM, as many as a row's code can name.
int ctas_of(int num_sms) { return std::min(num_sms, 2047); }

}  // namespace

long long prefix_attention_workspace(int tokens, int requests, int prefix, int q_heads, int kv_heads, int head_dim,
                                     int num_sms) {
  if (tokens == 0 || requests == 0) return 0;
  return make_layout(tokens, requests, prefix, q_heads, kv_heads, head_dim, ctas_of(num_sms)).bytes;
}

cudaError_t launch_prefix_attention(const PrefixAttnParams& p, int bf16, int num_sms, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, ctas_of(num_sms), stream) : launch_t<__half>(p, ctas_of(num_sms), stream);
}

MSST_DEFINE_ERROR_ACCESSOR(prefix_attn_device_error)

}  // namespace msst
