// cross_attn.cu — cross attention to an encoder's states of another length:
// out = softmax(scale q k^T) v over the kept keys, grouped heads, head_dim <= 128.
//
// The query rows of one key head (its group of G query heads times q_len tokens) are
// packed into 128-row tiles: row r of a tile is token n0 + r / gt, head g0 + r % gt
// with gt = min(G, 128), so one K/V tile serves all heads of the group.  A CTA works
// on a PAIR of row tiles that share every K/V tile; a lone last tile (or the only
// one, when there are few rows) runs as a pair of itself with the K/V tiles dealt to
// its two halves in turn, which are merged at the end.
//
// Work is cut into units (one K/V tile for a pair, two for a lone tile) and every CTA
// takes an equal contiguous run of all units, over items of any length (align_runs); the two
// items a run may share with its neighbours leave partial results (O, running
// reference and sum, fp32) in the workspace, which cross_combine_kernel joins in CTA
// order.  So few rows against a long encoder and ragged batches fill the GPU alike.
//
// CTA = 384 threads:
//   warp 0      TMA producer: Q tiles, K and V tiles through a ring each
//   warp 1      MMA issuer: S_w = Q_w K^T (SS) and O_w += P_w V (P from TMEM); owns TMEM
//   warp 2      once a V tile has landed: rows of keys that are not kept are zeroed
//               (0 * NaN would reach the sum otherwise), the tile's mask words published
//   warps 4-11  softmax, tile (warp - 4) / 4, one query row per thread
// The two tiles' steps (one K/V tile each) form one sequence s = 0, 1, 2, ..., tile s % 2.  S(s)
// goes to one of NB buffers of 128 columns in TMEM and P(s) over its first half; S(s + NB) is
// issued right after PV(s) and overwrites P(s) only once PV(s), issued before it by the same
// thread, has read it.  head_dim <= 64 leaves room for NB = 3 next to O_0 and O_1 (2 x 64
// columns): a tile's next scores are there before its softmax asks for them (two buffers:
// 116 us for 4 x 8 heads of 1895 x 3792, three: 99).  Above, NB = 2, one a tile (four of 64 keys:
// 980 us for the long prompts against 752; the 64-column MMAs read as much of Q for half the
// products).
//
// Bound: the chain scores, softmax, product.  4 x 8 heads of 1895 x 3792 x 64: 101 us (584 TFLOP/s), XU
// pipe 63 %, tensor pipe 32 % busy.  4 x 32/8 heads of 4096 x 4096 x 128, ragged: 754 to 759 us
// (1180 TFLOP/s); XU and tensor pipe 59 % busy for one batch entry of it.
//
// Softmax: the reference a row is exponentiated against starts at the maximum of its
// first 32 kept scores (less kRefShift) and moves lazily: a tile is taken in one pass without a
// maximum, and only a row sum above kSumLimit (or not finite) sends the warp through
// the exact two passes, which move the reference and rescale O.  Statistics are fp32;
// P is rounded to the operands' 16 bits for the tensor cores.
#include <algorithm>

#include "attn_steps.cuh"
#include "common.cuh"
#include "cross_attn.cuh"
#include "operators.cuh"
#include "runtime.h"

namespace msst {

namespace {

constexpr int kThreads = 384;
constexpr int kSoftmaxWarp0 = 4;
// Registers a thread after the split: 128 x 88 + 256 x 208 = 384 x 168, the block's launch share
// (2 % faster at both head sizes).  The compiler allocates 168 for every role and spills 88 (head_dim
// <= 64) to 128 bytes; none with the softmax role left out.
constexpr int kFewRegs = 88, kSoftmaxRegs = 208;
constexpr uint32_t kHalfBytes = 128 * 64 * 2;  // 128 rows x 64 columns

template <int DP>
struct Cfg {
  static constexpr int kHalves = DP / 64;
  static constexpr uint32_t kTile = kHalves * kHalfBytes;      // one Q, K or V tile
  static constexpr int kKSlots = DP == 128 ? 3 : 5, kVSlots = DP == 128 ? 2 : 5;
  static constexpr size_t kSmem = (2 + kKSlots + kVSlots) * kTile + 2560;
  static_assert((19 + 2 * kKSlots + 3 * kVSlots) * 8 + 40 + kVSlots * 16 + 2048 <= 2560, "barriers and exchange");
  static constexpr int kBufs = DP == 128 ? 2 : 3;              // NB
  static constexpr uint32_t kColO = kBufs * 128;
};

// First token and head of row tile w of the current segment.
__device__ __forceinline__ void tile_origin(const Walk& k, const Geom& g, int w, int& n0, int& g0) {
  const int tile = k.lone ? 2 * g.full : 2 * k.s.t + w;
  const int gi = tile / g.n_tiles;
  n0 = (tile - gi * g.n_tiles) * g.nt;
  g0 = gi * g.gt;
}

template <typename T, int DP, bool kMask>
__global__ void __launch_bounds__(kThreads, 1)
    cross_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CrossAttnParams p,
                           const __grid_constant__ Geom g) {
  using C = Cfg<DP>;
  constexpr uint32_t kIsBf16 = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzled tiles start on 1024 bytes
  constexpr int NB = C::kBufs;
  using KPos = RingPos<C::kKSlots>;
  using VPos = RingPos<C::kVSlots>;
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * C::kTile;
  uint8_t* sV = sK + C::kKSlots * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + C::kVSlots * C::kTile);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* s_full = bars + 2;   // [NB buffers]
  uint64_t* p_full = bars + 6;   // [NB buffers]
  uint64_t* pv_done = bars + 10; // [2 tiles], every step
  uint64_t* o_done = bars + 12;  // [2 tiles], every item
  uint64_t* meet = bars + 14;    // [4 lane quarters]: the two halves of a lone tile
  uint64_t* mma_end = bars + 18;
  uint64_t* k_full = bars + 19;
  uint64_t* k_empty = k_full + C::kKSlots;
  uint64_t* v_full = k_empty + C::kKSlots;   // landed
  uint64_t* v_ready = v_full + C::kVSlots;   // fit for the MMA
  uint64_t* v_empty = v_ready + C::kVSlots;
  Spot* s_spot = reinterpret_cast<Spot*>(v_empty + C::kVSlots);
  long long* s_count = reinterpret_cast<long long*>(s_spot + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_count + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* s_words = tmem_slot + 4;                                  // [V slots][4] kept keys
  float* s_ml = reinterpret_cast<float*>(s_words + C::kVSlots * 4);   // [2 halves][ref, l][128]

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
    mbar_fence_init();
    tma_prefetch_desc(&qmap);
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tc_fence_before();
  }
  if (warp == 2) {
    const long long U = total_units(p, g, lane);
    const long long u0 = U * blockIdx.x / gridDim.x, u1 = U * (blockIdx.x + 1) / gridDim.x;
    const Spot s = find_spot(p, g, u0, lane);
    if (lane == 0) {
      *s_spot = s;
      *s_count = u1 - u0;
    }
  }
  __syncthreads();
  dependents_may_start();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk k(*s_spot, *s_count);

  if (warp < kSoftmaxWarp0) {
    warpgroup_reg_dec<kFewRegs>();
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        KPos kp;
        VPos vp;
        uint32_t q_phase = 0;
        bool ok = true;
        while (ok && k.next(p, g)) {
          if (!(ok = mbar_wait<false>(q_empty, q_phase ^ 1, kErrTimeoutAttnQ, abort_flag))) break;
          q_phase ^= 1;
          const int nq = k.lone ? 1 : 2;
          mbar_arrive_expect_tx(q_full, nq * C::kHalves * (uint32_t)(g.gt * g.nt) * 128u);
          for (int w = 0; w < nq; ++w) {
            int n0, g0;
            tile_origin(k, g, w, n0, g0);
            for (int h = 0; h < C::kHalves; ++h)
              tma_load_5d(sQ + w * C::kTile + h * kHalfBytes, &qmap, q_full, h * 64, g0, n0, k.s.hk, k.s.b * g.q_batched);
          }
          const int kh = k.s.hk * g.k_headed, kb = k.s.b * g.k_batched;
          const int vh = k.s.hk * g.v_headed, vb = k.s.b * g.v_batched;
          const int streams = k.lone ? 2 : 1;  // K/V tiles of a unit
          // with three buffers S runs ahead of PV by up to two units, so K goes first
          constexpr int kLead = NB == 3 ? 1 : 0;
          for (int i = k.j0; ok && i < k.j1 + kLead; ++i) {
            for (int w = 0; w < streams && i < k.j1 && k.uses(w, i); ++w) {
              if (!(ok = mbar_wait<false>(&k_empty[kp.slot], kp.phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
              mbar_arrive_expect_tx(&k_full[kp.slot], C::kTile);
              for (int h = 0; h < C::kHalves; ++h)
                tma_load_4d(sK + kp.slot * C::kTile + h * kHalfBytes, &kmap, &k_full[kp.slot], h * 64,
                            k.kv_tile(w, i) * 128, kh, kb);
              kp = kp.plus(1);
            }
            const int v = i - kLead;
            for (int w = 0; ok && w < streams && v >= k.j0 && k.uses(w, v); ++w) {
              if (!(ok = mbar_wait<false>(&v_empty[vp.slot], vp.phase ^ 1, kErrTimeoutAttnKV, abort_flag))) break;
              mbar_arrive_expect_tx(&v_full[vp.slot], C::kTile);
              for (int h = 0; h < C::kHalves; ++h)
                tma_load_4d(sV + vp.slot * C::kTile + h * kHalfBytes, &vmap, &v_full[vp.slot], h * 64,
                            k.kv_tile(w, v) * 128, vh, vb);
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
        while (ok && k.next(p, g)) {
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
      // ------------------------------------------------------------ rows that are not kept
      VPos vp;
      bool ok = true;
      while (ok && k.next(p, g)) {
        const int streams = k.lone ? 2 : 1;
        for (int j = k.j0; ok && j < k.j1; ++j) {
          for (int w = 0; w < streams && k.uses(w, j); ++w) {
            if (!(ok = mbar_wait_warp<false>(&v_full[vp.slot], vp.phase, kErrTimeoutAttnKV, abort_flag))) break;
            const int key0 = k.kv_tile(w, j) * 128, khi = k.keys - key0;
            if (kMask || khi < 128) {
              bool touched = false;
#pragma unroll
              for (int ch = 0; ch < 4; ++ch) {
                const int row = ch * 32 + lane;
                bool keep = row < khi;
                if (kMask && keep) keep = p.key_mask[(size_t)k.s.b * p.k_len + key0 + row] != 0;
                const uint32_t word = __ballot_sync(0xffffffffu, keep);
                if (kMask && lane == 0) s_words[vp.slot * 4 + ch] = word;
                if (word == 0xffffffffu) continue;
                touched = true;
                if (!keep) {
                  // a lane's row, its pieces in an order that keeps the lanes on different banks
                  uint8_t* at = sV + vp.slot * C::kTile + row * 128;
#pragma unroll
                  for (int x = 0; x < 8 * C::kHalves; ++x)
                    *reinterpret_cast<uint4*>(at + (x >> 3) * kHalfBytes + (((x + lane) & 7) << 4)) =
                        make_uint4(0u, 0u, 0u, 0u);
                }
              }
              if (touched) fence_proxy_async_smem();
              __syncwarp();
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
    VPos vp;                            // V slot of the current unit (its mask words)
    uint32_t mine = 0, seq = 0;         // this tile's steps so far; sequence position of the segment
    uint32_t meets = 0;
    bool ok = true;
    while (ok && k.next(p, g)) {
      int n0, g0;
      tile_origin(k, g, w, n0, g0);
      const int rn = row / g.gt, n = n0 + rn, head = g0 + row - rn * g.gt;
      const bool valid = rn < g.nt && n < p.q_len && head < g.group;
      const bool warp_active = __any_sync(0xffffffffu, valid);
      float ref = 0.f, l = 0.f;
      bool have = false;  // the reference is set
      const int all_steps = k.j1 - k.j0, steps1 = k.uses(1, k.j1 - 1) ? all_steps : all_steps - 1;
      const int steps = w ? steps1 : all_steps;
      VPos vs = k.lone ? vp.plus(w) : vp;
      for (int t = 0; t < steps; ++t, ++mine) {
        const StepBuf<NB> b(w, mine, seq + 2 * t + w);
        const uint32_t sAddr = tmem + lane_off + b.buf * 128;
        uint32_t words[4];
        if constexpr (kMask) {
          if (!mbar_wait_warp<false>(&v_ready[vs.slot], vs.phase, kErrTimeoutAttnKV, abort_flag)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) words[ch] = s_words[vs.slot * 4 + ch];
          vs = vs.plus(k.lone ? 2 : 1);
        } else {
          const int khi = k.keys - k.kv_tile(w, k.j0 + t) * 128;
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) words[ch] = len_word(khi, ch);
        }
        uint32_t all = 0xffffffffu, any = 0u;
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) all &= words[ch], any |= words[ch];
        if (!mbar_wait_warp<false>(&s_full[b.buf], b.parity, kErrTimeoutAttnS, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_active) {
          uint32_t pk[64];
          if (any) {
            if (!have) {
              int ch = 0;
#pragma unroll
              for (int i = 3; i > 0; --i)
                if (!words[0] && words[i]) ch = i;
              uint32_t first = words[0];
#pragma unroll
              for (int i = 1; i < 4; ++i)
                if (i == ch) first = words[i];
              uint32_t r[32];
              tmem_ld32(sAddr + ch * 32, r);
              tmem_ld_wait(r);
              // -inf where these scores are: no reference yet, and sums against it are not finite,
              // which sends every step through the exact passes until one finds a score
              ref = chunk_max(r, first, c) - kRefShift<T>;
              have = true;
            }
            float sum = all == 0xffffffffu ? row_exp<T, true>(sAddr, words, c, ref, pk)
                                           : row_exp<T, false>(sAddr, words, c, ref, pk);
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
      if constexpr (kMask) {
        // past the V slots of the segment
        for (int i = k.lone ? all_steps + steps1 : all_steps; i > 0;) {
          const int m = min(i, C::kVSlots);
          vp = vp.plus(m);
          i -= m;
        }
      }
      if (!mbar_wait_warp<false>(&o_done[w], k.seg & 1, kErrTimeoutAttnO, abort_flag)) break;
      tc_fence_after();
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
      const bool whole = k.whole();
      const float inv = whole ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
      const float f0 = a0 * inv, f1 = a1 * inv;
      if (warp_active) {
        T* out = static_cast<T*>(p.out.data) + (long long)k.s.b * p.out.batch_stride +
                 (long long)n * p.out.seq_stride + (long long)(k.s.hk * g.group + head) * p.out.head_stride;
        // partial results go column by column, so that a warp's stores are contiguous
        float* po = p.ws + (size_t)(2 * blockIdx.x + (k.seg > 0)) * g.slot_rows * part_ld(p.head_dim) +
                    (k.lone ? 0 : w * 128) + row;
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
              if (whole) {
                *reinterpret_cast<uint4*>(out + c0 + 8 * u) =
                    make_uint4(pack2<T>(v[8 * u], v[8 * u + 1]), pack2<T>(v[8 * u + 2], v[8 * u + 3]),
                               pack2<T>(v[8 * u + 4], v[8 * u + 5]), pack2<T>(v[8 * u + 6], v[8 * u + 7]));
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) po[(c0 + 8 * u + i) * 256] = v[8 * u + i];
              }
            }
          }
        }
        if (!whole && valid && (!k.lone || w == 0)) {
          po[p.head_dim * 256] = ref;
          po[(p.head_dim + 1) * 256] = l;
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

// Joins the partial results of the items that span CTAs, in CTA order.
//
// kByItem false (at least as many items as CTAs, so a cut item has two or three parts): block
// x takes the item that the boundary between CTAs x and x + 1 cuts, if it is that item's
// first cut.  kByItem true (an item may span every CTA): block x takes item x.
// Slots of 256 rows (column by column): block (x, y, z) joins columns [8 z, 8 z + 8), a lane a
// row; kShare = 1: 8 warps take 32 rows each, kShare > 1 (items of many parts): the warps share
// the parts of rows [32 y, 32 y + 32) out.  Slots of 16 rows (row by row, cross_token.cu): block (x, y) joins row y,
// 4 columns a lane, its kShare = 8 warps sharing the parts out.
// Bound: latency.  7 to 22 us alone; its start overlaps the end of the first launch.
template <typename T, bool kByItem, bool kToken, int kShare>
__global__ void __launch_bounds__(kShare > 1 ? 32 * kShare : 256)
    cross_combine_kernel(const __grid_constant__ CrossAttnParams p, const __grid_constant__ Geom g) {
  __shared__ long long s_start, s_units;
  __shared__ Spot s_spot;
  __shared__ int s_c0, s_c1;
  // sums, references and columns of the warps that share an item's parts out
  __shared__ __align__(16) float s_o[kShare][kToken ? 128 : 8 * 32];
  __shared__ float s_m[kShare][32], s_l[kShare][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long G = g.contribs;
  wait_for_previous();
  if (warp == 0) {
    const long long U = total_units(p, g, lane);
    long long start = -1;
    Spot s{};
    if constexpr (kByItem) {
      // the item's first unit: units of the batch entries before, then inside its own
      s.b = blockIdx.x / g.items_batch;
      const int i = blockIdx.x - s.b * g.items_batch;
      long long before = 0;
      if (p.key_lens) {
        for (int b = lane; b < s.b; b += 32) before += batch_units(g, key_tiles(p, g, b));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
      } else {
        before = s.b * batch_units(g, key_tiles(p, g, 0));
      }
      const int tiles = key_tiles(p, g, s.b);
      s.hk = i / (g.full + g.lone);
      s.t = i - s.hk * (g.full + g.lone);
      start = before + batch_units(g, tiles) / g.kv_heads * s.hk + (long long)s.t * tiles;
    } else {
      const long long cut = U * (blockIdx.x + 1) / G;
      if (cut < U) {
        s = find_spot(p, g, cut, lane);
        start = cut - s.j;
        if (s.j == 0 || U * blockIdx.x / G > start) start = -1;  // no cut, or not its first
      }
    }
    if (lane == 0) {
      s_start = start;
      s_units = U;
      s_spot = s;
      s_c0 = s_c1 = 0;
      if (start >= 0) {
        const int tiles = key_tiles(p, g, s.b);
        const long long last = start + (s.t == g.full ? (tiles + 1) >> 1 : tiles) - 1;
        s_c0 = (int)(((start + 1) * G - 1) / U);
        s_c1 = (int)(((last + 1) * G - 1) / U);
      }
    }
  }
  __syncthreads();
  const long long start = s_start, U = s_units;
  const int c0 = s_c0, c1 = s_c1;
  if (c0 == c1) return;  // no cut, or one CTA had it whole
  const Spot s = s_spot;
  const bool lone = s.t == g.full;
  const int d = p.head_dim, ld = part_ld(d);
  // the parts: CTA c's first item is in slot 2c, its last in 2c + 1; without units it has none
  auto part = [&](int c) -> const float* {
    const long long u0 = U * c / G;
    if (u0 == U * (c + 1) / G) return nullptr;
    return p.ws + (size_t)(2 * c + (u0 < start)) * g.slot_rows * (size_t)ld;
  };
  // token and head of a row of the item, and whether it is one
  auto place = [&](int row, int& n, int& head) {
    const int tile = lone ? 2 * g.full : 2 * s.t + (row >> 7), r = row & 127;
    const int gi = tile / g.n_tiles, rn = r / g.gt;
    n = (tile - gi * g.n_tiles) * g.nt + rn;
    head = gi * g.gt + r - rn * g.gt;
    return rn < g.nt && n < p.q_len && head < g.group && !(lone && row >= 128);
  };
  auto target = [&](int n, int head, int col) {
    return static_cast<T*>(p.out.data) + (long long)s.b * p.out.batch_stride + (long long)n * p.out.seq_stride +
           (long long)(s.hk * g.group + head) * p.out.head_stride + col;
  };
  constexpr int kCols = kToken ? 4 : 8;
  const int row = kToken ? blockIdx.y : (kShare > 1 ? blockIdx.y : warp) * 32 + lane;
  const int col = kToken ? lane * 4 : blockIdx.z * 8;
  int n, head;
  const bool valid = place(row, n, head) && col < d;
  float m = -INFINITY, l = 0.f, o[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int c = c0 + (kShare > 1 ? warp : 0); c <= c1; c += kShare) {
    const float* r = part(c);
    if (!r || !valid) continue;
    float pm, pl, x[kCols];
    if constexpr (kToken) {
      r += (size_t)row * ld;
      const float2 ml = *reinterpret_cast<const float2*>(r + d);
      pm = ml.x, pl = ml.y;
      *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(r + col);
    } else {
      pm = r[d * 256 + row];
      pl = r[(d + 1) * 256 + row];
#pragma unroll
      for (int i = 0; i < kCols; ++i) x[i] = r[(col + i) * 256 + row];
    }
    if (pl == 0.f) continue;  // no kept key in that part
    const float mn = fmaxf(m, pm), a = fast_exp2(m - mn), e = fast_exp2(pm - mn);
    l = l * a + pl * e;
    m = mn;
#pragma unroll
    for (int i = 0; i < kCols; ++i) o[i] = o[i] * a + x[i] * e;
  }
  if constexpr (kShare > 1) {
    const int at = kToken ? 0 : lane;  // a warp's rows
    if (!kToken || lane == 0) {
      s_m[warp][at] = m;
      s_l[warp][at] = l;
    }
#pragma unroll
    for (int i = 0; i < kCols; ++i) s_o[warp][kToken ? col + i : i * 32 + lane] = o[i];
    __syncthreads();
    // the first kCols warps (row-by-row slots: the first one) add up
    if (warp >= (kToken ? 1 : kCols)) return;
    m = -INFINITY;
#pragma unroll
    for (int x = 0; x < kShare; ++x) m = fmaxf(m, s_l[x][at] == 0.f ? -INFINITY : s_m[x][at]);
    l = 0.f;
    float sum[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) sum[i] = 0.f;
#pragma unroll
    for (int x = 0; x < kShare; ++x) {
      if (s_l[x][at] == 0.f) continue;
      const float e = fast_exp2(s_m[x][at] - m);
      l += s_l[x][at] * e;
      if constexpr (kToken) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) sum[i] += s_o[x][col + i] * e;
      } else {
        sum[0] += s_o[x][warp * 32 + lane] * e;
      }
    }
    if constexpr (kToken) {
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] = sum[i];
    } else {
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the kCols warps have read the shares
      s_o[0][warp * 32 + lane] = sum[0];
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (warp != 0) return;
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] = s_o[0][i * 32 + lane];
    }
  }
  if (!valid) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* out = target(n, head, col);
  if constexpr (kToken)
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv),
                                                pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv));
}

// No key at all: every row is zero.
template <typename T>
__global__ void cross_zero_kernel(const __grid_constant__ CrossAttnParams p) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int pieces = p.head_dim / 8;
  if (i >= (long long)p.batch * p.q_len * p.q.heads * pieces) return;
  const int c = (int)(i % pieces);
  const long long r = i / pieces;
  const int h = (int)(r % p.q.heads);
  const long long bn = r / p.q.heads;
  const int b = (int)(bn / p.q_len), n = (int)(bn % p.q_len);
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out.data) + b * p.out.batch_stride + n * p.out.seq_stride +
                            h * p.out.head_stride + c * 8) = make_uint4(0u, 0u, 0u, 0u);
}

Geom make_geom(int batch, int q_len, int k_len, int q_heads, int kv_heads, int head_dim, int num_sms) {
  Geom g{};
  g.kv_heads = kv_heads;
  g.group = q_heads / kv_heads;
  g.gt = std::min(g.group, 128);
  g.nt = 128 / g.gt;
  g.g_tiles = (g.group + g.gt - 1) / g.gt;
  g.n_tiles = (q_len + g.nt - 1) / g.nt;
  g.ksteps = (head_dim + 15) / 16;
  if ((long long)g.group * q_len <= kTokenRows) {
    g.full = 1;  // one item a key head
    g.tile_shift = 6;
    g.slot_rows = kTokenRows;
  } else {
    const int tiles = g.g_tiles * g.n_tiles;
    g.full = tiles / 2;
    g.lone = tiles & 1;
    g.tile_shift = 7;
    g.slot_rows = 256;
  }
  g.items_batch = kv_heads * (g.full + g.lone);
  const long long kt = (k_len + (1 << g.tile_shift) - 1) >> g.tile_shift;
  const long long units = (long long)batch * kv_heads * (g.full * kt + g.lone * ((kt + 1) / 2));
  g.contribs = (int)std::min<long long>(num_sms, std::max<long long>(units, 1));
  return g;
}

// Takes fewer CTAs where runs of a few units more than an equal share end with the items, or cut
// them into equal parts; returns whether an item may be cut (for ragged batches, whose units the
// device counts, the runs stay equal).
// An item that is cut in odd places costs both CTAs another start and end, and the joining
// launch: 8 x 8 heads of 100 x 600 x 64, items of 3 units: 148 runs of 1.3 units 19.6 us, 64 of 3 units, whole
// items without a joining launch, 11.6; 5 x 12/4 heads of 77 x 1501 x 80, items of 12: 148 runs of 1.6
// 29.6, 120 of 2 23.5; one token, 32/8 heads of 128, 4096 keys: 148 runs of 3.5 14.5, 128 of 4 11.2.
// At most two units more than an equal share, as a unit of 128-row tiles takes 1.5 to 3 us and a cut
// and its joining 3 to 8.  Such tiles' runs have two units at least for the same reason (items of
// 12, 48 units in all: one 23.3 us, two 20.4; the other way: items of 16, 128 in all, 17.2 and 18.0 to 18.5).
bool align_runs(Geom& g, const CrossAttnParams& p, int num_sms) {
  if (g.contribs <= 1) return false;
  if (p.key_lens) return true;
  const long long kt = (p.k_len + (1 << g.tile_shift) - 1) >> g.tile_shift, kl = (kt + 1) / 2;
  const long long head = g.full * kt + g.lone * kl, units = (long long)p.batch * g.kv_heads * head;
  if ((g.full ? kt : kl) == 1) return false;  // items of one unit
  const long long least = (units + num_sms - 1) / num_sms;
  for (long long r = std::max<long long>(least, g.tile_shift == 7 ? 2 : 1); r * num_sms <= units + 2 * num_sms; ++r) {
    const bool whole = r % head == 0 || (!g.lone && r % kt == 0) || (!g.full && r % kl == 0);
    const bool even = (!g.full || kt % r == 0) && (!g.lone || kl % r == 0);
    if (units % r != 0 || !(whole || even)) continue;
    g.contribs = (int)(units / r);
    return !whole;
  }
  return true;
}

CUtensorMap query_map(const HeadsView& q, const CrossAttnParams& p, const Geom& g, int& batched) {
  // {d, group, seq, key heads, batch} in boxes of 64 x gt x nt; see cross_kv_map on stride 0
  batched = q.batch_stride != 0;
  auto st = [](long long s) { return (uint64_t)(s ? s * 2 : 16); };
  const uint64_t dims[5] = {(uint64_t)p.head_dim, (uint64_t)g.group, (uint64_t)p.q_len, (uint64_t)g.kv_heads,
                            batched ? (uint64_t)p.batch : 1};
  const uint64_t str[4] = {st(q.head_stride), st(q.seq_stride), st(q.head_stride * g.group), st(q.batch_stride)};
  const uint32_t box[5] = {64, (uint32_t)g.gt, (uint32_t)g.nt, 1, 1};
  return make_tensor_map(q.data, 5, dims, str, box);
}

template <typename T>
cudaError_t launch_combine(const CrossAttnParams& p, const Geom& g, cudaStream_t s) {
  const long long items = (long long)p.batch * g.items_batch;
  const bool by_item = items < g.contribs;
  const unsigned x = (unsigned)(by_item ? items : g.contribs - 1);
  LaunchScope scope("cross_combine", 0.0, 0.0, s);
  if (g.slot_rows == kTokenRows) {
    DependentLaunch l(dim3(x, g.group * p.q_len), 256, 0, s);
    return by_item ? cudaLaunchKernelEx(&l.cfg, cross_combine_kernel<T, true, true, 8>, p, g)
                   : cudaLaunchKernelEx(&l.cfg, cross_combine_kernel<T, false, true, 8>, p, g);
  }
  const int rows = g.full ? 256 : g.gt * std::min(g.nt, p.q_len);
  // an item has about contribs / items parts: 32 warps share them where there are many
  const bool share = by_item && g.contribs / items >= 16;
  DependentLaunch l(dim3(x, share ? (rows + 31) / 32 : 1, p.head_dim / 8), share ? 1024 : 256, 0, s);
  return share     ? cudaLaunchKernelEx(&l.cfg, cross_combine_kernel<T, true, false, 32>, p, g)
         : by_item ? cudaLaunchKernelEx(&l.cfg, cross_combine_kernel<T, true, false, 1>, p, g)
                   : cudaLaunchKernelEx(&l.cfg, cross_combine_kernel<T, false, false, 1>, p, g);
}

template <typename T, int DP, bool kMask>
cudaError_t launch_k(const CrossAttnParams& p, Geom g, cudaStream_t s) {
  static std::atomic<unsigned long long> configured;
  cudaError_t e = ensure_smem_limit(cross_attention_kernel<T, DP, kMask>, (int)Cfg<DP>::kSmem, configured);
  if (e != cudaSuccess) return e;
  const CUtensorMap mq = query_map(p.q, p, g, g.q_batched);
  const CUtensorMap mk = cross_kv_map(p.k, p.batch, p.k_len, p.head_dim, 128, g.k_batched, g.k_headed);
  const CUtensorMap mv = cross_kv_map(p.v, p.batch, p.k_len, p.head_dim, 128, g.v_batched, g.v_headed);
  const double rows = (double)p.batch * p.q_len * p.q.heads, keys = (double)p.batch * p.k_len * p.k.heads;
  LaunchScope scope("cross_attention", 4.0 * rows * p.k_len * p.head_dim, 4.0 * (rows + keys) * p.head_dim, s);
  cross_attention_kernel<T, DP, kMask><<<g.contribs, kThreads, Cfg<DP>::kSmem, s>>>(mq, mk, mv, p, g);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const CrossAttnParams& p, int num_sms, cudaStream_t s) {
  if (p.k_len == 0) {
    const long long n = (long long)p.batch * p.q_len * p.q.heads * (p.head_dim / 8);
    LaunchScope scope("cross_zero", 0.0, 16.0 * n, s);
    cross_zero_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p);
    return cudaGetLastError();
  }
  Geom g = make_geom(p.batch, p.q_len, p.k_len, p.q.heads, p.k.heads, p.head_dim, num_sms);
  const bool cut = align_runs(g, p, num_sms);
  cudaError_t e;
  if (g.slot_rows == kTokenRows)
    e = launch_cross_token<T>(p, g, s);
  else if (p.head_dim <= 64)
    e = p.key_mask ? launch_k<T, 64, true>(p, g, s) : launch_k<T, 64, false>(p, g, s);
  else
    e = p.key_mask ? launch_k<T, 128, true>(p, g, s) : launch_k<T, 128, false>(p, g, s);
  if (e != cudaSuccess || !cut) return e;
  return launch_combine<T>(p, g, s);
}

}  // namespace

long long cross_attention_workspace(int batch, int q_len, int k_len, int q_heads, int kv_heads, int head_dim,
                                    int num_sms) {
  if (batch == 0 || q_len == 0 || k_len == 0) return 0;
  const Geom g = make_geom(batch, q_len, k_len, q_heads, kv_heads, head_dim, num_sms);
  return g.contribs > 1 ? 2LL * g.contribs * g.slot_rows * part_ld(head_dim) * 4 : 0;
}

// A dimension walked with stride 0 is left out (extent 1, coordinate 0); a stride that is
// never walked only has to be a legal one.
CUtensorMap cross_kv_map(const HeadsView& v, int batch, int seq, int d, int box_rows, int& batched, int& headed) {
  batched = v.batch_stride != 0;
  headed = v.head_stride != 0;
  auto st = [](long long s) { return (uint64_t)(s ? s * 2 : 16); };
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)seq, headed ? (uint64_t)v.heads : 1, batched ? (uint64_t)batch : 1};
  const uint64_t str[3] = {st(v.seq_stride), st(v.head_stride), st(v.batch_stride)};
  const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
  // What a DRAM read may bring into L2 beside the bytes asked for: no more than a key's row,
  // where the next bytes are another head's, which another CTA reads at another time
  const bool dense = v.seq_stride == d;
  return make_tensor_map(v.data, 4, dims, str, box, CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_128B,
                         dense || d >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                           : (d >= 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                                      : CU_TENSOR_MAP_L2_PROMOTION_L2_64B));
}

cudaError_t launch_cross_attention(const CrossAttnParams& p, int bf16, int num_sms, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, num_sms, stream) : launch_t<__half>(p, num_sms, stream);
}

MSST_DEFINE_ERROR_ACCESSOR(cross_attn_device_error)

}  // namespace msst
