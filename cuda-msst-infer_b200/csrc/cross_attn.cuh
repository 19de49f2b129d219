// cross_attn.cuh — how the cross-attention kernels cut their work: items (row tiles of one key
// head), units (K/V tiles of an item) and equal contiguous runs of units per CTA.
#pragma once

#include "common.cuh"
#include "operators.cuh"

namespace msst {

// Geometry of a launch.
struct Geom {
  int kv_heads, group;       // G query heads a key head
  int gt, nt;                // heads and tokens of a tile
  int g_tiles, n_tiles;      // tiles along heads and tokens
  int full, lone;            // per key head: pairs, and 1 if a lone tile is left
  int q_batched;             // 0: shared by the batch through stride 0
  int k_batched, k_headed;
  int v_batched, v_headed;
  int ksteps;                // ceil(head_dim / 16)
  int contribs;              // CTAs of the attention launch
  int tile_shift;            // log2 of the keys of a K/V tile
  int slot_rows;             // rows of a partial result's slot
  int items_batch;           // items of a batch entry
};

__device__ __forceinline__ int key_count(const CrossAttnParams& p, int b) {
  return p.key_lens ? min(max(__ldg(p.key_lens + b), 0), p.k_len) : p.k_len;
}
// K/V tiles of a batch entry (one masked tile where no key is left, so that every item
// has a unit that writes its rows)
__device__ __forceinline__ int key_tiles(const CrossAttnParams& p, const Geom& g, int b) {
  return max(1, (key_count(p, b) + (1 << g.tile_shift) - 1) >> g.tile_shift);
}
__device__ __forceinline__ long long batch_units(const Geom& g, int tiles) {
  return (long long)g.kv_heads * ((long long)g.full * tiles + g.lone * ((tiles + 1) >> 1));
}

// A position in the list of units: batch entry, key head, item of the key head, unit.
struct Spot {
  int b, hk, t, j;
};
// Spot of unit u < batch_units(tiles of b), counted from batch entry b's first.
__device__ __forceinline__ Spot spot_in_batch(const Geom& g, int b, int tiles, long long u) {
  const long long per_head = batch_units(g, tiles) / g.kv_heads;
  Spot s;
  s.b = b;
  s.hk = (int)(u / per_head);
  const long long r = u - s.hk * per_head;
  if (r < (long long)g.full * tiles) {
    s.t = (int)(r / tiles);
    s.j = (int)(r - (long long)s.t * tiles);
  } else {
    s.t = g.full;
    s.j = (int)(r - (long long)g.full * tiles);
  }
  return s;
}

// One warp: total units of the launch (ragged batches summed 32 entries at a time).
__device__ inline long long total_units(const CrossAttnParams& p, const Geom& g, int lane) {
  if (!p.key_lens) return p.batch * batch_units(g, key_tiles(p, g, 0));
  long long sum = 0;
  for (int b = lane; b < p.batch; b += 32) sum += batch_units(g, key_tiles(p, g, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// One warp: the spot of unit u and the units before its batch entry.
__device__ inline Spot find_spot(const CrossAttnParams& p, const Geom& g, long long u, int lane) {
  if (!p.key_lens) {
    const int tiles = key_tiles(p, g, 0);
    const long long per = batch_units(g, tiles);
    const int b = (int)(u / per);
    return spot_in_batch(g, b, tiles, u - b * per);
  }
  long long before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int tiles = b < p.batch ? key_tiles(p, g, b) : 0;
    const long long mine = b < p.batch ? batch_units(g, tiles) : 0;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const long long start = before + __shfl_sync(0xffffffffu, incl - mine, src);
      return spot_in_batch(g, b0 + src, __shfl_sync(0xffffffffu, tiles, src), u - start);
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return Spot{p.batch - 1, 0, 0, 0};  // u past the end: not reached
}

// Walks the segments (one item each) of a CTA's run.
struct Walk {
  Spot s;
  long long left;
  int seg;
  // of the current segment: K/V tiles of the batch entry, its key count, units [j0, j1)
  int tiles, keys, j0, j1, units;
  bool lone;
  __device__ Walk(const Spot& s0, long long n) : s(s0), left(n), seg(-1) {}
  __device__ __forceinline__ bool next(const CrossAttnParams& p, const Geom& g) {
    if (seg >= 0) {
      s.j = 0;
      if (++s.t == g.full + g.lone) {
        s.t = 0;
        if (++s.hk == g.kv_heads) {
          s.hk = 0;
          ++s.b;
        }
      }
    }
    if (left <= 0) return false;
    ++seg;
    keys = key_count(p, s.b);
    tiles = max(1, (keys + (1 << g.tile_shift) - 1) >> g.tile_shift);
    lone = s.t == g.full;
    units = lone ? (tiles + 1) >> 1 : tiles;
    j0 = s.j;
    j1 = (int)min((long long)units, j0 + left);
    left -= j1 - j0;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == units; }
  // K/V tile of query tile w in unit j, and whether it has one
  __device__ __forceinline__ int kv_tile(int w, int j) const { return lone ? 2 * j + w : j; }
  __device__ __forceinline__ bool uses(int w, int j) const { return kv_tile(w, j) < tiles; }
};


// Partial results of the items that span CTAs: CTA c's first item in slot 2c, its last in
// slot 2c + 1, each slot_rows rows of head_dim values of O, the reference (log2) and the
// sum: row by row, head_dim + 4 floats apart, for 16 rows; column by column for 256.
__host__ __device__ inline int part_ld(int head_dim) { return head_dim + 4; }

// cross_token.cu: up to 16 query rows a key head.
constexpr int kTokenRows = 16;
template <typename T>
cudaError_t launch_cross_token(const CrossAttnParams& p, Geom g, cudaStream_t s);

// cross_attn.cu: a tensor map over k or v in boxes of 64 columns x box_rows keys.
CUtensorMap cross_kv_map(const HeadsView& v, int batch, int seq, int d, int box_rows, int& batched, int& headed);

}  // namespace msst
