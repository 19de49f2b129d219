// attn_steps.cuh — what the attention kernels over K/V tiles share: ring positions, the softmax of a
// 128-row tile's step from TMEM (tcgen05 path) and the fragments of up to 16 rows (mma.sync path).
#pragma once

#include "common.cuh"

namespace msst {

// ---------------------------------------------------------------- 128-row tiles
// fp16 weights are taken 2^4 larger (the reference 4 lower, in powers of two), since fp16 drops what is
// below 2^-25 while the row sum counts it: 2^18 such keys were 0.8 % of a result.  A step's row sum bounds
// each of its weights, and 61440 is inside fp16's 65504, so a row may grow as far as without the shift.
template <typename T>
constexpr float kRefShift = std::is_same<T, __half>::value ? 4.f : 0.f;
template <typename T>
constexpr float kSumLimit = std::is_same<T, __half>::value ? 61440.f : 4096.f;

// A position in a ring of N slots: the slot and the parity of its current use.
template <int N>
struct RingPos {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ RingPos plus(uint32_t n) const {  // n <= N
    RingPos r;
    r.slot = slot + n >= N ? slot + n - N : slot + n;
    r.phase = slot + n >= N ? phase ^ 1 : phase;
    return r;
  }
};

// The S buffer of a step and the parity of that use.  Two buffers: one a tile, by the
// tile's own count of steps; three: in turn over the sequence of both tiles.
template <int NB>
struct StepBuf {
  uint32_t buf, parity;
  __device__ __forceinline__ StepBuf(int w, uint32_t mine, uint32_t seq) {
    if constexpr (NB == 2) {
      buf = (uint32_t)w;
      parity = mine & 1;
    } else {
      const uint32_t q = seq / 3;
      buf = seq - 3 * q;
      parity = q & 1;
    }
  }
};

// Kept keys among the 32 of chunk ch of a tile that has khi valid keys.
__device__ __forceinline__ uint32_t len_word(int khi, int ch) {
  const int n = khi - 32 * ch;
  return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
}

// Maximum of s c over the kept scores of a chunk.
__device__ __forceinline__ float chunk_max(const uint32_t (&r)[32], uint32_t word, float c) {
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    if (word >> i & 1) m0 = fmaxf(m0, __uint_as_float(r[i]) * c);
    if (word >> (i + 1) & 1) m1 = fmaxf(m1, __uint_as_float(r[i + 1]) * c);
  }
  return fmaxf(m0, m1);
}

// P of one 32-column chunk against the reference: 2^(s c - ref), packed into pk.  P is rounded to the operands' 16 bits:
// the product with V has operands of one type on the tensor core, and an fp32 one would run at a fraction of its rate.
// Each weight is off by half a step at most, the row sum is taken of the unrounded ones in fp32; a result's error
// against 64 bits grows 1.2 to 1.4 times by it.
template <typename T>
__device__ __forceinline__ void chunk_exp(const uint32_t (&r)[32], uint32_t word, float2 c2, float2 nref2, float2& sum2,
                                          uint32_t* pk) {
  if (word == 0xffffffffu) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 a = __ffma2_rn(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), c2, nref2);
      const float2 e = make_float2(fast_exp2(a.x), fast_exp2(a.y));
      sum2 = __fadd2_rn(sum2, e);
      pk[i] = pack2<T>(e.x, e.y);
    }
  } else if (word == 0u) {
#pragma unroll
    for (int i = 0; i < 16; ++i) pk[i] = 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 a = __ffma2_rn(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), c2, nref2);
      const float e0 = word >> (2 * i) & 1 ? fast_exp2(a.x) : 0.f;
      const float e1 = word >> (2 * i + 1) & 1 ? fast_exp2(a.y) : 0.f;
      sum2 = __fadd2_rn(sum2, make_float2(e0, e1));
      pk[i] = pack2<T>(e0, e1);
    }
  }
}

// P and the row sum of a step's 128 columns; the next chunk's load is in flight while
// one is processed.  kAll: every key is kept.
template <typename T, bool kAll>
__device__ __forceinline__ float row_exp(uint32_t sAddr, const uint32_t (&words)[4], float c, float ref,
                                         uint32_t (&pk)[64]) {
  const float2 c2 = make_float2(c, c), nref2 = make_float2(-ref, -ref);
  float2 sum2 = make_float2(0.f, 0.f);
  uint32_t ra[32], rb[32];
  tmem_ld32(sAddr, ra);
  tmem_ld_wait(ra);
  tmem_ld32(sAddr + 32, rb);
  chunk_exp<T>(ra, kAll ? 0xffffffffu : words[0], c2, nref2, sum2, pk);
  tmem_ld_wait(rb);
  tmem_ld32(sAddr + 64, ra);
  chunk_exp<T>(rb, kAll ? 0xffffffffu : words[1], c2, nref2, sum2, pk + 16);
  tmem_ld_wait(ra);
  tmem_ld32(sAddr + 96, rb);
  chunk_exp<T>(ra, kAll ? 0xffffffffu : words[2], c2, nref2, sum2, pk + 32);
  tmem_ld_wait(rb);
  chunk_exp<T>(rb, kAll ? 0xffffffffu : words[3], c2, nref2, sum2, pk + 48);
  return sum2.x + sum2.y;
}

// ---------------------------------------------------------------- up to 16 rows
// fp16 weights reach up to 2^15 instead of 1 (the reference is the maximum), so that they are dropped
// below 2^-40 of the largest and not below 2^-25: a long row can hold many of those.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.f : 0.f;


template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

}  // namespace msst
