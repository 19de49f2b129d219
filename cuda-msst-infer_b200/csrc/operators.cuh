// operators.cuh — host-visible description of the operators of conditioned blocks:
// per-head norms of queries and keys with the rotation (qk_norm.cu), cross
// attention to an encoder's states (cross_attn.cu) and a shared projection with
// the low-rank adapters of many requests beside it (adapter_gemm.cu).  The
// reference has no counterpart of any of them.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace msst {

// [batch, seq, heads, head_dim] 16-bit, unit stride along head_dim (elements)
struct HeadsView {
  void* data;
  int heads;
  long long batch_stride, seq_stride, head_stride;
};

// y = x * rsqrt(mean(x^2) + eps) * gamma per head vector, then the rotation of its
// first rot_dim columns by the angle of the token's position.
struct QkNormParams {
  HeadsView x[2], out[2];   // q, k; heads = 0 for an absent k
  const float* gamma[2];    // [head_dim] or nullptr (ones)
  float eps;
  int batch, seq, head_dim, rot_dim;
  int halves;               // pairing: 0 = (2i, 2i + 1), 1 = (i, i + rot_dim / 2)
  const float* cos_tab;     // [num_pos, rot_dim / 2]
  const float* sin_tab;
  int num_pos;
  const int* positions;     // [batch, seq] or nullptr (the index in the sequence)
};
cudaError_t launch_qk_norm(const QkNormParams& p, int bf16, cudaStream_t stream);
// The group of heads that a thread of the 8-column kernel works on: blocks of 128 threads, lpv (a
// divisor of 128) threads a group.  Dividing first keeps the index in 32 bits for as many groups as
// 32 bits count; the number of threads before a block may pass 2^32.
__host__ __device__ __forceinline__ unsigned qk_norm_item(unsigned block, unsigned thread, unsigned lpv) {
  return block * (128u / lpv) + thread / lpv;
}

struct CrossAttnParams {
  HeadsView q, k, v, out;
  int batch, q_len, k_len, head_dim;
  float scale_log2;                 // softmax scale * log2(e)
  const int* key_lens;              // [batch] or nullptr
  const unsigned char* key_mask;    // [batch, k_len], nonzero = kept, or nullptr
  float* ws;                        // cross_attention_workspace() bytes
};
long long cross_attention_workspace(int batch, int q_len, int k_len, int q_heads, int kv_heads, int head_dim,
                                    int num_sms);
cudaError_t launch_cross_attention(const CrossAttnParams& p, int bf16, int num_sms, cudaStream_t stream);

struct AdapterGemmParams {
  const void* x;             // [rows, K], row stride ldx
  const void* w;             // [N, K]
  const float* bias;         // [N] or nullptr
  const void* lora_a;        // [adapters, rank, K]
  const void* lora_b;        // [adapters, N, rank]
  const float* scales;       // [adapters] or nullptr (ones)
  const int* row_adapter;    // [rows], outside [0, adapters) = none
  void* out;                 // [rows, N], row stride ldo
  void* ws;                  // adapter_gemm_workspace() bytes
  long long ldx, ldo;
  int rows, K, N, adapters, rank;
};
long long adapter_gemm_workspace(int rows, int K, int N, int adapters, int rank, int num_sms);
cudaError_t launch_adapter_gemm(const AdapterGemmParams& p, int bf16, int num_sms, cudaStream_t stream);

}  // namespace msst
