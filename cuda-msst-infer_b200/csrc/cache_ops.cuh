// cache_ops.cuh — host-visible description of the operators of a cache of generated
// tokens behind one shared prefix: block tables and slots from request lengths
// (cache_plan.cu), rotated keys and values written to the cache's pages
// (rope_append.cu) and attention to the prefix and each request's own pages
// (prefix_attn.cu).  The reference has no counterpart of any of them.
#pragma once

#include <cuda_runtime.h>

#include "operators.cuh"

namespace msst {

// Requests of a plan: four numbers each are kept in shared memory.
constexpr int kMostPlanRequests = 8192;

struct CachePlanParams {
  const int* new_tokens;  // [requests], negative: the request has ended
  const int* lens;        // [requests]
  int* table;             // [requests, blocks], row stride table_stride
  int* free_pages;        // [pages], a stack
  const int* free_count;  // its height
  int* out_lens;          // may be lens
  int* out_count;         // may be free_count
  int* q_starts;          // [requests + 1]
  int* slots;             // [tokens]
  int* positions;         // [tokens]
  long long table_stride;
  int requests, blocks, pages, page_shift, start, tokens;
};
cudaError_t launch_cache_plan(const CachePlanParams& p, cudaStream_t stream);

struct RopeAppendParams {
  HeadsView q, k, v, out_q;     // batch 1, seq = tokens
  HeadsView k_cache, v_cache;   // batch = pages, seq = page
  const int* positions;         // [tokens]
  const int* slots;             // [tokens], negative: not written
  const double* freq;           // [rot_dim / 2] radians a position
  float amplitude;
  int tokens, head_dim, rot_dim, halves, page_shift;
  long long num_slots;
};
cudaError_t launch_rope_append(const RopeAppendParams& p, int bf16, cudaStream_t stream);

struct PrefixAttnParams {
  HeadsView q, out;             // batch 1, seq = tokens
  HeadsView prefix_k, prefix_v; // batch 1, seq = prefix
  HeadsView k_cache, v_cache;   // batch = pages, seq = page
  const int* q_starts;          // [requests + 1] or nullptr (one token each)
  const int* lens;              // [requests] own tokens, the new ones included
  const int* table;             // [requests, blocks], row stride table_stride
  long long table_stride;
  int tokens, requests, prefix, pages, page_shift, blocks, head_dim;
  int zero_rest;                // rows of no request: 0 left as they were, 1 zeroed
  float scale_log2;             // softmax scale * log2(e)
  float* ws;                    // prefix_attention_workspace() bytes
};
long long prefix_attention_workspace(int tokens, int requests, int prefix, int q_heads, int kv_heads, int head_dim,
                                     int num_sms);
cudaError_t launch_prefix_attention(const PrefixAttnParams& p, int bf16, int num_sms, cudaStream_t stream);

}  // namespace msst
