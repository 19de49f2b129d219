/*
 * msst_b200.h — C ABI of libmsst_b200, a B200-native (sm_100a) implementation of
 * the Roformer transformer stack of HuanLinOTO/CUDA-MSST-Infer
 * (MelBandRoformer and BS-Roformer: band split, axial time/band transformers,
 * mask estimators, mask merge).
 *
 * Conventions (all entry points):
 *   - plain pointers and sizes, no C++ types; device pointers unless named *_host
 *   - `stream` is a cudaStream_t passed as void* (NULL = legacy default stream)
 *   - return MSST_OK (0) or an MSST_ERR_* code; msst_last_error() gives the
 *     message of the calling thread's last failure.  The reference throws
 *     std::runtime_error for the same conditions (src/tensor.h:28-34); its C++
 *     call sites get that behaviour back from a thin wrapper that throws on a
 *     non-zero status.
 *   - 16-bit operands are fp16 (MSST_F16) or bf16 (MSST_BF16); accumulation is
 *     fp32; the residual stream and all model inputs/outputs are fp32.
 *   - K (the reduction length) of every GEMM is a multiple of 64; hidden sizes
 *     of the Roformer (dim, heads*64, 4*dim) satisfy this, band inputs are padded.
 *   - head_dim is 64 on the Roformer path; msst_sdpa takes head_dim <= 64.
 *   - devices: a msst_model runs on the GPU it was loaded on; its device buffers
 *     must live on that GPU (or be managed memory), anything else is refused with
 *     MSST_ERR_INVALID before a kernel runs.  Op-level calls run on the GPU of
 *     their first operand.  Every call leaves the calling thread's current device
 *     as it found it.
 */
#ifndef MSST_B200_H
#define MSST_B200_H

#ifdef __cplusplus
extern "C" {
#endif

#define MSST_OK 0
#define MSST_ERR_INVALID 1     /* bad argument or unsupported shape            */
#define MSST_ERR_CUDA 2        /* CUDA runtime / cuFFT / driver error          */
#define MSST_ERR_IO 3          /* cannot read or parse a .csm file             */
#define MSST_ERR_UNSUPPORTED 4 /* model feature outside this implementation    */
#define MSST_ERR_DEVICE 5      /* a kernel's bounded wait gave up (see msst_device_error) */

#define MSST_F16 0
#define MSST_BF16 1
#define MSST_F32 2 /* output type of msst_layernorm only */

/* GEMM epilogues */
#define MSST_EPI_STORE16 0 /* out16 = act(x W^T + b)                               */
#define MSST_EPI_RESID32 1 /* out32 += x W^T + b   (residual add)                  */
#define MSST_EPI_STORE32 2 /* out32  = x W^T + b                                   */
#define MSST_EPI_GLU32 3   /* out32[j] = y[2j] * sigmoid(y[2j+1]), y = x W^T + b    */

#define MSST_ACT_NONE 0
#define MSST_ACT_GELU 1    /* erf form, src/ops_fused.cu:21-24 */
#define MSST_ACT_TANH 2
#define MSST_ACT_SIGMOID 3

#define MSST_AXIS_TIME 0
#define MSST_AXIS_BAND 1

/* msst_model_separate flags */
#define MSST_SEPARATE_FIX_TAIL_PADDING 1 /* pad the final short chunk from each channel's own
                                            samples instead of reproducing the reference's
                                            contiguous-source read (src/tensor.cu:377-405) */

typedef struct msst_model msst_model;

typedef struct msst_model_info {
  int model_type; /* 1 MelBandRoformer, 2 BSRoformer (app::ModelType order) */
  int dim, depth, heads, dim_head, num_bands, num_stems, channels;
  int n_fft, hop_length, sample_rate, chunk_size, num_overlap;
  int sum_band_dims; /* width of one mask row, sum over bands of 2*channels*freqs */
  int precision;     /* MSST_F16 or MSST_BF16 */
  /* config switches of the reference drivers (MBRConfig / BSRConfig::from_json) */
  int stft_normalized, skip_connection, match_input_audio_length;
  int bands_from_file; /* MelBandRoformer: 1 = __precomputed__ band tables of the .csm,
                          0 = computed at load (the reference's mel fallback) */
  float load_ms;       /* wall time of msst_model_load (read, convert, upload) */
} msst_model_info;

const char* msst_last_error(void);
/* Code recorded by kernels since the last reset, 0 = none: 1 to 13 where a bounded wait gave up
 * (results since then are garbage), 14 where a position, 15 where an adapter index, 17 where a
 * slot and 18 where a page lay outside the range that its operator documents, 16 where a cache had
 * no room for a request's tokens.  A wait comes before the others; where several are
 * recorded, clear != 0 resets the returned one (of the waits, all) and the next call gives the next. */
unsigned msst_device_error(int clear);
int msst_version(void);
/* Number of kernels this library has launched (process-wide); reset != 0 returns and zeroes it. */
unsigned long long msst_kernel_launches(int reset);

/* Per-kernel timing of this library's launches, a measurement aid with no
 * counterpart in the reference.  msst_kernel_timing(1) discards earlier records
 * and starts recording: each launch is bracketed by two CUDA events on its stream
 * and tagged with its kernel name and its algorithmic FLOPs and DRAM bytes (the
 * operands read once and the results written once).  msst_kernel_timing(0) stops
 * recording.  msst_kernel_timing_report waits for the recorded launches, writes up
 * to `cap` per-name aggregates to `out` and the number of names to *count. */
typedef struct msst_kernel_stat {
  char name[40];
  unsigned long long launches;
  double total_ms;
  double flop;
  double bytes;
} msst_kernel_stat;
int msst_kernel_timing(int enable);
int msst_kernel_timing_report(msst_kernel_stat* out, int cap, int* count);

/* ---------------------------------------------------------------- op level -- */

/* RMSNorm of the reference, y = x * rsqrt(sum(x^2) + 1e-12) * gamma * scale
 * (replaces ops::rms_norm, src/ops_norm.cu:455-491).  x fp32 [rows, D]
 * (D % 128 == 0, D <= 1024) -> out16 [rows, D].  If wg != NULL also writes
 * gates[rows, heads] = sigmoid(y wg^T + bg) (the attention gate projection,
 * ops::linear_sigmoid at src/model_mel_band_roformer.cu:575). */
int msst_rmsnorm(const float* x, long long rows, int D, const float* gamma, float scale, int dtype, void* out16,
                 const float* wg, const float* bg, int heads, float* gates, void* stream);

/* out = epilogue(x W^T + b): x 16-bit [rows, K] (row stride ldx elements),
 * W 16-bit [N, K], bias fp32 [N] or NULL.  out is 16-bit for MSST_EPI_STORE16,
 * fp32 otherwise, row stride ldo.  Replaces ops::linear / linear_no_bias /
 * linear_gelu / linear_sigmoid (src/ops_linear.cu:150,349, src/ops_fused.cu:264,285)
 * and the residual Tensor::add_ (src/tensor.cu:1439). */
int msst_gemm(const void* x, long long rows, int K, long long ldx, const void* w, int N, const float* bias,
              int epilogue, int act, int dtype, void* out, long long ldo, void* stream);

/* QKV projection with the rotary embedding fused into the epilogue: qkv16
 * [rows, 3*heads*64] = x W^T with interleaved-pair rotation of the q and k
 * columns at position (row / pos_div) % pos_mod, tables cos/sin [pos_mod, 32]
 * (replaces linear_no_bias + split_qkv_heads + apply_rotary_emb,
 * src/model_mel_band_roformer.cu:540-559, src/ops_misc.cu:39-131). */
int msst_gemm_qkv_rope(const void* x, long long rows, int K, const void* w, int heads, const float* cos_tab,
                       const float* sin_tab, int pos_div, int pos_mod, int dtype, void* qkv16, void* stream);

/* Axial attention over a fused QKV buffer [B*T*F tokens, 3*heads*64] in
 * [B, T, F] token order: axis MSST_AXIS_TIME attends over t for every (b, f),
 * MSST_AXIS_BAND over f for every (b, t).  softmax(scale * q k^T) v, multiplied by
 * gates[token, head] when gates != NULL, heads merged: out16 [tokens, heads*64].
 * Replaces ops::scaled_dot_product_attention (src/ops_attention.cu:522-599) and
 * apply_gates_and_merge_heads (src/model_mel_band_roformer.cu:94-163). */
int msst_attention(const void* qkv16, int B, int T, int F, int heads, int axis, float scale, const float* gates,
                   int dtype, void* out16, void* stream);

/* ---- ops the reference shares with its conv model (HTDemucs' transformer,
 * src/model_htdemucs.cu:542-659); its linear and linear_gelu calls map to msst_gemm. */

/* LayerNorm over the last dimension, y = (x - mean) * rsqrt(var + eps) * gamma + beta
 * with the biased variance (replaces ops::layer_norm, src/ops_norm.cu:496-533;
 * the reference's default eps is 1e-5).  x fp32 [rows, D], D % 4 == 0 and
 * D <= 1024; out [rows, D] as out_dtype MSST_F32, MSST_F16 or MSST_BF16. */
int msst_layernorm(const float* x, long long rows, int D, const float* gamma, const float* beta, float eps,
                   int out_dtype, void* out, void* stream);

/* out = softmax(scale * q k^T) v per (batch, head), non-causal: q [B, H, Nq, d],
 * k and v [B, H, Nk, d], out [B, H, Nq, d], all 16-bit (dtype), d a multiple of 8
 * and <= 64; scale 0 selects 1/sqrt(d) (replaces ops::scaled_dot_product_attention,
 * src/ops_attention.cu:522-599, including its cross-attention form Nq != Nk). */
int msst_sdpa(const void* q, const void* k, const void* v, int B, int H, int Nq, int Nk, int head_dim, float scale,
              int dtype, void* out, void* stream);

/* ---- operators of conditioned blocks: a block that attends to an encoder's states
 * and serves the fine-tunes of many requests from one set of weights.  The
 * reference has no counterpart of them. */

/* A 16-bit tensor [batch, sequence, heads, head_dim] in any order of its first three
 * dimensions: element (b, n, h, i) at data + b*batch_stride + n*seq_stride +
 * h*head_stride + i, strides in elements and >= 0 (of a tensor that is written, above 0
 * wherever the extent is above 1).  Batch, sequence and head_dim
 * are arguments of the call. */
typedef struct msst_heads {
  void* data;
  int heads;
  long long batch_stride, seq_stride, head_stride;
} msst_heads;

#define MSST_PAIRS_INTERLEAVED 0 /* pairs (2i, 2i + 1), as msst_gemm_qkv_rope         */
#define MSST_PAIRS_HALVES 1      /* pairs (i, i + rot_dim / 2)                        */

/* Norms of queries and keys for each head with the position rotation in the same
 * pass: every head vector x of q and k becomes
 *   y = x * rsqrt(mean(x^2) + eps) * gamma
 * and each pair (a, b) of y's first rot_dim columns (a cos - b sin, b cos + a sin),
 * cos and sin from row positions[b*seq + n] (row n when positions is NULL) of the
 * tables [num_pos, rot_dim / 2]; fp32 inside, one rounding at the end.  k may be
 * NULL; gammas fp32 [head_dim] or NULL (ones).  head_dim is even and <= 256,
 * rot_dim even and <= head_dim (0: no rotation, tables may be NULL).  q_out / k_out
 * may be q / k themselves (same strides), and otherwise must not overlap them.
 * A token whose position lies outside the tables is normed but not rotated, and
 * msst_device_error reports it. */
int msst_qk_norm_rope(const msst_heads* q, const msst_heads* k, int batch, int seq, int head_dim,
                      const float* q_gamma, const float* k_gamma, float eps, const float* cos_tab,
                      const float* sin_tab, int num_pos, int rot_dim, const int* positions, int pairing, int dtype,
                      const msst_heads* q_out, const msst_heads* k_out, void* stream);

/* Cross attention to an encoder's states: out = softmax(scale * q k^T) v over the
 * keys that are kept, q and out [batch, q_len, q.heads, head_dim], k and v [batch,
 * k_len, k.heads, head_dim], q.heads a multiple of k.heads (query head h reads
 * key head h / (q.heads / k.heads)).  head_dim is a multiple of 8 and <= 128, scale 0
 * selects 1/sqrt(head_dim).  Kept are the first key_lens[b] keys (int32, taken into
 * [0, k_len]; NULL: all k_len) whose key_mask[b*k_len + j] is nonzero (NULL: all).
 * What the others hold, infinities and NaN included, has no influence.  A row
 * without a kept key gives zeros.  Scores, sums and products are fp32; the softmax's
 * weights are rounded to the operands' type before the product with v (fp16: to within
 * 2^-29 of the largest where they are subnormal), the result once.  Data pointers are 16-byte aligned and strides
 * multiples of 8 elements; batch and head strides of k and v may be 0 (states shared
 * by the whole batch).  `workspace` holds at least the bytes that
 * msst_cross_attention_workspace gives for the call's sizes with the operands' GPU
 * current (16-byte aligned; may be NULL when that is 0); calls that may overlap need workspaces of their own. */
int msst_cross_attention_workspace(int batch, int q_len, int k_len, int q_heads, int kv_heads, int head_dim,
                                   long long* bytes);
int msst_cross_attention(const msst_heads* q, const msst_heads* k, const msst_heads* v, int batch, int q_len, int k_len,
                         int head_dim, float scale, const int* key_lens, const unsigned char* key_mask, int dtype,
                         const msst_heads* out, void* workspace, long long workspace_bytes, void* stream);

/* A shared projection with the low-rank adapters of many requests beside it:
 *   out16[t] = W x[t] + bias + scales[a] * B_a (A_a x[t]),   a = row_adapter[t],
 * without the last term where a is -1.  x 16-bit [rows, K] (row stride ldx), W 16-bit
 * [N, K], bias fp32 [N] or NULL, lora_a 16-bit [adapters, rank, K] (the A_a), lora_b
 * 16-bit [adapters, N, rank] (the B_a), scales fp32 [adapters] or NULL (ones),
 * row_adapter int32 [rows], out row stride ldo.  K, N, rank, ldx and ldo are
 * multiples of 8, rank <= 256, and all pointers but scales and row_adapter 16-byte
 * aligned; rows of one request need not be adjacent.  An index
 * outside [-1, adapters) counts as -1, and msst_device_error reports it.  A row's
 * result does not depend on the other rows of the call beyond the order of sums.
 * Sums are fp32; scales[a] A_a x is rounded once to the operands' type (fp16: to within
 * 2^-25 where it is subnormal; what lies beyond +-65504 is kept in fp32, at a lower
 * speed), the result once.
 * `workspace` as in msst_cross_attention. */
int msst_adapter_gemm_workspace(long long rows, int K, int N, int adapters, int rank, long long* bytes);
int msst_adapter_gemm(const void* x, long long rows, int K, long long ldx, const void* w, int N, const float* bias,
                      const void* lora_a, const void* lora_b, const float* scales, int adapters, int rank,
                      const int* row_adapter, int dtype, void* out, long long ldo, void* workspace,
                      long long workspace_bytes, void* stream);

/* ---- operators of a cache of generated tokens behind one shared prefix: what a block
 * with single tokens needs beside its cross attention.  Requests have their own tokens in
 * pages of page_size tokens (a power of two from 16 to 256; slot = page * page_size +
 * place in the page), a block table [requests, blocks] int32 (row stride table_stride)
 * names a request's pages in order.  At most 8192 requests a call. */

/* Block tables and slots from request lengths.  free_pages [pages] is a stack of free
 * pages, *free_count its height (the entries below it are distinct and in no row).
 * First, in order of requests, each with new_tokens[r] < 0 has ended: its ceil(lens[r] /
 * page_size) pages go on top of the stack and its length becomes 0.  Then, in the same
 * order, the others take the pages that new_tokens[r] more tokens need off its top.  A
 * request whose need, added to those before it, passes what is free, whose tokens pass
 * its row of the table, or end past row `tokens`, is refused: it stays as it was, its rows have
 * slots -1, and msst_device_error reports 16.
 * Written: out_lens [requests] and *out_free_count (which may be lens and free_count
 * themselves), block_table and free_pages in place; q_starts [requests + 1], the first
 * row of each request among the call's new tokens, and for each of the `tokens` rows its
 * slot and its position start + place in the request (2^31 - 1 where a refused request's is
 * more; rows behind the last request: -1 and 0).  With outputs of their own a call may be repeated with the same result.
 * Lengths are taken into [0, blocks * page_size], the count into [0, pages]. */
int msst_cache_plan(const int* new_tokens, const int* lens, int requests, int* block_table, int blocks,
                    long long table_stride, int* free_pages, int pages, const int* free_count, int page_size, int start,
                    int tokens, int* out_lens, int* out_free_count, int* q_starts, int* slots, int* positions,
                    void* stream);

/* The position rotation of queries and keys, whose keys go to the pages with their
 * values.  q, k, v and q_out are [tokens, heads, head_dim] (msst_heads with tokens as the
 * sequence, batch_stride unused), the caches [pages, page_size, heads, head_dim] (pages as the
 * batch).  Each pair (a, b) of the first rot_dim columns of q and k (`pairing` as in
 * msst_qk_norm_rope) becomes amplitude * (a cos - b sin, b cos + a sin) of the angle
 * positions[t] * inv_freq[i] (double, [rot_dim / 2], radians; the angle is reduced in 64
 * bits, so far positions lose nothing), fp32 inside, one rounding.  The other columns and v
 * are copied.  q goes to q_out (which may be q itself, same strides, and otherwise must not
 * overlap it), k and v to slots[t] of the caches.  A token with a negative slot is not written to
 * them, one with a slot past the last page neither, and msst_device_error reports 17; the
 * slots of a call's tokens differ (of tokens that share one, either's columns may end up
 * there).  head_dim is a multiple of 8, <= 256, rot_dim a multiple of 8, <= head_dim (0:
 * no rotation); data pointers are 16-byte aligned, strides multiples of 8 elements. */
int msst_rope_append(const msst_heads* q, const msst_heads* k, const msst_heads* v, int tokens, int head_dim,
                     const int* positions, const int* slots, const double* inv_freq, int rot_dim, float amplitude,
                     int pairing, const msst_heads* k_cache, const msst_heads* v_cache, int pages, int page_size,
                     int dtype, const msst_heads* q_out, void* stream);

/* Attention to a prefix that all requests share and to each request's own tokens:
 * out = softmax(scale * q k^T) v over the prefix_len keys of prefix_k / prefix_v [prefix_len,
 * heads, head_dim] (none: prefix_len 0, the views may be NULL) and the request's own keys in the
 * caches.  q and out are [tokens, q.heads, head_dim], rows q_starts[r] to q_starts[r + 1]
 * (ascending, [requests + 1]; NULL: one row a request) request r's new tokens, which are
 * the last of its lens[r] own ones: the i-th of n sees the first lens[r] - n + i + 1 of them (not below 0).
 * The prefix is read once for all requests where these have fewer than 256 rows (tokens * q.heads / heads) on
 * average, and by each request for its own rows otherwise: a call of prompts had better not hold single tokens too.
 * q.heads is a multiple of the caches' heads, head_dim a multiple of 8 and <= 128,
 * scale 0 selects 1/sqrt(head_dim).  What a row does not see, the rest of a page
 * included, has no influence on it, whatever it holds; an infinity or
 * NaN in a v that it sees leaves that column infinite or NaN.  A row that sees no key gives zeros; rows of no request (before
 * the first or behind the last) are left as they were, or zeroed with zero_rest != 0.  A page outside the caches reads as zeros, and
 * msst_device_error reports 18.  lens is taken into [0, blocks * page_size].  out must
 * not overlap the inputs.  Precision, alignment and workspace as in msst_cross_attention
 * (head strides of the prefix and the caches may be 0). */
int msst_prefix_attention_workspace(int tokens, int requests, int prefix_len, int q_heads, int kv_heads, int head_dim,
                                    long long* bytes);
int msst_prefix_attention(const msst_heads* q, int tokens, const int* q_starts, int requests,
                          const msst_heads* prefix_k, const msst_heads* prefix_v, int prefix_len,
                          const msst_heads* k_cache, const msst_heads* v_cache, int pages, int page_size,
                          const int* block_table, int blocks, long long table_stride, const int* lens, int head_dim,
                          float scale, int dtype, const msst_heads* out, int zero_rest, void* workspace,
                          long long workspace_bytes, void* stream);

/* The three calls above with their arguments in one array, in their order, each an integer, a pointer or (float)
 * a double in 64 bits, a msst_heads as its five members (a NULL one: data NULL and 0 heads); integers beyond 32
 * bits count as the largest or smallest int.  For hosts whose foreign calls cost by the argument (Python's ctypes: 4.5 us for
 * 18, 1.2 for two). */
typedef union msst_word {
  long long i;
  double f;
  void* p;
} msst_word;
#define MSST_CALL_CACHE_PLAN 0
#define MSST_CALL_ROPE_APPEND 1
#define MSST_CALL_PREFIX_ATTENTION 2
int msst_call(int op, const msst_word* args);

/* One problem of msst_grouped_gemm: rows [a_row0, a_row0 + m) and columns
 * [a_col0, a_col0 + k) of x times rows [b_row0, b_row0 + n) (same k columns from
 * b_col0) of W, written to out rows out_row0.. and columns out_col0.. (for
 * MSST_EPI_GLU32 out_col0 counts output columns, n/2 per row); bias [n] or NULL. */
typedef struct msst_gemm_group {
  long long m, a_row0, out_row0;
  int n, k, a_col0, b_row0, b_col0, out_col0;
  const float* bias;
} msst_gemm_group;

/* Up to 64 independent GEMMs in one launch over one packed 16-bit x [x_rows, ldx]
 * and one packed 16-bit W [w_rows, ldw], all with the same epilogue (as
 * msst_gemm) into one output matrix out [out_rows, ldo].  Per group: k is a
 * multiple of 64 (pad K slices with zero columns); a_col0 and b_col0 are
 * multiples of 8 and out_col0 starts on 16 bytes (multiple of 8 for 16-bit, 4
 * for fp32 output).  The store / reduce epilogues write 32x32 blocks, so a
 * group's m (n) is a multiple of 32 unless its block ends at out_rows (ldo).
 * Replaces the reference's per-band GEMM loops of the band split and the mask
 * estimators (apply_band_split, apply_mask_estimator,
 * src/model_mel_band_roformer.cu:657-738, src/model_bs_roformer.cu:337-414),
 * which launch one cuBLAS GEMM per band. */
int msst_grouped_gemm(int num_groups, const msst_gemm_group* groups, const void* x, long long x_rows, long long ldx,
                      const void* w, long long w_rows, long long ldw, int epilogue, int act, int dtype, void* out,
                      long long out_rows, long long ldo, void* stream);

/* Device tables of a model's band gather and mask merge (read-only, owned by the
 * model; valid until msst_model_free).  Band b gathers nfreq[b] STFT bins
 * bin_list[bin_start[b] ..] into columns [kcol[b], kcol[b] + kpad[b]) of the
 * band-split input (2 * channels * nfreq[b] values, zero padding after), scaled
 * by gamma[gcol[b] ..].  Bin i of the mask merge sums the mask columns
 * contrib_col[contrib_off[i] .. contrib_off[i+1]) and divides by denom[i]. */
typedef struct msst_band_tables {
  int num_bands, nbins, channels, sum_kpad, sum_dims;
  const int* bin_start;
  const int* nfreq;
  const int* bin_list;
  const int* kcol;
  const int* kpad;
  const int* gcol;
  const float* gamma;
  const int* contrib_off;
  const int* contrib_col;
  const float* denom;
} msst_band_tables;
int msst_model_band_tables(const msst_model* m, msst_band_tables* tables);

/* Band gather + per-band RMSNorm (scale sqrt(band dims)) + 16-bit cast: spec is
 * the complex STFT in cuFFT R2C layout [B*C*T, nbins] (interleaved re/im fp32);
 * out16 [B*T, ldo] gets band b at columns [kcol[b], kcol[b] + kpad[b]) in the
 * reference's (bin, channel, re/im) order.  Replaces the per-band slice +
 * contiguous copy + rms_norm of apply_band_split and the mel-bin gather of
 * forward (src/model_mel_band_roformer.cu:657-690,808-829,
 * src/model_bs_roformer.cu:337-369,465-473). */
int msst_band_gather(const float* spec, int B, int T, const msst_band_tables* tables, int dtype, void* out16,
                     long long ldo, void* stream);

/* Mask merge: masks fp32 [S][B*T][sum_dims] (band-concatenated estimator output)
 * are averaged into bins (sum of the contributing bands / denom), multiplied
 * into the STFT spec [B*C*T, nbins] complex and written to out [(b*S + s)*C + c]
 * [T][nbins] complex (the iSTFT input), bin 0 zeroed when zero_dc != 0.
 * Replaces the scatter_add + average + complex multiply + zero-DC sequence of
 * forward (src/model_mel_band_roformer.cu:926-1015,
 * src/model_bs_roformer.cu:552-590). */
int msst_mask_apply(const float* spec, const float* masks, int B, int S, int T, const msst_band_tables* tables,
                    int zero_dc, float* out, void* stream);

/* ------------------------------------------------------------- model level -- */

/* Load a .csm model (format: src/weights.h:83-96) onto `device` with 16-bit
 * operands of type `precision` (replaces app::load_model,
 * src/inference_app.cpp:363-441, and the drivers' load(),
 * src/model_mel_band_roformer.cu:319-481, src/model_bs_roformer.cu:94-199). */
int msst_model_load(const char* path, int device, int precision, msst_model** out);
void msst_model_free(msst_model* m);
int msst_model_get_info(const msst_model* m, msst_model_info* info);

/* Whole forward pass on device buffers: audio [batch, channels, length] fp32 ->
 * out [batch, num_stems, channels, (length/hop)*hop] fp32 (the stem axis is
 * absent from the reference's shape when num_stems == 1; the memory layout is
 * the same).  Replaces MelBandRoformer::forward / BSRoformer::forward
 * (src/model_mel_band_roformer.cu:744, src/model_bs_roformer.cu:420). */
int msst_model_forward(msst_model* m, const float* audio, int batch, int channels, long long length, float* out,
                       void* stream);

/* Forward steps up to the mask estimators: fp32 masks
 * [batch, num_stems, T, sum_band_dims], T = length/hop + 1. */
int msst_model_masks(msst_model* m, const float* audio, int batch, int channels, long long length, float* masks,
                     void* stream);

/* One axial transformer (all its layers, plus the MelBandRoformer's final norm)
 * applied in place to the residual stream x fp32 [batch, T, num_bands, dim]
 * (replaces apply_transformer, src/model_mel_band_roformer.cu:628-651,
 * src/model_bs_roformer.cu:310-331, with the permutes of forward() folded away). */
int msst_model_transformer(msst_model* m, int depth_index, int axis, float* x, int batch, int T, void* stream);

/* Block level, in place on the residual stream x fp32 [batch, T, num_bands, dim]:
 * layer `layer` of the transformer (depth_index, axis).  The attention block is
 * RMSNorm + gate projection, QKV + RoPE, attention with gates and head merge, out
 * projection and residual add (replaces apply_attention + the residual add of
 * apply_transformer, src/model_mel_band_roformer.cu:519-591,628-651,
 * src/model_bs_roformer.cu:236-284,310-331); the feed-forward block is RMSNorm,
 * Linear + GELU, Linear and residual add (apply_feedforward,
 * src/model_mel_band_roformer.cu:597-622, src/model_bs_roformer.cu:290-304).
 * Neither applies the MelBandRoformer's per-transformer final norm
 * (msst_model_transformer does). */
int msst_roformer_attn_block(msst_model* m, int depth_index, int axis, int layer, float* x, int batch, int T,
                             void* stream);
int msst_roformer_ffn_block(msst_model* m, int depth_index, int axis, int layer, float* x, int batch, int T,
                            void* stream);

/* msst_model_transformer for callers that cannot allocate device memory while
 * they run: real-time audio hosts, whose processing callback has a hard deadline
 * that a cudaMalloc / cudaFree (which can block and synchronise the device)
 * would break, and applications that own every device allocation themselves.
 * There is no counterpart in the reference.  All intermediates live in one
 * fixed 48 MiB device array inside the library (held on every GPU that loads
 * it, until exit); nothing is allocated.  A call over batch*T*num_bands tokens
 * needs about dim*2 + heads*4 + 2*max(3*heads*64, 4*dim) + heads*128 bytes per
 * token (about 10,000 tokens at dim 384) and larger calls fail with
 * MSST_ERR_INVALID.  Calls on one device share the array: calls that overlap on
 * the GPU race.  The first call on a device looks up the array's device address,
 * and under CUDA's lazy module loading it is also when the driver loads the
 * library's module and backs the array with device memory: make one warm-up
 * call per device at start-up, off the real-time thread and before any stream
 * capture.  Later calls allocate nothing and do not synchronise the stream. */
int msst_model_transformer_noalloc(msst_model* m, int depth_index, int axis, float* x, int batch, int T,
                                   void* stream);

/* Chunked overlap-add separation of one track (replaces app::run_inference /
 * process_chunked, src/inference_app.cpp:100-324,443-497).  track [channels,
 * length] -> out [num_stems, channels, length].  overlap: (0,1) = overlap
 * ratio, >= 1 = num_overlap, 0 = model default.  chunk_batch <= 0 uses the
 * reference default (2).  *_host variants take host memory (copies included). */
int msst_model_separate(msst_model* m, const float* track, int channels, long long length, float overlap,
                        int chunk_batch, int flags, float* out, void* stream);
int msst_model_separate_host(msst_model* m, const float* track_host, int channels, long long length, float overlap,
                             int chunk_batch, int flags, float* out_host);

/* Sharded separation of one track across GPUs (the reference is single-GPU;
 * these split msst_model_separate at its independent unit, the chunk).
 * msst_model_forward_chunks runs chunks [first_chunk, first_chunk + count) of the
 * track's chunk plan: track [channels, length] (device) -> out [count,
 * num_stems*channels, chunk_size] (device).  msst_model_stitch overlap-adds the
 * outputs of all chunks of the plan, chunks [num_chunks, num_stems*channels,
 * chunk_size], into out [num_stems, channels, length], in chunk order, so the
 * result equals msst_model_separate's. */
int msst_model_forward_chunks(msst_model* m, const float* track, int channels, long long length, float overlap,
                              int first_chunk, int count, int chunk_batch, int flags, float* out, void* stream);
int msst_model_stitch(msst_model* m, const float* chunks, int channels, long long length, float overlap, float* out,
                      void* stream);

/* Round-robin sharding (chunk i on rank i % world, the reference's chunk list of
 * src/inference_app.cpp:131-137 dealt out): msst_model_forward_chunks over chunks
 * first_chunk, first_chunk + chunk_stride, ... (count of them). */
int msst_model_forward_chunks_strided(msst_model* m, const float* track, int channels, long long length,
                                      float overlap, int first_chunk, int chunk_stride, int count, int chunk_batch,
                                      int flags, float* out, void* stream);

/* The overlap-add of msst_model_stitch (src/inference_app.cpp:252-306,
 * src/ops_fused.cu:138-188) for output samples [begin, end) only, written into
 * out [num_stems, channels, length] (other samples untouched).  Chunk k's output
 * [num_stems*channels, chunk_size] is read from slot (k % slot_ranks) * slot_cap +
 * k / slot_ranks of `chunks` (slot_ranks = 1, slot_cap = num_chunks: chunk order;
 * slot_ranks = world: each rank's round-robin shard after the previous rank's).
 * Each sample is summed over its chunks in chunk order, so stitching a track in
 * ranges gives the same result as one msst_model_stitch. */
int msst_model_stitch_range(msst_model* m, const float* chunks, int slot_ranks, int slot_cap, int channels,
                            long long length, float overlap, long long begin, long long end, float* out,
                            void* stream);

/* Sample ranges of chunk `chunk_index` of a track's plan.  in_ranges[4] receives
 * two ranges [begin, end) of the track its gather reads: its own reflect-padded
 * window, and (only for a short final chunk with the reference's padding, i.e.
 * without MSST_SEPARATE_FIX_TAIL_PADDING) the first samples of the track that
 * padding reads, else an empty range.  [*out_begin, *out_end) is the output its
 * overlap-add touches: output samples before chunk k's out_begin are final once
 * chunks 0..k-1 are stitched. */
int msst_model_chunk_span(const msst_model* m, long long length, float overlap, int chunk_index, int flags,
                          long long* in_ranges, long long* out_begin, long long* out_end);

/* Chunk plan of msst_model_separate for a track length (src/inference_app.cpp:119-138). */
int msst_model_chunk_plan(const msst_model* m, long long length, float overlap, int* chunk_size, int* step,
                          long long* border, long long* padded_length, int* num_chunks);

#ifdef __cplusplus
}
#endif

#endif /* MSST_B200_H */
