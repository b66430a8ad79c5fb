/*
 * flash_hog.h - C ABI of the MI355X-native Flash-HOG attention kernels.
 *
 * Plain pointers and sizes only. Every entry point enqueues its kernels on the
 * given HIP stream and returns without synchronising; it allocates nothing,
 * frees nothing and keeps no pointer after it returns (all outputs and the
 * fp32 row-statistic workspace are caller owned, as the reference's XLA FFI
 * handler exposes its dD/B scratch as results). No entry point except
 * fhog_attention_bwdbwd_noalloc holds mutable global state, so concurrent
 * calls on different streams are safe.
 *
 * Layouts (identical to the reference's attention seam):
 *   q, o, dout, ddq, dq, dq2, ddo   : (batch, n_q, heads, head_dim) contiguous
 *   k, v, ddk, ddv, dk, dv, dk2, dv2: (batch, n_k, kv_heads, head_dim) contiguous
 *   lse, delta, ddelta, bstat       : (batch, heads, n_q) fp32 contiguous
 * lse is the natural-log logsumexp of the scaled, masked logits
 * (flash_hog/jax/_pallas_gpu_kernel.py:97).
 *
 * Grouped-query attention: heads must be a multiple of kv_heads; query head h
 * attends with key/value head h / (heads / kv_heads), and dk, dv, dk2, dv2 sum
 * over the heads of a group (_pallas_gpu_kernel.py:99, 106-107, 333-370).
 *
 * causal (enum fhog_causal): FHOG_CAUSAL_TOP_LEFT shows key j to query i iff
 * j <= i (_pallas_gpu_kernel.py:37-41, the reference kernel's mask);
 * FHOG_CAUSAL_BOTTOM_RIGHT iff j <= i + n_k - n_q
 * (flash_hog/_jax_refs/jax_impl.py:104-109); the two agree when n_q == n_k.
 * A query that sees no key (bottom-right with n_q > n_k) gets o = 0,
 * lse = +inf and zero gradients.
 * Tensor pointers must be 16-byte aligned, row-statistic pointers 4-byte aligned.
 *
 * Supported: dtype FHOG_DTYPE_{BF16,F16} with head_dim 64, 128 or 256,
 * FHOG_DTYPE_F32 with head_dim 64 or 128; any n_q, n_k >= 1 (ragged tails
 * are masked); any finite nonzero scale, negative included (scale 0 returns
 * FHOG_ERR_UNSUPPORTED).
 */
#ifndef FLASH_HOG_H_
#define FLASH_HOG_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same type as hipStream_t. */
typedef struct ihipStream_t* fhog_stream_t;

enum fhog_status {
  FHOG_OK = 0,
  FHOG_ERR_INVALID_ARGUMENT = 1, /* null/misaligned pointer, bad size, bad enum */
  FHOG_ERR_UNSUPPORTED = 2,      /* valid request the library has no kernel for */
  FHOG_ERR_LAUNCH = 3            /* the HIP runtime rejected a kernel launch */
};

/* E4M3: paged caches only. */
enum fhog_dtype { FHOG_DTYPE_F32 = 0, FHOG_DTYPE_F16 = 1, FHOG_DTYPE_BF16 = 2, FHOG_DTYPE_E4M3 = 3 };

/* Values of the `causal` argument. */
enum fhog_causal { FHOG_CAUSAL_NONE = 0, FHOG_CAUSAL_TOP_LEFT = 1, FHOG_CAUSAL_BOTTOM_RIGHT = 2 };

/* Version of this ABI (major * 100 + minor). */
int fhog_abi_version(void);

/* Static description of a status code. */
const char* fhog_status_string(int status);

/* Message of the last failed call on this thread ("" if none). */
const char* fhog_last_error(void);

/*
 * Whether this library has kernels for the given problem, without launching
 * or allocating anything: FHOG_OK, or the status (with its fhog_last_error
 * message) that the entry points would return for these sizes, dtype, causal
 * and scale. device >= 0 also requires HIP device `device` to be a gfx950
 * GPU (else FHOG_ERR_UNSUPPORTED); device < 0 checks the arguments only.
 * Counterpart of the reference's supported() (flash_hog/jax/_tk_gpu.py:70-80),
 * which answers the same question for its ThunderKittens kernels before a
 * call, so that a caller can route unsupported shapes elsewhere.
 */
int fhog_attention_supported(int device, int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                             int dtype, int causal, float scale);

/* Bytes of fp32 row-statistic workspace per (delta, ddelta, bstat) array:
 * batch * heads * n_q * 4. */
size_t fhog_row_stat_bytes(int batch, int heads, int n_q);

/*
 * Forward: o = softmax(scale q k^T [causal]) v and lse.
 * Replaces the cuDNN forward the reference reaches through
 * dot_product_attention_fwd / dot_product_attention_fwd_rule
 * (flash_hog/jax/_attention_impl.py:224-239), which returns (out, activation)
 * with activation = the (B, N, T) fp32 logsumexp.
 */
int fhog_attention_fwd(fhog_stream_t stream,
                       const void* q, const void* k, const void* v,
                       void* o, float* lse,
                       int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                       int dtype, int causal, float scale);

/*
 * First backward: dq, dk, dv from (q, k, v, o, lse, dout).
 * Replaces the cuDNN backward the reference reaches through
 * dot_product_attention_bwd_rule (flash_hog/jax/_attention_impl.py:242-261).
 * delta (caller-owned, fhog_row_stat_bytes) receives D = rowsum(o * dout).
 */
int fhog_attention_bwd(fhog_stream_t stream,
                       const void* q, const void* k, const void* v,
                       const void* o, const void* dout, const float* lse,
                       void* dq, void* dk, void* dv, float* delta,
                       int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                       int dtype, int causal, float scale);

/*
 * Double backward (Flash-HOG): given the residual (q, k, v, o, lse, dout) of
 * the first backward and the cotangents (ddq, ddk, ddv) of its outputs,
 * returns dq2, dk2, dv2 (cotangents of q, k, v) and ddo (cotangent of dout).
 * Replaces dot_product_attention_bwd_rule_bwd_rule
 * (flash_hog/jax/_attention_impl.py:278-303) -> flash_bwdbwd
 * (flash_hog/jax/_pallas_gpu.py:51-114) -> flash_bwdbwd0
 * (flash_hog/jax/_pallas_gpu_kernel.py:49-422), and the XLA FFI handler
 * TkBwdBwd (flash_hog/csrc/tk_bwdbwd/ffi.cu:26-98), whose inputs
 * (Q,K,V,dO,ddQ,ddK,ddV,L,D), attribute scale and results
 * (dQ2,ddO,dK2,dV2,dD,B) it mirrors, except that D is computed here from o
 * (as flash_bwdbwd0 does at _pallas_gpu_kernel.py:110) and written to delta.
 * delta, ddelta, bstat: caller-owned workspace, fhog_row_stat_bytes each;
 * on return they hold D, dD and B. Like TkBwdBwd's dD and B they are
 * scratch between the two passes (pass 4 uses B through c = D dD + B).
 * Accuracy: D, dD and B are fp32 sums of fp32 per-pair terms (2-byte types:
 * B = sum_j X_j - dD (sum_j P_j u_j + D), the per-pair form; fp32:
 * B = r1 - dD r2 - D dD + r3). Over a call each is within the dtype's
 * tolerance of its exact value relative to its own largest entry. Per row,
 * B = c - D dD is a difference that any formula for it must take, so a row
 * whose B is much smaller than its D dD holds B only to about 1e-7 |c|
 * (fp32 rounding of c), not to 1e-7 |B|.
 * Two kernels are enqueued on stream; the second reads the statistics the
 * first writes.
 */
int fhog_attention_bwdbwd(fhog_stream_t stream,
                          const void* q, const void* k, const void* v,
                          const void* o, const void* dout,
                          const void* ddq, const void* ddk, const void* ddv,
                          const float* lse,
                          void* dq2, void* dk2, void* dv2, void* ddo,
                          float* delta, float* ddelta, float* bstat,
                          int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                          int dtype, int causal, float scale);

/*
 * One stage of fhog_attention_bwdbwd: stage 1 = passes 1-3 (tiled over
 * queries; computes D, dD, B into delta/ddelta/bstat and writes dq2, ddo),
 * stage 2 = pass 4 (tiled over keys; reads delta/ddelta/bstat, writes dk2,
 * dv2). Running stage 1 then stage 2 on one stream equals
 * fhog_attention_bwdbwd. The reference's handler always launches both
 * (ffi.cu:71-73); the split exists so that the stages can be timed, profiled
 * or ordered by the caller (stage 2 must see stage 1's statistics). Pointers
 * a stage does not touch may be null: stage 1 ignores dk2, dv2; stage 2
 * ignores o, dq2, ddo.
 */
int fhog_attention_bwdbwd_stage(fhog_stream_t stream, int stage,
                                const void* q, const void* k, const void* v,
                                const void* o, const void* dout,
                                const void* ddq, const void* ddk, const void* ddv,
                                const float* lse,
                                void* dq2, void* dk2, void* dv2, void* ddo,
                                float* delta, float* ddelta, float* bstat,
                                int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                                int dtype, int causal, float scale);

/*
 * fhog_attention_bwdbwd without the row-statistic workspace arguments: D, dD
 * and B go to a static device array inside the library (12 MiB per device,
 * for batch * heads * n_q up to 1048576 rows; larger calls return
 * FHOG_ERR_UNSUPPORTED). Outputs are those of fhog_attention_bwdbwd, bit for
 * bit. It calls no allocating routine, for callers that cannot allocate
 * device memory (code under HIP graph capture, serving loops, harnesses
 * that forbid hipMalloc); the first call on a device looks up the array's
 * address there once. It has no counterpart in the reference; it is for
 * callers that cannot allocate. Every call on a device shares
 * that device's array: calls that overlap on one device (concurrent streams)
 * race on it and must be serialised by the caller.
 */
int fhog_attention_bwdbwd_noalloc(fhog_stream_t stream,
                                  const void* q, const void* k, const void* v,
                                  const void* o, const void* dout,
                                  const void* ddq, const void* ddk, const void* ddv,
                                  const float* lse,
                                  void* dq2, void* dk2, void* dv2, void* ddo,
                                  int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                                  int dtype, int causal, float scale);

/*
 * Attention over a window of keys with sinks: with p = i (causal 1, top-left) or
 * p = i + n_k - n_q (causal 2, bottom-right; causal 0 is invalid), query i sees key j iff
 * j <= p and (j > p - window or j < sinks), window >= 1, sinks >= 0. Everything else is as
 * in the entry points of the same name without a window, the double backward included; a
 * query that sees no key (also top-left, n_q > n_k, behind the last key's window) gets o = 0,
 * lse = +inf and zero gradients. These have no counterpart in the reference.
 * Work and memory grow with n_q * window and n_q + n_k.
 *
 * workspace (caller-owned, 16-byte aligned, fhog_window_workspace_bytes; may be null when
 * that is 0, as without sinks): fp32 parts of the sinks' dk and dv rows, scratch between the
 * kernels of one call. Calls that may overlap need one each.
 */
size_t fhog_window_workspace_bytes(int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype,
                                   int causal, int window, int sinks);

int fhog_window_attention_fwd(fhog_stream_t stream,
                              const void* q, const void* k, const void* v,
                              void* o, float* lse,
                              int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                              int dtype, int causal, int window, int sinks, float scale);

int fhog_window_attention_bwd(fhog_stream_t stream,
                              const void* q, const void* k, const void* v,
                              const void* o, const void* dout, const float* lse,
                              void* dq, void* dk, void* dv, float* delta, void* workspace,
                              int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                              int dtype, int causal, int window, int sinks, float scale);

int fhog_window_attention_bwdbwd(fhog_stream_t stream,
                                 const void* q, const void* k, const void* v,
                                 const void* o, const void* dout,
                                 const void* ddq, const void* ddk, const void* ddv,
                                 const float* lse,
                                 void* dq2, void* dk2, void* dv2, void* ddo,
                                 float* delta, float* ddelta, float* bstat, void* workspace,
                                 int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                                 int dtype, int causal, int window, int sinks, float scale);

/*
 * The paged key/value cache (no counterpart in the reference): serving the attention that the
 * entry points above train.
 *
 * k_cache, v_cache: (num_pages, kv_heads, page_size, head_dim) contiguous, of the calls' dtype
 * (bf16 or fp16) or FHOG_DTYPE_E4M3; page_size a power of two >= 16, head_dim 64, 128 or 256.
 * k_scale, v_scale: (num_pages, kv_heads, page_size) e8m0 bytes of an e4m3 cache (a row's values
 * are code * 2^(byte - 127)), ignored otherwise.
 * page_table: (batch, pages_per_seq) int32; token s of sequence b is row s % page_size of page
 * page_table[b][s / page_size]. lengths: (batch) int32, the tokens that each sequence holds,
 * the new ones included.
 * query_offsets: (batch + 1) int32, rising: the new tokens of sequence b are the packed rows
 * query_offsets[b] to query_offsets[b + 1], its last positions in order. Null: one new token a
 * sequence (total == batch).
 * table, lengths and offsets are device memory and read by the kernels only: no entry point
 * waits for the device. Entries that no visible token needs may hold anything. A needed entry
 * outside [0, num_pages), or a length beyond pages_per_seq * page_size, gives NaN rows
 * (attention, read) or leaves the token unwritten (write); offsets are cut to [0, total].
 */

/* Bytes of workspace of fhog_paged_attention on the current device; single: query_offsets is
 * null. Calls that may overlap need one each. */
size_t fhog_paged_workspace_bytes(int batch, int total, int single, int heads, int kv_heads, int head_dim,
                                  int page_size, int pages_per_seq, int window, int sinks);

/*
 * out (total, heads, head_dim): attention of the new tokens q (same shape) over the cached
 * keys of their sequences, their own among them (written before). Token i of n new ones is at
 * position p = length - n + i and sees the keys j <= p, with window > 0 those with j > p - window
 * or j < sinks only. A token that sees no key gets 0. Rows of no sequence (before
 * query_offsets[0], from query_offsets[batch] on) are zeroed if clear_rest, else left as they were.
 */
int fhog_paged_attention(fhog_stream_t stream, const void* q, const void* k_cache, const void* v_cache,
                         const void* k_scale, const void* v_scale, const int* page_table, const int* lengths,
                         const int* query_offsets, void* out, void* workspace, size_t workspace_bytes, int batch,
                         int total, int heads, int kv_heads, int head_dim, int num_pages, int page_size,
                         int pages_per_seq, int dtype, int cache_dtype, int window, int sinks, int clear_rest,
                         float scale);

/*
 * Writes the keys and values of the new tokens, (total, kv_heads, head_dim), to their places.
 * e4m3: a row's scale is the smallest power of two (at least 2^-126) with which its largest
 * finite magnitude stays within 448; values round to nearest even, infinities become NaN.
 * Every token's place must be its own; a place that two tokens name holds either's bytes.
 */
int fhog_paged_cache_write(fhog_stream_t stream, const void* k, const void* v, void* k_cache, void* v_cache,
                           void* k_scale, void* v_scale, const int* page_table, const int* lengths,
                           const int* query_offsets, int batch, int total, int kv_heads, int head_dim, int num_pages,
                           int page_size, int pages_per_seq, int dtype, int cache_dtype);

/* Tokens [0, min(length, max_length)) of each sequence, as k and v (batch, max_length, kv_heads,
 * head_dim); zeros behind a sequence's length. */
int fhog_paged_cache_read(fhog_stream_t stream, const void* k_cache, const void* v_cache, const void* k_scale,
                          const void* v_scale, const int* page_table, const int* lengths, void* k, void* v, int batch,
                          int max_length, int kv_heads, int head_dim, int num_pages, int page_size,
                          int pages_per_seq, int dtype, int cache_dtype);

/*
 * The cache's allocator. The page table and the lengths are its only state: a page is used if a row of the
 * table has it among its first ceil(length / page_size) entries (those in [0, num_pages)), else free.
 *
 * extend: in place and in one step for all rows, row b becomes row parents[b] (null: each its own; an
 * index outside [0, batch): an empty row) and then grows by max(0, new_tokens[b]) tokens (null:
 * new_each). If its last page is not full and it grows, that page becomes its own: it keeps it if all other
 * users are rows of higher index that grow in it as well, else the rows held in it are copied (keys,
 * values, scales) to a new page. New pages are the free ones (by the rows' state after parents), lowest
 * first, to the rows in order, each row's columns in order. Entries behind a row's last page become -1, and so do
 * those that no page was left for; *free_pages (device memory) = the free pages that are left, less
 * those that were lacking. A length may grow beyond its table, and past 2^31 - 1 it stays there.
 * parents, new_tokens (batch) int32. k_scale, v_scale: of an e4m3 cache.
 */
size_t fhog_paged_pages_workspace_bytes(int batch, int num_pages, int pages_per_seq);

int fhog_paged_cache_extend(fhog_stream_t stream, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                            int* page_table, int* lengths, const int* parents, const int* new_tokens, int new_each,
                            int* free_pages, void* workspace, size_t workspace_bytes, int batch, int kv_heads,
                            int head_dim, int num_pages, int page_size, int pages_per_seq, int cache_dtype);

/* The used pages, in their order, as the first pages of another cache of out_pages pages (zero bytes behind them),
 * and the table (batch, pages_per_seq) for it: -1 where there is no page, and for used ones that out_pages
 * has no room for. key_means, means_out: fhog_paged_key_means' of both, or null. All tensors 16-byte
 * aligned, the outputs apart from the inputs. */
int fhog_paged_cache_compact(fhog_stream_t stream, const void* k_cache, const void* v_cache, const void* k_scale,
                             const void* v_scale, const float* key_means, const int* page_table, const int* lengths,
                             void* k_out, void* v_out, void* k_scale_out, void* v_scale_out, float* means_out,
                             int* table_out, void* workspace, size_t workspace_bytes, int batch, int kv_heads,
                             int head_dim, int num_pages, int page_size, int pages_per_seq, int out_pages,
                             int cache_dtype);

/*
 * Attention over chosen blocks. A block is a page, named by its column of the page table.
 *
 * key_means (num_pages, kv_heads, head_dim) fp32: the means of the full pages' keys (summed in 64 bits, rounded
 * once; e4m3 keys are code * scale). This call writes those of the pages that the new tokens fill, the
 * last query_offsets[b + 1] - query_offsets[b] (null: one) of each sequence, and leaves the others.
 */
int fhog_paged_key_means(fhog_stream_t stream, const void* k_cache, const void* k_scale, float* key_means,
                         const int* page_table, const int* lengths, const int* query_offsets, int batch, int kv_heads,
                         int head_dim, int num_pages, int page_size, int pages_per_seq, int cache_dtype);

/*
 * chosen (total, kv_heads, blocks) int32: for each new token, at position p, and key/value head the columns to attend
 * to, rising, -1 behind them. Of columns 0 to p / page_size: the first `first` (>= 0), the last `last` (>= 1, so that
 * a page that is not full yet is never chosen by its mean), and of the others those whose mean has the largest
 * product with the sum of the queries q (total, heads, head_dim) of the head's group, formed in 64 bits (in an order
 * that goes with the number of tokens, so products apart by a rounding there may change places), ties to the lowest
 * column, NaN (also: a page outside the cache) last; `blocks` (>= first + last) in all, or all there are. Tokens of no
 * sequence, before position 0 or beyond the table: -1 throughout. Offsets that fall somewhere may leave lists of any values.
 */
size_t fhog_paged_block_select_workspace_bytes(int batch, int total, int single, int kv_heads, int head_dim,
                                               int pages_per_seq, int first, int last);
int fhog_paged_block_select(fhog_stream_t stream, const void* q, const float* key_means, const int* page_table,
                            const int* lengths, const int* query_offsets, int* chosen, void* workspace,
                            size_t workspace_bytes, int batch, int total, int heads, int kv_heads, int head_dim,
                            int num_pages, int page_size, int pages_per_seq, int dtype, int blocks, int first, int last);

/*
 * fhog_paged_attention (without a window) in which a token sees, through each key/value head, only the keys
 * of the pages in columns chosen[token][head], up to its own position. Columns outside [0, pages_per_seq) and
 * ones behind the token show nothing; one that is named twice counts twice. Offsets that fall somewhere may give NaN
 * in every row. The workspace of many tokens is as large as an fp32 output for each of their blocks, and 12 bytes for each
 * column of 64 tokens and a key/value head; that of long lists as a few outputs for each token. Up to 1.1 GiB: more tokens
 * are taken in turn.
 */
size_t fhog_paged_block_workspace_bytes(int batch, int total, int single, int heads, int kv_heads, int head_dim,
                                        int page_size, int pages_per_seq, int blocks);
int fhog_paged_block_attention(fhog_stream_t stream, const void* q, const int* chosen, const void* k_cache,
                               const void* v_cache, const void* k_scale, const void* v_scale, const int* page_table,
                               const int* lengths, const int* query_offsets, void* out, void* workspace,
                               size_t workspace_bytes, int batch, int total, int heads, int kv_heads, int head_dim,
                               int num_pages, int page_size, int pages_per_seq, int dtype, int cache_dtype, int blocks,
                               int clear_rest, float scale);

/*
 * Norms of queries and keys for each head with the position rotation, and their derivatives (no
 * counterpart in the reference): what stands before the attention of either kind.
 *
 * A row x of head_dim values of q (batch, tokens, heads, head_dim) or k (.., kv_heads, ..) becomes
 * R(w x (mean x^2 + eps)^-1/2), where R turns pairs of its first `rotated` columns (even; 0: none) by the
 * angles position * frequencies[i], formed in 64 bits: columns i and i + rotated / 2, or 2 i and 2 i + 1
 * if interleaved. norm 0: R(x). Any head_dim from 1 to 256, bf16, fp16 or fp32; sums are fp32.
 */
typedef struct fhog_rotary {
  int batch, tokens, heads, kv_heads, head_dim, rotated;
  int dtype;        /* of the rows */
  int weight_dtype; /* of the weights and their gradients: dtype or FHOG_DTYPE_F32 */
  int interleaved, norm;
  float eps;
  int position_bytes;       /* 4 or 8: an element of `positions`; otherwise ignored */
  int position_rows;        /* of `positions`: 1 (tokens) or batch (batch, tokens) */
  int sequences;            /* of `lengths` */
  long long q_stride[3];    /* elements between batches, tokens and heads of q, whose rows are contiguous */
  long long k_stride[3];
  const float* frequencies; /* (rotated / 2), null if rotated is 0 */
  const void* positions;    /* whole numbers, or null */
  /* A paged cache's (see there), with batch 1 and positions null: the tokens are packed and take the last
   * positions of their sequences; rows of no sequence are at position 0. Both null, and positions
   * too: a token's place in its batch. */
  const int* lengths;
  const int* query_offsets;
} fhog_rotary;

/* Bytes of workspace of the two backwards on the current device (0 without norms; without weights it may be
 * null). Calls that may overlap need one each. */
size_t fhog_qk_norm_rotary_workspace_bytes(const fhog_rotary* shape);

/* q_out, k_out (contiguous, as all tensors but q and k) from q, k and the weights (head_dim) of their
 * norms; a null weight is ones. shape and the arrays in it are read before the call returns. */
int fhog_qk_norm_rotary_fwd(fhog_stream_t stream, const fhog_rotary* shape, const void* q, const void* k,
                            const void* q_weight, const void* k_weight, void* q_out, void* k_out);

/* dq, dk and the weights' gradients (null where the weight is) from the cotangents of q_out and k_out.
 * Without norms q and k are not read and may be null. */
int fhog_qk_norm_rotary_bwd(fhog_stream_t stream, const fhog_rotary* shape, const void* q, const void* k,
                            const void* q_weight, const void* k_weight, const void* dq_out, const void* dk_out,
                            void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace);

/* With cotangents (ddq, ddk, ddq_weight, ddk_weight) of the backward's results: cotangents of its
 * inputs q, k, the weights, dq_out and dk_out. Norms only (without them the backward is
 * linear, and its derivative the forward). */
int fhog_qk_norm_rotary_bwdbwd(fhog_stream_t stream, const fhog_rotary* shape, const void* q, const void* k,
                               const void* q_weight, const void* k_weight, const void* dq_out, const void* dk_out,
                               const void* ddq, const void* ddk, const void* ddq_weight, const void* ddk_weight,
                               void* dq2, void* dk2, void* dq_weight2, void* dk_weight2, void* ddq_out, void* ddk_out,
                               void* workspace);

#ifdef __cplusplus
}
#endif

#endif /* FLASH_HOG_H_ */
