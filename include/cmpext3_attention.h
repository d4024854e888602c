/*
 * cmpext3_attention.h -- C ABI of the attention operators of the MI355X (gfx950)
 * library (libcmpext3_gemm.so): norms and rotation of queries and keys, a paged
 * cache of keys and values in 16 or 8 bits, and attention over packed prompts or
 * over that cache.
 *
 * The conventions are those of cmpext3_gemm.h: device pointers owned by the
 * caller, strides in elements, no allocation, no synchronisation, work enqueued on
 * `stream`, CMPEXT3_OK or a CMPEXT3_ERR_* / hipError_t as the result, nothing
 * launched when an argument is rejected.  A structure that is cleared to zero
 * before its fields are set stays valid when fields are added behind the last one.
 *
 * What only the device knows (lengths, starts, page numbers, slots, positions) is
 * checked there: no value makes a kernel read or write outside the given tensors.
 */
#ifndef CMPEXT3_ATTENTION_H
#define CMPEXT3_ATTENTION_H

#include <stdint.h>

#include "cmpext3_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of a cache: 8-bit floats with 4 exponent and 3 mantissa bits, no
 * infinities (OCP e4m3), with one fp32 scale for each token and head. */
#define CMPEXT3_E4M3 3

/*
 * Norms of queries and keys for each head, then the rotation of positions, in one pass:
 *   y = x * rsqrt(mean(x^2) + eps) * weight       (weight NULL: y = x)
 *   (a, b) -> (a cos - b sin, b cos + a sin)      for the pairs of the first rotary_dim elements
 * with pairs (i, i + rotary_dim/2), or (2i, 2i+1) if `interleaved`, and
 * cos/sin[position * table_row + i]; the elements past rotary_dim are not turned.
 * All arithmetic in fp32, rounded once.  q is [tokens, heads, dim], k [tokens, kv_heads,
 * dim], with unit stride inside a head; the outputs may be the inputs.  A token whose
 * position is outside [0, table_rows) gets NaN in its rotated elements.
 */
typedef struct cmpext3_qk_norm_rope_args {
  int32_t dtype; /* CMPEXT3_F16, CMPEXT3_BF16, CMPEXT3_F32 (q, k, weights and outputs) */
  int32_t interleaved;
  int32_t heads, kv_heads, dim, rotary_dim;
  int64_t tokens;
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_token, q_head, k_token, k_head;             /* strides of the inputs  */
  int64_t q_out_token, q_out_head, k_out_token, k_out_head; /* strides of the outputs */
  const void* q_weight; /* [dim] or NULL */
  const void* k_weight;
  const float* cos; /* [table_rows, rotary_dim / 2] */
  const float* sin;
  int64_t table_rows, table_row;
  const int64_t* positions; /* [tokens] */
  float eps;
} cmpext3_qk_norm_rope_args;
int cmpext3_qk_norm_rope(const cmpext3_qk_norm_rope_args* args, void* stream);

/*
 * A paged cache: k and v are [pages, page_size, kv_heads, dim] with any strides of
 * multiples of 16 bytes and unit stride inside a head.  With kv_dtype CMPEXT3_E4M3 each
 * token and head holds codes and a scale (k_scale, v_scale: [pages, page_size, kv_heads]):
 *   scale = max(max |x|, 2^-100) / 448,   code = e4m3(x * (448 / max(max |x|, 2^-100)))
 * over the finite elements; an element that is not finite is held as NaN.
 */
typedef struct cmpext3_kv_cache {
  int32_t kv_dtype; /* CMPEXT3_F16, CMPEXT3_BF16 or CMPEXT3_E4M3 */
  int32_t pages, page_size, kv_heads, dim;
  void* k;
  void* v;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;
  float* k_scale;
  float* v_scale;
  int64_t ks_page, ks_token, ks_head, vs_page, vs_token, vs_head;
} cmpext3_kv_cache;

/*
 * Writes k and v ([tokens, kv_heads, dim], dtype CMPEXT3_F16 or CMPEXT3_BF16, that of a
 * 16-bit cache) into the slots slots[token] = page * page_size + place.  A token whose slot
 * is outside the cache is left out; two tokens with one slot leave it undefined which is held.
 */
int cmpext3_kv_cache_write(const cmpext3_kv_cache* cache, int dtype, const void* k, int64_t k_token, int64_t k_head,
                           const void* v, int64_t v_token, int64_t v_head, const int64_t* slots, int64_t tokens,
                           void* stream);

/*
 * Reads the sequences' tokens back as packed rows k_out, v_out ([total, kv_heads, dim]
 * contiguous, of `dtype`): rows starts[b] .. starts[b+1]-1 are tokens 0, 1, ... of sequence
 * b, found through block_table[b * table_row + token / page_size].  Rows in no sequence, past
 * the table's table_pages columns or with a page number outside the cache are zeros.  Starts that
 * fall leave it undefined which sequence a row is taken from.
 */
int cmpext3_kv_cache_read(const cmpext3_kv_cache* cache, const int32_t* block_table, int64_t table_row,
                          int32_t table_pages, const int32_t* starts, int32_t batch, int64_t total, int dtype,
                          void* k_out, void* v_out, void* stream);

/*
 * Attention with grouped heads (heads a multiple of kv_heads; head h uses kv head
 * h / (heads / kv_heads)):
 *   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale * q_i . k_j)
 * over j < len_k, and with `causal` j <= i + len_k - len_q (the last query sees the last
 * key).  A query that sees no key gets zeros, one whose scores are all -inf NaN; keys, values and
 * scales that a query does not see take no part in its row, NaN and infinity among them.
 * Products on the matrix cores with fp32 sums, softmax statistics in fp32.  For the second
 * product the weights p (times their values' scales) are held
 *   pages, up to 32 rows of a sequence and kv head on average: as two 16-bit numbers each (over
 *     e4m3 both bf16), so that the result is off by its own rounding only;
 *   otherwise: rounded to the type of q.  In fp16, which ends at 2^-25, a row's largest weight is
 *     taken as 2^10 to 2^14, and the scales of each 64 values in a power of two of their own size.
 *
 * Keys and values: packed (cache.k/v with k_token, k_head, ...; block_table NULL), where
 * cache.k_page is the stride between batch entries of uniform length; or paged (block_table
 * set).  cache.dim and cache.kv_heads always hold; cache.pages and page_size for pages only.
 * Lengths: starts_q NULL means batch entries of len_q queries each at a stride of q_batch,
 * else sequence b has rows starts_q[b] .. starts_q[b+1]-1 of total_q, starts_q not falling (rows
 * before the first sequence and past the last get zeros); the same for keys with starts_k,
 * len_k, total_k when packed, and seq_lens[b] keys when paged.
 */
typedef struct cmpext3_attention_args {
  int32_t dtype; /* of q and out: CMPEXT3_F16 or CMPEXT3_BF16 */
  int32_t batch, heads, causal;
  float scale; /* positive, finite */
  int32_t len_q, len_k, total_q, total_k;
  const void* q;
  void* out;
  int64_t q_batch, q_token, q_head, out_batch, out_token, out_head;
  cmpext3_kv_cache cache;
  const int32_t* starts_q;
  const int32_t* starts_k;
  const int32_t* block_table;
  int64_t table_row;
  int32_t table_pages;
  const int32_t* seq_lens;
} cmpext3_attention_args;
/* Bytes of workspace (16-byte aligned, contents dead after the call) that the call needs. */
int64_t cmpext3_attention_workspace_size(const cmpext3_attention_args* args);
int cmpext3_attention(const cmpext3_attention_args* args, void* workspace, int64_t workspace_bytes, void* stream);
/* One-line description of the kernel, tile and split the call would run; host only. */
int cmpext3_attention_describe(const cmpext3_attention_args* args, char* buf, int buflen);

#ifdef __cplusplus
}
#endif

#endif /* CMPEXT3_ATTENTION_H */
