/*
 * glacier_cache.h -- C ABI of the paged key/value cache of
 * libglacier_attn.so: what a decoder needs between its q/k/v projections and
 * its O projection when it answers instead of training.
 *
 *   glacier_attn_cache_append   the new tokens' keys (rotated on the way) and
 *                               values into the pages; their queries rotated
 *                               in the same launch
 *   glacier_attn_cache_forward  attention of the new tokens over everything
 *                               their sequences have cached, one new token a
 *                               sequence (a step of an answer) or a chunk of
 *                               a prompt
 *
 * Per layer: glacier_proj_forward (q, k, v); for models that norm queries and
 * keys per head glacier_rmsnorm_qk_forward; glacier_attn_cache_append;
 * glacier_attn_cache_forward; glacier_proj_forward (O).  The reference trains
 * only: it leaves answering to its sibling package, so these calls have no
 * counterpart in its sources.
 *
 * The cache.  K and V pages are [n_pages][n_heads_kv][page_size][head_dim] in
 * the io dtype, page_stride elements from one page to the next (so that K and
 * V, or all layers, may share one allocation).  Sequence b's token at position
 * p lives in page page_table[b * table_stride + p / page_size], row
 * p % page_size.  An entry outside [0, n_pages), or a position at or past
 * max_pages * page_size, holds no key: appending drops the token, attention
 * passes over the keys.
 *
 * The batch.  Rows cu_tokens[b] .. cu_tokens[b+1] - 1 of q, k, v and out are
 * the new tokens of sequence b, and kv_lens[b] is its length with them, so its
 * i-th new token is at position kv_lens[b] - (cu_tokens[b+1] - cu_tokens[b])
 * + i.  A sequence may have no new token.  Rows at or past cu_tokens[n_seqs]
 * (a batch padded to a fixed size) change nothing and are not written.  cu_tokens,
 * kv_lens and page_table are device arrays, so a captured graph replays with
 * whatever they hold then; both calls are safe to capture: they allocate
 * nothing and do not wait.  K and V rows past a sequence's end may hold
 * anything, NaN included.
 *
 * The rotation turns pairs (i, i + head_dim / 2) by pos * theta^(-2i/head_dim),
 * with the angle reduced in 64 bits: exact to fp32 rounding at any position.
 * (glacier_attn_forward forms its angles in fp32 as the reference does, which
 * puts them off by up to pos * 2^-23 at far positions.)
 *
 * bf16 tensors: bf16 operands, fp32 sums and softmax; weights multiply V as two
 * bf16 terms, 16 bits of them.  fp32 tensors: fp32 throughout, whatever the
 * context's precision.  Results are
 * bitwise repeatable for one layout of the work (below: max_new, max_kv).  NaN
 * and infinities in a token's K or V reach only the rows that see the token.  Sums
 * of up to as many terms of V as there are keys stay within fp32 (|V| below 2^127
 * divided by their number).
 * Contexts, status codes and dtypes are those of glacier_attn.h; calls enqueue on
 * the context's stream.  Tensors are 16-byte aligned, q, k, v and out contiguous;
 * head_dim is a multiple of 8 up to 256.
 * One call takes fewer than 2^26 rows (tokens times its heads) and 2^22
 * sequences times KV heads.
 */
#ifndef GLACIER_CACHE_H
#define GLACIER_CACHE_H

#include "glacier_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct glacier_kv_cache {
  void *k_pages;        /* [n_pages][n_heads_kv][page_size][head_dim] (device) */
  void *v_pages;        /* as k_pages */
  int64_t page_stride;  /* elements between two pages of k_pages, and of v_pages; a multiple of 8 */
  int32_t n_pages;
  int32_t page_size;    /* tokens per page: a power of two, 16 to 1024 */
  int32_t n_heads_kv;
  int32_t head_dim;     /* a multiple of 8, at most 256 */
  int32_t io_dtype;     /* GLACIER_ATTN_IO_*: the pages and every tensor of the calls */
} glacier_kv_cache;

typedef struct glacier_cache_batch {
  const int32_t *cu_tokens;   /* device [n_seqs + 1], 0 = cu[0] <= ... <= cu[n_seqs] <= total_tokens */
  const int32_t *kv_lens;     /* device [n_seqs]: lengths with the new tokens */
  const int32_t *page_table;  /* device [n_seqs][max_pages], rows table_stride apart */
  int64_t table_stride;
  int32_t n_seqs;
  int32_t total_tokens;       /* rows of q, k, v and out */
  int32_t max_pages;
  int32_t max_new;            /* new tokens of the longest chunk, or 0 if not known (the tokens
                                 are then taken to be spread evenly over the sequences) */
  int32_t max_kv;             /* the longest kv_lens, or 0 (then what max_pages allows).  Both only
                                 steer how the work is laid out; results are right whatever they say */
} glacier_cache_batch;

/* Writes k (rotated when rope_freq_base > 0; 0: as it is, for keys that are
 * rotated already) and v, [total_tokens][n_heads_kv][head_dim], into the pages.
 * q [total_tokens][n_heads_q][head_dim], when not NULL, is rotated into q_rot,
 * which may be q; it needs rope_freq_base > 0.  n_heads_q is read only then.
 * Sequences may share pages that they only read; a page that takes new tokens
 * belongs to one of them.  K pages, V pages, k, v, q and q_rot share no memory
 * (but q_rot and q); pages of K and V may alternate. */
int glacier_attn_cache_append(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                              const glacier_cache_batch *batch, const void *k, const void *v,
                              float rope_freq_base, int32_t n_heads_q, const void *q, void *q_rot);

/* Bytes of device workspace glacier_attn_cache_forward needs for this cache
 * and batch (0 if it needs none, or if the arguments are not valid). */
size_t glacier_attn_cache_workspace(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                                    const glacier_cache_batch *batch, int32_t n_heads_q);

/* out[t][h] = sum_j softmax_j(q[t][h] . k_j / sqrt(head_dim)) v_j over the keys
 * 0 .. position of t of its sequence, h reading KV head h / (n_heads_q /
 * n_heads_kv).  q: rotated queries.  lse, when not NULL: [n_heads_q]
 * [total_tokens] fp32, the natural log-sum-exp of the scores.  A row without a
 * key gets 0 and -inf.  workspace: at least glacier_attn_cache_workspace bytes,
 * 256-byte aligned, the call's own until it has run (calls that overlap need
 * one each).  out may be q; out and lse lie outside the pages. */
int glacier_attn_cache_forward(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                               const glacier_cache_batch *batch, int32_t n_heads_q, const void *q,
                               void *out, float *lse, void *workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif /* GLACIER_CACHE_H */
