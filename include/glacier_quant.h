/*
 * glacier_quant.h -- C ABI of answering in 4 bits in libglacier_attn.so: a paged
 * key/value cache that holds keys and values in 4 bits, and products with base
 * weights held in 4 bits.
 *
 *   glacier_attn_qcache_append   as glacier_attn_cache_append: the new tokens' keys
 *                                (rotated on the way) and values into the pages,
 *                                quantised as they are written
 *   glacier_attn_qcache_read     the batch's tokens back from the pages
 *   glacier_attn_qcache_forward  as glacier_attn_cache_forward, over such pages
 *   glacier_proj_quant_pack      4-bit weights laid out for the products
 *   glacier_proj_quant_forward   as glacier_proj_forward, with such weights: the
 *                                step of an answer of a model whose frozen base
 *                                weights are in 4 bits, with the tuned adapters
 *
 * Per layer of a step: glacier_proj_quant_forward (q, k, v); for models that norm
 * queries and keys per head glacier_rmsnorm_qk_forward; glacier_attn_qcache_append;
 * glacier_attn_qcache_forward; glacier_proj_quant_forward (O).  The reference trains
 * only, so the cache's calls have no counterpart in its sources; its 4-bit base
 * products are tune_bwd.cu's gemm_q4_0_batch (:133).
 *
 * All calls enqueue on the context's stream, allocate nothing, do not wait and can
 * be captured; results are bitwise repeatable.  Contexts, status codes and dtypes
 * are those of glacier_attn.h, the batch that of glacier_cache.h.
 */
#ifndef GLACIER_QUANT_H
#define GLACIER_QUANT_H

#include "glacier_cache.h"
#include "glacier_qkv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- a paged cache in 4 bits -----------------------------------------------
 *
 * A token's head is held in groups of 32 columns: 4-bit numbers n and one fp16
 * scale s, standing for (n - 8) s.  With m the group's element of largest
 * magnitude (the positive one of two), s is m / -8 rounded to five significant
 * bits (ties to even) and kept within +-2688, and n = floor(x / s + 1/2) + 8 kept
 * within 0 .. 15.  So an element is off by at most half a step |s|, one near -m by
 * up to five quarters of one; magnitudes past 21504 are cut to it; where |m| is
 * below 2^-17 s has fewer bits, below 2^-22 it is zero.  What is held has at most eight
 * significant bits: it is exact in bf16, fp16 and fp32.  A group of zeros has
 * s = 0; one with a NaN or an infinity has s = NaN and reads back as NaN.  Keys
 * are rotated in 64 bits and rounded to fp32 before they are quantised.
 *
 * Pages.  A page of K, and one of V, is [n_heads_kv][18 G page_size] bytes, G the
 * groups of a head: 1, 2, 3, 4, 6 or 8, the least with 32 G >= head_dim (columns
 * past head_dim are held as zeros).  A head's part: 16 G page_size bytes of 32-bit
 * words, then 2 G page_size bytes of scales.  A word holds columns 8 x + 2 j in its
 * bits 4 j .. and 8 x + 2 j + 1 in its bits 16 + 4 j .., j = 0 .. 3.
 *   K  word (row 4 + c) G + i: columns 32 i + 8 c ..; scale row G + i: group i
 *   V  word (row / 4 4 G + r) 4 + row % 4: columns 8 r ..; scale (row / 4 G + i) 4
 *      + row % 4: group i
 * In glacier_kv_cache, page_stride counts bytes here (a multiple of 16), and
 * io_dtype is that of q, k, v and out.  The page table, kv_lens and cu_tokens are
 * used as in glacier_cache.h, with the same bounds; rows past a sequence's end
 * may hold anything. */

/* Bytes of a page of K (and of V), n_heads_kv 18 G page_size; 0 if the cache is
 * not valid (page_stride is not looked at). */
size_t glacier_attn_qcache_page_bytes(const glacier_kv_cache *cache);

/* glacier_attn_cache_append into 4-bit pages: k, v [total_tokens][n_heads_kv]
 * [head_dim] and q, q_rot [total_tokens][n_heads_q][head_dim] as there.  A page
 * that takes new tokens belongs to one sequence. */
int glacier_attn_qcache_append(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                               const glacier_cache_batch *batch, const void *k, const void *v,
                               float rope_freq_base, int32_t n_heads_q, const void *q, void *q_rot);

/* The batch's tokens (row i of sequence b: position kv_lens[b] - (cu_tokens[b + 1]
 * - cu_tokens[b]) + i) from the pages into k and v [total_tokens][n_heads_kv]
 * [head_dim], exactly.  With cu_tokens the running sum of kv_lens that is all of
 * every sequence.  Tokens without a page give zeros; rows behind the last sequence
 * are not written. */
int glacier_attn_qcache_read(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                             const glacier_cache_batch *batch, void *k, void *v);

/* Bytes of device workspace glacier_attn_qcache_forward needs (0 if it needs none,
 * or if the arguments are not valid). */
size_t glacier_attn_qcache_workspace(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                                     const glacier_cache_batch *batch, int32_t n_heads_q);

/* glacier_attn_cache_forward over 4-bit pages, which are read exactly.  fp32 tensors:
 * to fp32 rounding.  bf16 tensors: a score, and so lse, is an fp32 sum of terms (128
 * + n) s q and -136 s q, whose additions are off by 2^-24 of sums of up to 143 |s| |q|
 * each (random queries: the score by 2^-21 of its terms' length, as a root mean
 * square), and weights multiply V as two bf16 terms, 16 bits of them.  Queries may have
 * any finite size for which q k stays within fp32.  A NaN in the pages reaches only the
 * rows that see its token. */
int glacier_attn_qcache_forward(glacier_attn_ctx *ctx, const glacier_kv_cache *cache,
                                const glacier_cache_batch *batch, int32_t n_heads_q, const void *q,
                                void *out, float *lse, void *workspace, size_t workspace_bytes);

/* ---- products with 4-bit weights ------------------------------------------ */

/* Weights W [out][in] in groups of `group` columns of a row: W = (n - 8) s, or
 * (n - 8) s + o where there are offsets, n of 4 bits, s and o fp16. */
typedef struct glacier_quant_weights {
  int32_t out_features;  /* a multiple of 4 */
  int32_t in_features;   /* a multiple of 32 and of group, below 2^24 */
  int32_t group;         /* 32, 64 or 128 */
  int32_t offsets;       /* 0, or 1: weights have offsets */
} glacier_quant_weights;

/* Bytes of packed weights, below 2^31 (0 if w is not valid).  Their layout, rows padded to a
 * multiple of 16 and columns to one of 128 with zeros:
 *   [out / 16][in / 128][64] entries of four 32-bit words: word i of entry 16 c + r
 *     holds row r's columns 32 i + 8 c .. of the block, in a cache word's order
 *   [out / 16][in / 128][16][128 / group] scales, fp16
 *   the offsets alike, where there are any */
size_t glacier_proj_quant_bytes(const glacier_quant_weights *w);

/* Lays weights out: numbers [out][in / 2] (two to a byte, the even column in the
 * low half), scales and offsets [out][in / group] fp16, all on the device, into
 * packed (glacier_proj_quant_bytes bytes, 16-byte aligned). */
int glacier_proj_quant_pack(glacier_attn_ctx *ctx, const glacier_quant_weights *w, const void *numbers,
                            const void *scales, const void *offsets, void *packed);

typedef struct glacier_quant_proj_desc {
  int32_t total_tokens;  /* T (may be 0) */
  int32_t in_features;   /* a multiple of 32 and of group */
  int32_t group;         /* of every projection's weights */
  int32_t offsets;       /* likewise */
  int32_t rank;          /* 1..GLACIER_PROJ_MAX_RANK when any adapter is given */
  int32_t io_dtype;      /* GLACIER_ATTN_IO_*: x and y.  F32: to fp32 rounding; BF16: fp32 sums
                            of terms (128 + n) s x and -136 s x, whose additions are off by
                            2^-24 of sums of up to 143 |s| |x| each; each output rounded once */
} glacier_quant_proj_desc;

/* Bytes of device workspace glacier_proj_quant_forward needs (0 if it needs none,
 * or if the arguments are not valid). */
size_t glacier_proj_quant_workspace(const glacier_quant_proj_desc *desc, const glacier_lora_proj *proj,
                                    int n_proj);

/* y_p = x W_p^T + bias_p + s_p (x A_p) B_p for n_proj (1..GLACIER_PROJ_MAX_PROJ)
 * projections of x [T][in]: as glacier_proj_forward, with proj[p].w the packed
 * weights.  x, y, lora_a, lora_b and w 16-byte aligned; outputs share no memory
 * with inputs or each other.  workspace: at least glacier_proj_quant_workspace
 * bytes, 256-byte aligned, the call's own until it has run.  Sums of eight (bf16
 * tensors: 143) times a group's |x| pass through fp32: a token for which they pass
 * its range, or with a value that is not finite, gets outputs that are not finite;
 * no other token is touched. */
int glacier_proj_quant_forward(glacier_attn_ctx *ctx, const glacier_quant_proj_desc *desc, const void *x,
                               const glacier_lora_proj *proj, int n_proj, void *workspace,
                               size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif /* GLACIER_QUANT_H */
