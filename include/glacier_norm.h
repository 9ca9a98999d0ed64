/*
 * glacier_norm.h -- C ABI of the residual add and RMSNorm either side of the
 * attention sub-block in libglacier_attn.so, forward and backward, on device
 * tensors.  With glacier_proj_* (glacier_qkv.h) for the O projection and its
 * LoRA adapter, the whole path from the attention output to the FFN input,
 * and back, stays in HBM.
 *
 *   forward   x1 = x + delta,  y = RMSNorm(x1) weight
 *             (y_i = (x1_i r) weight_i,  r = 1 / sqrt(mean_i x1_i^2 + eps))
 *   backward  dx = RMSNormBackward(dy; x, weight) + d_residual
 *             (dx_i = r weight_i dy_i - (r^3 / n) x_i sum_j weight_j dy_j x_j)
 *
 * Replaces ElementwiseKernels.RMSNorm / RMSNormBackward and TensorOps.Add
 * (Glacier.Tensor 1.1.0) at the block's call sites
 * (src/Glacier.Tune/Model/TransformerBlock.cs):
 *   :318        norm1X = RMSNorm(x)                      forward, delta NULL
 *   :505-506    x1 = x + OProj(attnOut); :524 norm2X = RMSNorm(x1)
 *                                                        forward, delta = OProj output
 *   :579        output = x1 + downOut (normalised by the next block's :318)
 *                                                        forward, delta = downOut
 *   :672, :677  dX1 = dOutput + RMSNormBackward(dNorm2X, X1)
 *                                                        backward, d_residual = dOutput
 *   :827, :836  dX = dX1 + RMSNormBackward(dNorm1X, x)   backward, d_residual = dX1
 *   :751, :759  per-head Q/K norms in place (rows = tokens x heads, n = head_dim)
 *
 * Layouts (row-major): x, delta, x1, y, dy, d_residual, dx [rows][n] in the
 * io dtype; weight, d_weight [n] fp32.  Sums and the norm are fp32.  The
 * contexts, status codes and dtype constants are those of glacier_attn.h; calls
 * enqueue on the context's stream.
 */
#ifndef GLACIER_NORM_H
#define GLACIER_NORM_H

#include "glacier_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* widest normalised row */
#define GLACIER_NORM_MAX_N 8192

typedef struct glacier_norm_desc {
  int32_t rows;      /* tokens, or tokens x heads for a per-head norm (may be 0) */
  int32_t n;         /* normalised width: a multiple of 4, at most GLACIER_NORM_MAX_N */
  int32_t io_dtype;  /* GLACIER_ATTN_IO_F32 or GLACIER_ATTN_IO_BF16 */
  float eps;         /* rms_norm_eps, finite and >= 0 */
} glacier_norm_desc;

/* x1 = x + delta and y = RMSNorm(x1) weight.  delta NULL: y = RMSNorm(x)
 * weight, and x1 is not written (may be NULL).  With delta, x1 is required
 * (the backward takes it as x); in the bf16 io dtype the norm is taken of x1
 * as stored.  y may alias x or delta; x1 may alias x. */
int glacier_rmsnorm_forward(glacier_attn_ctx *ctx, const glacier_norm_desc *desc, const void *x,
                            const void *delta, const float *weight, void *x1, void *y);

/* dx = RMSNormBackward(dy; x, weight) + d_residual (NULL: nothing added),
 * overwritten; x is the forward's normalised input (x1 there).  d_weight
 * (NULL: not formed, as at every reference call site) is accumulated (+=).
 * dx may alias dy or d_residual. */
int glacier_rmsnorm_backward(glacier_attn_ctx *ctx, const glacier_norm_desc *desc, const void *dy,
                             const void *x, const float *weight, const void *d_residual, void *dx,
                             float *d_weight);

/* ---- queries and keys of one layer --------------------------------------- */

/* The per-head norms of a layer's queries and keys with the position rotation
 * in the same pass:
 *   forward   y = R(pos) (x r w),  r = 1 / sqrt(mean_i x_i^2 + eps) per token and head
 *   backward  g = R(-pos) dy,  dx = r w g - (r^3 / D) x sum_j w_j g_j x_j,
 *             d_weight += sum over tokens and heads of g x r
 * (TransformerBlock.cs:413, :421, :751, :759, and the rotation of the call that
 * follows them).  R turns the pairs (i, i + D/2) by pos * theta^(-2i/D), the
 * angle reduced in 64 bits; rope_freq_base 0 leaves it out (for
 * glacier_attn_forward, which rotates by itself).  The sums are fp32, and every
 * result is rounded once. */
typedef struct glacier_rmsnorm_qk_desc {
  int32_t total_tokens;  /* T (may be 0), at most 2^26 - 4 */
  int32_t n_heads_q;     /* q [T][n_heads_q][D] */
  int32_t n_heads_kv;    /* k [T][n_heads_kv][D] */
  int32_t head_dim;      /* D: a multiple of 8, at most 256 */
  int32_t io_dtype;      /* GLACIER_ATTN_IO_F32 or GLACIER_ATTN_IO_BF16 */
  float eps;             /* finite and >= 0 */
  float rope_freq_base;  /* theta, or 0 for no rotation */
} glacier_rmsnorm_qk_desc;

/* q_weight, k_weight [D] fp32; positions: device int32 [T], or NULL for
 * 0 .. T - 1 (not read without a rotation).  q_out may be q, k_out may be k. */
int glacier_rmsnorm_qk_forward(glacier_attn_ctx *ctx, const glacier_rmsnorm_qk_desc *desc,
                               const void *q, const void *k, const float *q_weight,
                               const float *k_weight, const int32_t *positions, void *q_out,
                               void *k_out);

/* Bytes of device workspace the backward needs when it forms weight gradients
 * (0 if the arguments are not valid). */
size_t glacier_rmsnorm_qk_workspace(const glacier_rmsnorm_qk_desc *desc);

/* q, k: the forward's inputs.  dq, dk are overwritten and may be dq_out, dk_out.
 * dq_weight, dk_weight [D] fp32 are accumulated (+=), each formed only when not
 * NULL; then workspace holds at least glacier_rmsnorm_qk_workspace bytes,
 * 256-byte aligned, the call's own until it has run. */
int glacier_rmsnorm_qk_backward(glacier_attn_ctx *ctx, const glacier_rmsnorm_qk_desc *desc,
                                const void *dq_out, const void *dk_out, const void *q,
                                const void *k, const float *q_weight, const float *k_weight,
                                const int32_t *positions, void *dq, void *dk, float *dq_weight,
                                float *dk_weight, void *workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif /* GLACIER_NORM_H */
