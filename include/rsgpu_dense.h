/*
 * rsgpu_dense.h -- C-ABI of librsgpu's dense operators over factor tables (device pointers).  Contexts, status codes
 * and errors are rsgpu.h's.
 *
 * Not functions of the reference: what a model with user and item factor tables needs to be trained for ranking
 * over the whole catalogue and to answer with the whole catalogue.
 *
 * All matrices are row-major device memory of ctx's device with a row stride (ld, in elements) of at least their
 * columns; element types RS_TYPE_*.  A call enqueues its kernels on `stream` (NULL: the ctx stream,
 * RS_STREAM_DEFAULT: the device's default stream) and returns without waiting: it synchronises nothing, allocates
 * nothing, keeps nothing, and may be captured into a graph.
 * `ws` is device scratch of at least the bytes that the operator's _workspace call gives (16-byte aligned); it is
 * free for other use once the call's kernels have run, and two calls that may overlap need a workspace each.  The
 * caller's current device is put back before a call returns.  Calls whose sizes leave nothing to do return RS_OK
 * without a launch.  Sums are held in fp32, int32 or fp64 and each output is rounded once; results do not depend on
 * timing (no floating-point atomics).  Outputs and ws overlap neither the inputs nor each other.  n_factors up to
 * RS_DENSE_MAX_FACTORS. */
#ifndef RSGPU_DENSE_H
#define RSGPU_DENSE_H

#include "rsgpu.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RS_TYPE_F32 0
#define RS_TYPE_BF16 1
#define RS_TYPE_F16 2
#define RS_DENSE_MAX_FACTORS 512
/* `stream` value of the device's default (null) stream, which NULL does not name here */
#define RS_STREAM_DEFAULT ((void*)1)

/* Softmax cross entropy of every row of H (n_rows x n_factors: users' vectors) against the whole catalogue W
 * (n_items x n_factors), without keeping the logits:
 *   l_nv = h_n . w_v + bias_v      lse_n = log sum_v exp(l_nv)      loss_n = lse_n - l_{n, target_n}
 * and, where dH, dW and dbias are given (all three or none), the gradient of sum_n weight_n loss_n:
 *   c_nv = weight_n (exp(l_nv - lse_n) - [v = target_n])   dH_n = sum_v c_nv w_v   dW_v = sum_n c_nv h_n   dbias_v = sum_n c_nv
 * H, W, dH, dW have the element type `type`; bias, weight, loss, lse and dbias are fp32; target int32.
 *   bias NULL: zeros.  bias_v = -inf withdraws item v: it takes no part in any row, whatever its row of W holds (NaN
 *     included), and its rows of dW and dbias are zero.
 *   weight NULL: ones.  It is read for gradients only.
 *   target outside [0, n_items) (-1: unknown): the row takes no part, whatever its row of H and its weight hold;
 *     loss, lse and its row of dH are zero.
 *   Every item withdrawn: lse -inf, loss 0, no gradient.  target withdrawn, others not: lse as defined, loss +inf,
 *     no gradient from that row.
 *   Finite biases are held to +-2^120: the type's lowest value is no withdrawal.
 * The products run on fp16, each matrix scaled by a power of two from its largest finite element, which may be of any
 * size: RS_TYPE_F32 as pairs (hi + lo), so an element is off by at most 2^-23 of itself or 2^-38 of the matrix's largest
 * element, whichever is more, and the product lo lo (2^-22 at most) is left out; RS_TYPE_BF16 exactly down to 2^-27 of
 * the largest, and to 2^-38 of it below; RS_TYPE_F16 as it is.  Logits beyond fp32's range have no defined outputs.
 * Coefficients c_nv are rounded to 11 bits before they meet a bf16 matrix, to 22 otherwise, or to 2^-32 (dH; 2^-25 where a
 * row's logits pass 22700) and 2^-33 (dW) of the largest so far in the same sum, whichever is more: each row of dW keeps
 * its precision however improbable its item and small the weights.  A probability below 2^-126 counts as zero.  The
 * target's coefficient is minus the sum of the row's others: the gradients of a row keep their precision where its
 * target's probability is near one, as does its loss.
 * n_rows and n_items from 1 to 2^31 - 1025 (or both 0). */
int rs_softmax_ce_workspace(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_items, int32_t n_factors, int32_t with_grad,
                            int64_t* bytes);
int rs_softmax_ce(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_items, int32_t n_factors, const void* H, int64_t ldh,
                  const void* W, int64_t ldw, const float* bias, const int32_t* target, const float* weight,
                  float* loss, float* lse, void* dH, int64_t lddh, void* dW, int64_t lddw, float* dbias,
                  void* ws, int64_t ws_bytes, void* stream);

/* Rows in 8 bits with a scale each: scale_r = max_c |x_rc| * (1/127), both factors and the product in fp32,
 * q_rc = x_rc / scale_r to the nearest integer, ties to even, decided on the exact quotient, held to |q| <= 127 (a
 * subnormal scale may be rounded down so far that the quotient passes it).  A row of zeros, or whose scale underflows
 * to 0, has scale 0 and q 0; a row with an infinity or NaN has scale NaN and q 0, so that all its products are NaN.
 * X of `type`, q int8 with row stride ldq (bytes); columns past n_cols are left as they are.  n_cols >= 1. */
int rs_quantize_rows(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_cols, const void* X, int64_t ldx, int8_t* q,
                     int64_t ldq, float* scale, void* stream);

/* int8 product with a scale per row of A (a user, a token) and per row of B (an item, a channel):
 *   C_mn = a_scale_m * b_scale_n * sum_k A_mk B_nk + row_bias_m + col_bias_n
 * A (m x k), B (n x k) int8, any value, any alignment and stride (rows of 16-byte multiples at 16-byte addresses are
 * read fastest); the sums are exact in int32 (k <= RS_I8_MAX_K); the rest is fp32, the two scales' product first (where
 * that is no normal number, C has its precision), C of out_type rounded once.
 * row_bias, col_bias may be NULL.  An entry of col_bias of -inf gives -inf scores (a withdrawn item).  k >= 1. */
#define RS_I8_MAX_K 65536
int rs_i8_matmul(rs_ctx* ctx, int64_t m, int64_t n, int64_t k, const int8_t* A, int64_t lda, const float* a_scale,
                 const int8_t* B, int64_t ldb, const float* b_scale, const float* row_bias, const float* col_bias,
                 int32_t out_type, void* C, int64_t ldc, void* stream);

/* The orthogonalised form of an update G (rows x cols) of a factor table, by `steps` Newton-Schulz products:
 *   X_0 = G / |G|_F      X_{j+1} = a X_j + (b A_j + c A_j^2) X_j,  A_j = X_j X_j^T      X = X_steps
 * (for rows > cols the same with A_j = X_j^T X_j on the other side): every singular value s of X_0 becomes
 * p(p(..p(s))), p(s) = a s + b s^3 + c s^5; (3.4445, -4.7750, 2.0315) in 5 steps brings all but the smallest near 1.
 * G = 0 gives X = 0.  G and X have the element type `type`; X may be G itself (same pointer and stride; the
 * shorter side at most 256), otherwise they must not overlap.  The shorter side is at most RS_DENSE_MAX_FACTORS,
 * 1 <= steps <= RS_ORTHO_MAX_STEPS.
 * The polynomials are formed on the shorter side's Gram matrix, so the table is read twice and written once.  The Gram
 * matrix of RS_TYPE_F32 with at most 2048 long-side rows is fp64; otherwise it is a sum of fp16 products in fp32, joined
 * in fp64 (RS_TYPE_F32: of pairs, so an element is off by at most 2^-23 of itself or 2^-37 of the largest element near
 * it, whichever is more; fewer bits below 2^-114); the polynomials are fp64.  The last product takes an fp32 element to
 * 2^-23 of itself or 2^-49 of |G|, a bf16 or fp16 one to 2^-38 of |G|, its sums are fp32.  An infinity or NaN in G makes
 * all of X NaN.  ((3.4445, -4.7750, 2.0315) are the published coefficients of the orthogonalised-momentum optimiser.) */
#define RS_ORTHO_MAX_STEPS 16
int rs_orthogonalize_workspace(rs_ctx* ctx, int64_t rows, int64_t cols, int64_t* bytes);
int rs_orthogonalize(rs_ctx* ctx, int32_t type, int64_t rows, int64_t cols, const void* G, int64_t ldg, int32_t steps, double a,
                     double b, double c, void* X, int64_t ldx, void* ws, int64_t ws_bytes, void* stream);

/* ---- the operators on a plan's resident factors (host arrays, as rs_svd_plan_predict) -------------------------- */

/* One training step for ranking: n interactions (inner user, inner item; -1 or out of range = unknown, left out), the
 * loss is the mean over the m known ones of the softmax cross entropy of p_u . q_i + b_i against all items (GlobalBias and
 * b_u are the same for every item and play no part).  With g the gradient of that mean:
 *   p_u -= lr (g_pu + reg (c_u / m) p_u) for every user of the batch, c_u its interactions in it (a user may come several
 *     times: its gradients are added in batch order)
 *   b_i -= lr g_bi
 *   Q   -= q_lr (O + reg Q), O = rs_orthogonalize(g_Q) with 5 steps of (3.4445, -4.7750, 2.0315)
 * *loss (may be NULL): the mean loss before the step; NaN, and nothing changed, where no interaction is known.  A step
 * that would make a finite factor or bias infinite or NaN (a logit that is not finite does) changes nothing either:
 * RS_ERR_NUMERIC, *loss NaN.  The call waits for the step.  Its scratch on the device stays with the plan, grown
 * to its largest call: the gradient of the item table (twice where n_items and n_factors both pass 256), what
 * rs_softmax_ce_workspace asks for fp32 with gradients, and the batch's rows (4096 x 3706 x 100: 41 MB; 1024 x 1e6 x 256:
 * 2.1 GB).
 * A plan joined to a group is refused (RS_ERR_UNSUPPORTED): its factors are replicas.  n <= 2^20. */
int rs_svd_plan_rank_step(rs_svd_plan* plan, int64_t n, const int32_t* users, const int32_t* items, double lr, double q_lr,
                          double reg, double* loss);

/* Scores of n users (inner ids, -1 = unknown) against all items, out[r][i] = GlobalBias + b_u + b_i + p_u . q_i in fp32 (n x
 * n_items, host), the products in 8 bits: p_u and q_i by rs_quantize_rows (their scales s_p, s_q), so a score is off by at
 * most sum_f (s_p |q_f| + s_q |p_f|) / 2 + s_p s_q / 4 and fp32 rounding.  Unknown users: GlobalBias + b_i (svd.go:39-48).
 * The item table is quantised once a call.  Scratch on the device, kept with the plan as rank_step's: the 8-bit table
 * and up to 256 MiB of scores. */
int rs_svd_plan_score_items(rs_svd_plan* plan, int64_t n, const int32_t* users, float* out);

#ifdef __cplusplus
}
#endif

#endif /* RSGPU_DENSE_H */
