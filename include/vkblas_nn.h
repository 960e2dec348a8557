/*
 * vkblas_nn.h — what a training or serving step runs next to its GEMMs:
 * layer norm, the gated feed-forward projection and the output projection
 * with softmax cross entropy, each with its gradients.
 *
 * No reference counterpart: the reference intercepted the GEMMs alone and
 * left these to the framework above it.  Conventions are vkblas_ext.h's:
 * row-major matrices in device memory with leading dimensions in elements,
 * a HIP stream (NULL = null stream), asynchronous launches, no wait.
 *
 * Types: F32, F16 or BF16 throughout; sums, row statistics and
 * exponentials are fp32, and every result is rounded once, to nearest even.
 * Pointers need only their element's alignment; 16-byte aligned operands
 * with leading dimensions and K in whole 16-byte units are fastest.
 * M = 0 is a call on an empty batch: forward passes do nothing, weight
 * gradients get beta times what they held (zero for beta = 0).
 *
 * Weight gradients: dw = beta * dw + gradient, of dw_type, which is the
 * weight's type or F32 (a program's fp32 accumulators).  dw is read only
 * when beta != 0.  A gradient whose pointer is NULL is not computed.
 *
 * Workspace: calls that need one take their stream's workspace, as GEMMs that
 * split K do (vkblas_workspace_release frees it), and return VKBLAS_ERR_INIT
 * under stream capture; each function says when it needs one.  A call that would
 * use it for nothing but the partial sums of a K split then runs without the
 * split, as a GEMM does (products of up to 64 rows, the decode kernels', aside).
 *
 * Status: VKBLAS_OK; VKBLAS_ERR_PARAM (null pointer, zero size, leading
 * dimension shorter than its row, dimension above 2^31 - 1, unknown type or
 * activation), nothing launched; VKBLAS_ERR_INIT (no GPU, no workspace,
 * launch failure before an output was enqueued to be written);
 * VKBLAS_ERR_PARTIAL (a launch failed after that).
 */
#pragma once
#include "vkblas_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Layer norm of M rows of N: y = (x - mean) * rstd * w + b, with the row's
 * mean, and rstd = 1 / sqrt(variance + eps) (variance over N, about the mean).
 *   type: of x and y; w_type: of w and b, F32 or type
 *   w, b: N values, or NULL (ones, zeros)
 *   mean, rstd: M floats each, kept for the backward pass, or NULL
 * y may be x.  Needs no workspace.
 */
vkblas_status_t vkblas_layer_norm_async(
    vkblas_dtype_t type, vkblas_dtype_t w_type,
    uint32_t M, uint32_t N,
    const void* x, uint32_t ldx,
    const void* w, const void* b, float eps,
    void* y, uint32_t ldy,
    float* mean, float* rstd,
    void* stream);

/*
 * Its gradients, with xh = (x - mean) * rstd and g = dy * w:
 *   dx = rstd * (g - mean_n(g) - xh * mean_n(g * xh))
 *   dw = beta * dw + sum_m dy * xh,  db = beta * db + sum_m dy
 *   w: NULL = ones; mean, rstd: as the forward pass wrote them
 *   dx, dw, db: each NULL or computed; dw, db of g_type (w_type or F32)
 * dx may be dy or x.  Sums over rows run in an order that depends on M and N
 * alone: equal calls give equal bits.  Needs a workspace when dw or db is wanted
 * of more than 512 rows (1024 for N up to 4096), or for N below 8 or above 16384.
 */
vkblas_status_t vkblas_layer_norm_backward_async(
    vkblas_dtype_t type, vkblas_dtype_t w_type,
    uint32_t M, uint32_t N,
    const void* dy, uint32_t lddy,
    const void* x, uint32_t ldx,
    const void* w, const float* mean, const float* rstd,
    void* dx, uint32_t lddx,
    void* dw, void* db, vkblas_dtype_t g_type, float beta,
    void* stream);

/* Activation of the gated projection. */
typedef enum {
    VKBLAS_ACT_SILU = 0,       /* g / (1 + exp(-g))                          */
    VKBLAS_ACT_GELU = 1,       /* g (1 + erf(g / sqrt 2)) / 2                */
    VKBLAS_ACT_GELU_TANH = 2,  /* g (1 + tanh(sqrt(2/pi) (g + 0.044715 g^3))) / 2 */
    VKBLAS_ACT_RELU = 3        /* max(g, 0)                                  */
} vkblas_act_t;

/*
 * Gated feed-forward projection: [G | U] = x w^T, h = act(G) * U.
 *   x: M x K; w: 2N x K, rows 0 .. N-1 the gate's, N .. 2N-1 the up
 *   projection's; h: M x N; all of one type
 *   gu: NULL, or M x 2N of the same type: G and U, kept for the backward
 *   pass (h is computed from their fp32 values)
 * Needs no workspace for
 *  - up to 4 rows, K of at least 16 bytes; where rows lie off 16-byte units up to
 *    16 rows, or 32 for N of at least 2048;
 *  - more than 64 rows whose h has at least 96 tiles of 128 x 64 (200 in fp32), K
 *    in whole 16-byte units and all rows on whole lines of 128 bytes (fp32: on
 *    16-byte units).
 * Other calls may take one; most small ones (h of at most 256 tiles of 64 x 32, K up
 * to 2048) are one launch of small tiles and take none.
 */
vkblas_status_t vkblas_glu_async(
    vkblas_dtype_t type, vkblas_act_t act,
    uint32_t M, uint32_t N, uint32_t K,
    const void* x, uint32_t ldx,
    const void* w, uint32_t ldw,
    void* h, uint32_t ldh,
    void* gu, uint32_t ldgu,
    void* stream);

/*
 * Its gradients, from dh (M x N) and the kept gu:
 *   dG = dh * U * act'(G), dU = dh * act(G)
 *   dx = [dG | dU] w,  dw = beta * dw + [dG | dU]^T x
 *   dgu: NULL, or M x 2N of type: receives [dG | dU], rounded to type (the
 *   two products read it); may be gu itself.  NULL: kept in the workspace.
 *   dx: M x K or NULL; dw: 2N x K of dw_type or NULL
 * Takes a workspace for [dG | dU] (without dgu), for the sums of products that
 * split K, and for copies of operands that lie off 16-byte units or whole steps.
 */
vkblas_status_t vkblas_glu_backward_async(
    vkblas_dtype_t type, vkblas_act_t act,
    uint32_t M, uint32_t N, uint32_t K,
    const void* dh, uint32_t lddh,
    const void* gu, uint32_t ldgu,
    const void* x, uint32_t ldx,
    const void* w, uint32_t ldw,
    void* dgu, uint32_t lddgu,
    void* dx, uint32_t lddx,
    void* dw, uint32_t lddw, vkblas_dtype_t dw_type, float beta,
    void* stream);

/*
 * Softmax cross entropy of the logits z = x w^T, which are not kept:
 *   lse[m] = log sum_v exp(z[m][v]),  loss[m] = lse[m] - z[m][target[m]]
 *   x: M x K; w: V x K, of one type; target: M class indices
 *   target[m] == ignore_index: loss[m] = 0 (lse[m] is computed)
 *   any other target outside [0, V): loss[m] is NaN
 *   loss, lse: M floats each (loss may be NULL: then target may be NULL too)
 * Needs a workspace.
 */
vkblas_status_t vkblas_linear_xent_async(
    vkblas_dtype_t type,
    uint32_t M, uint32_t V, uint32_t K,
    const void* x, uint32_t ldx,
    const void* w, uint32_t ldw,
    const int64_t* target, int64_t ignore_index,
    float* loss, float* lse,
    void* stream);

/*
 * Its gradients from the rows' loss gradients dloss (M floats) and lse:
 *   D[m][v] = dloss[m] * (exp(z[m][v] - lse[m]) - [v == target[m]]), 0 for
 *   ignored rows, NaN for rows whose target is outside [0, V)
 *   dx = D w,  dw = beta * dw + D^T x
 * The logits are computed again in pieces of the vocabulary.  D is rounded
 * to type for the two products, divided by the largest finite |dloss| of the
 * rows that count (fp16: times 2^13 more, which keeps it in range), a factor
 * they take out again in fp32.  dloss of an ignored row may hold anything.
 *   dx: M x K or NULL; dw: V x K of dw_type or NULL
 * Needs a workspace.
 */
vkblas_status_t vkblas_linear_xent_backward_async(
    vkblas_dtype_t type,
    uint32_t M, uint32_t V, uint32_t K,
    const void* x, uint32_t ldx,
    const void* w, uint32_t ldw,
    const int64_t* target, int64_t ignore_index,
    const float* lse, const float* dloss,
    void* dx, uint32_t lddx,
    void* dw, uint32_t lddw, vkblas_dtype_t dw_type, float beta,
    void* stream);

#ifdef __cplusplus
}
#endif
