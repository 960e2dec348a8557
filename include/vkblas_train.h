/*
 * vkblas_train.h — the two ends of a training step around the operators of
 * vkblas_nn.h: the tokens' embedding, and the losses beside the plain cross
 * entropy, distillation from a teacher's top logits on the output projection
 * and the clipped policy loss on token log probabilities; each with its
 * gradient.
 *
 * No reference counterpart: the reference intercepted the GEMMs alone.
 * Conventions are vkblas_nn.h's: row-major matrices in device memory with
 * leading dimensions in elements, pointers of their element's alignment, a HIP
 * stream, asynchronous launches; F32, F16 or BF16 with sums, exponentials and
 * row statistics in fp32 or more and one rounding of each result, to nearest
 * even; weight gradients dw = beta * dw + gradient, dw read only when beta != 0;
 * a gradient whose pointer is NULL is not computed; an empty batch (M or B of 0)
 * does nothing but scale dw; its workspaces, also under stream capture, and its
 * status codes (a constant outside its range is VKBLAS_ERR_PARAM too).
 */
#pragma once
#include "vkblas_nn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Embedding: y[m] = scale * w[ids[m]], M rows of N out of a w of V x N.
 *   type: of y; w_type: of w, F32 or type
 *   ids: M token ids.  ids[m] == pad_id: a row of zeros (pad_id of -1 where a
 *   program pads with nothing of its own); any other id outside [0, V): a row
 *   of NaN, w is not read
 * y is not w.  Needs no workspace.
 */
vkblas_status_t vkblas_embedding_async(
    vkblas_dtype_t type, vkblas_dtype_t w_type,
    uint32_t M, uint32_t V, uint32_t N,
    const int64_t* ids, int64_t pad_id,
    const void* w, uint32_t ldw, float scale,
    void* y, uint32_t ldy,
    void* stream);

/*
 * Its gradient, over the whole vocabulary:
 *   dw[v] = beta * dw[v] + scale * sum of dy[m] over the m with ids[m] == v
 * Padding and ids outside [0, V) add nothing.  dw (V x N) is of dw_type, type or
 * F32.  beta = 1 reads and writes the rows of the tokens that occur alone: the
 * gradient of a w that is the output projection's too (tied weights) adds to
 * what vkblas_linear_xent_backward_async left there.
 * The rows of a token are summed in fp32 in an order that depends on ids, M, V, N
 * and the types alone: equal calls give equal bits.  Needs a workspace for more
 * than VKBLAS_EMBEDDING_SMALL tokens or a gradient of more than
 * VKBLAS_EMBEDDING_SMALL_BYTES (V * N of dw_type), or N above 2^24 - 256.
 */
#define VKBLAS_EMBEDDING_SMALL 4096
#define VKBLAS_EMBEDDING_SMALL_BYTES ((uint64_t)64 << 20)
vkblas_status_t vkblas_embedding_backward_async(
    vkblas_dtype_t type,
    uint32_t M, uint32_t V, uint32_t N,
    const int64_t* ids, int64_t pad_id,
    const void* dy, uint32_t lddy, float scale,
    void* dw, uint32_t lddw, vkblas_dtype_t dw_type, float beta,
    void* stream);

/*
 * Distillation from a teacher's top logits, for the student's logits
 * z = x w^T, which are not kept.  With T = temperature, q = the softmax of
 * t[m][j] / T over the row's entries j, and p = the softmax of z[m][v] / T over
 * all V classes:
 *   lse[m] = log sum_v exp(z[m][v] / T)
 *   loss[m] = T^2 * sum_j q_j (log q_j - log p[top[m][j]])
 *   x: M x K; w: V x K, of one type
 *   T > 0, T^2 and log2(e) / T within fp32's range; the loss's error is T^2 times
 *   that of log-sum-exps in fp32
 *   top: M x n_top classes (leading dimension ldtop); t: the teacher's logits
 *   there, M x n_top of t_type, F32 or type; n_top up to VKBLAS_DISTILL_TOP
 *   top[m][j] < 0: the entry is absent, whatever t holds there; a t of -inf
 *   is a probability of 0.  A row whose entries are all so is not counted:
 *   loss 0 (lse is computed), no gradient
 *   a class of V or more: loss[m] and the row's gradient are NaN
 *   a class that occurs twice in a row has both entries' probability
 *   z_top: M x n_top floats (packed), z[m][top[m][j]] kept for the backward
 *   pass; 0 for absent entries, NaN for classes past V
 * Needs a workspace.
 */
#define VKBLAS_DISTILL_TOP 1024
vkblas_status_t vkblas_linear_distill_async(
    vkblas_dtype_t type,
    uint32_t M, uint32_t V, uint32_t K,
    const void* x, uint32_t ldx,
    const void* w, uint32_t ldw,
    uint32_t n_top, const int64_t* top, uint32_t ldtop,
    vkblas_dtype_t t_type, const void* t, uint32_t ldt, float temperature,
    float* loss, float* lse, float* z_top,
    void* stream);

/*
 * Its gradients from the rows' loss gradients dloss (M floats), lse and z_top:
 *   D[m][v] = T * dloss[m] * (p[v] - sum of q_j over the j with top[m][j] == v)
 *   dx = D w,  dw = beta * dw + D^T x
 * D is scaled and rounded as vkblas_linear_xent_backward_async's.  dloss of a row
 * that is not counted may hold anything (its x adds 0 times itself to dw).
 *   dx: M x K or NULL; dw: V x K of dw_type or NULL
 * Needs a workspace.
 */
vkblas_status_t vkblas_linear_distill_backward_async(
    vkblas_dtype_t type,
    uint32_t M, uint32_t V, uint32_t K,
    const void* x, uint32_t ldx,
    const void* w, uint32_t ldw,
    uint32_t n_top, const int64_t* top, uint32_t ldtop,
    vkblas_dtype_t t_type, const void* t, uint32_t ldt, float temperature,
    const float* lse, const float* z_top, const float* dloss,
    void* dx, uint32_t lddx,
    void* dw, uint32_t lddw, vkblas_dtype_t dw_type, float beta,
    void* stream);

/* How the policy loss weighs a token that counts. */
typedef enum {
    VKBLAS_REDUCE_TOKENS = 0,     /* 1 / the tokens of the batch                */
    VKBLAS_REDUCE_SEQUENCES = 1,  /* 1 / (its sequence's tokens * the sequences
                                     that have any)                             */
    VKBLAS_REDUCE_SUM = 2         /* 1                                          */
} vkblas_reduce_t;

/*
 * Clipped policy loss with a KL term over a padded batch of B sequences of T
 * tokens, from the log probabilities of the tokens taken (vkblas_linear_xent_async's
 * losses are their negatives).  For a token with r = exp(logp - old_logp),
 * d = ref_logp - logp and the advantage A:
 *   L = -min(r A, c A) + kl_coef * (exp(d) - d - 1),
 *   c = r held within [1 - clip_low, 1 + clip_high]
 *   logp, old_logp, ref_logp: B x T, leading dimensions ldp, ldo, ldr.
 *   ref_logp: NULL = no KL term (with kl_coef 0 it is measured only)
 *   adv: A[b][t] = adv[b * ldadv + t * adv_step]; adv_step 1, or 0 where a
 *   sequence has one advantage
 *   mask: B x T bytes, 0 = the token does not count, whatever the arrays hold
 *   there; NULL = all count
 *   clip_low, clip_high >= 0 (infinite: no such bound), kl_coef finite
 *   norm: B floats, the weight of a token of each sequence (vkblas_reduce_t),
 *   0 for a sequence without any; kept for the backward pass
 *   stats: 4 floats, sums over the tokens that count, by weight: of L (the
 *   loss), of exp(d) - d - 1, of the tokens whose bound was taken (c A < r A), of r
 * Which side of a bound r lies on is decided in fp64.  A token's terms are fp32,
 * and so are the sums of four tokens that a lane takes at once; those are added
 * up in fp64.  r and exp(d) past fp32's range are infinite; an advantage of 0
 * takes no part in L whatever r is, unless logp - old_logp is not finite.
 * Needs a workspace for more than VKBLAS_POLICY_SMALL tokens (B * T, a sequence's
 * rounded up to 256).
 */
#define VKBLAS_POLICY_SMALL 4096
vkblas_status_t vkblas_policy_loss_async(
    vkblas_reduce_t reduce, uint32_t B, uint32_t T,
    const float* logp, uint32_t ldp,
    const float* old_logp, uint32_t ldo,
    const float* ref_logp, uint32_t ldr,
    const float* adv, uint32_t ldadv, uint32_t adv_step,
    const uint8_t* mask, uint32_t ldmask,
    float clip_low, float clip_high, float kl_coef,
    float* stats, float* norm,
    void* stream);

/*
 * Its gradient, dlogp[b][t] = dloss[0] * norm[b] * dL/dlogp (dloss one float in
 * device memory, of stats[0]); 0 where the token does not count:
 *   dL/dlogp = -A r [r A <= c A] + kl_coef * (1 - exp(d))
 * A dloss of 0 gives zeros where the inputs are finite, whatever r and exp(d) are.
 * dlogp (B x T) may be logp, with its leading dimension.  Needs no workspace.
 */
vkblas_status_t vkblas_policy_loss_backward_async(
    uint32_t B, uint32_t T,
    const float* logp, uint32_t ldp,
    const float* old_logp, uint32_t ldo,
    const float* ref_logp, uint32_t ldr,
    const float* adv, uint32_t ldadv, uint32_t adv_step,
    const uint8_t* mask, uint32_t ldmask,
    float clip_low, float clip_high, float kl_coef,
    const float* norm, const float* dloss,
    float* dlogp, uint32_t lddp,
    void* stream);

#ifdef __cplusplus
}
#endif
