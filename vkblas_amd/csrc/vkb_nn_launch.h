/*
 * vkb_nn_launch.h — internal C ABI between the host side of the operators in
 * vkblas_nn.h (nn.c) and their gfx950 kernels.  As vkb_launch.h: plain
 * pointers and sizes, element types VKB_T_*, every launcher enqueues on the
 * stream and returns 0 or a hipError_t value.
 */
#pragma once
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Layer norm (layer_norm.hip).  The backward pass writes its partial sums of
 * dw and db to part, vkb_layer_norm_parts rows of 2 N floats (dw's N, then
 * db's), and vkb_launch_layer_norm_reduce adds them up. */
int vkb_launch_layer_norm(int type, int w_type, uint32_t M, uint32_t N, const void* x, int64_t ldx, const void* w,
                          const void* b, float eps, void* y, int64_t ldy, float* mean, float* rstd, void* stream);
uint32_t vkb_layer_norm_parts(int type, uint32_t M, uint32_t N);
/* dx, dw and db (NULL: not) of few rows in one launch, without partial sums;
 * not for vkb_layer_norm_long rows, nor dx in dy's or x's place along with dw or
 * db */
int vkb_launch_layer_norm_few(int type, int w_type, uint32_t M, uint32_t N, const void* dy, int64_t lddy, const void* x,
                              int64_t ldx, const void* w, const float* mean, const float* rstd, void* dx, int64_t lddx,
                              void* dw, void* db, int g_type, float beta, void* stream);
int vkb_layer_norm_long(uint32_t N);   /* rows past a workgroup's registers */
int vkb_launch_layer_norm_backward(int type, int w_type, uint32_t M, uint32_t N, const void* dy, int64_t lddy,
                                   const void* x, int64_t ldx, const void* w, const float* mean, const float* rstd,
                                   void* dx, int64_t lddx, float* part, void* stream);
int vkb_launch_layer_norm_reduce(const float* part, uint32_t parts, uint32_t N, void* dw, void* db, int g_type,
                                 float beta, void* stream);

/* C = beta * C on M x N (a gradient over an empty batch). */
int vkb_launch_scale(int type, uint32_t M, uint32_t N, void* C, int64_t ldc, float beta, void* stream);

/* Copies (pad.hip) between a program's S matrices of M x N below each other
 * (leading dimension ld) and the workspace, one launch for all of a call's.
 * pad: to S of Mp x Np, Np a multiple of 16 bytes, zero past M and N; all of
 * type.  With scale, also the device scalars of products of a gradient that
 * is divided by the largest finite |dloss| of the M rows that count (target in
 * [0, V) and not ignore: another row's loss gradient, whatever it holds, is no
 * part of D): scal[0] = s = 1 / max |dloss| (fp16: 2^13 times that; a
 * largest outside 1e-33 .. 8e37 counts as that end), scal[1] = 1 / s, scal[2] = beta,
 * scal[3] = 1, scal[4] = 0. */
/* ... or found by the kernels that compute D themselves (find; M of at most
 * VKB_SCALE_ROWS), which saves the launch where there are no copies. */
#define VKB_SCALE_ROWS 1024u
typedef struct vkb_scale {
    float* scal;                     /* NULL: no scale */
    float beta;
    int find;
    uint32_t M, V;
    const float* dloss;
    const int64_t* target;
    int64_t ignore;
} vkb_scale;
#define VKB_PAD_JOBS 3
typedef struct vkb_pad_job {
    const void* src;
    void* dst;
    int64_t ld;
    uint32_t S, M, N, Mp, Np;
} vkb_pad_job;
int vkb_launch_pad(int type, const vkb_pad_job* jobs, int n, const vkb_scale* scale, void* stream);   /* scale NULL: none */
/* unpad (up to 2): dst = beta * dst + src, src in rows of ldp and matrices of
 * Mp rows; type and out_type fp32 or one and the same 16-bit type */
typedef struct vkb_unpad_job {
    const void* src;
    void* dst;
    int64_t ldp, ldc;
    uint32_t S, M, N, Mp;
    int type, out_type;
    float beta;
} vkb_unpad_job;
int vkb_launch_unpad(const vkb_unpad_job* jobs, int n, void* stream);

/* Gated projection (glu.hip), from projections computed before:
 * h = act(G) * U from z = [G | U] in fp32, and gu = z rounded (NULL: not
 * stored); and [dG | dU] from dh and gu, Np >= N columns each on Mp >= M
 * rows, zero past N and M. */
int vkb_launch_glu_join(int type, int act, uint32_t M, uint32_t N, const float* z, int64_t ldz, void* h, int64_t ldh,
                        void* gu, int64_t ldgu, void* stream);
int vkb_launch_glu_join_backward(int type, int act, uint32_t M, uint32_t N, const void* dh, int64_t lddh,
                                 const void* gu, int64_t ldgu, void* dgu, int64_t lddgu, uint32_t Mp, uint32_t Np,
                                 void* stream);
/* ... of a small call in one launch, product and all (glu_direct.hip) */
int vkb_glu_direct_fits(int type, uint32_t M, uint32_t N, uint32_t K, uint32_t ldx, uint32_t ldw);
int vkb_launch_glu_direct(int type, int act, uint32_t M, uint32_t N, uint32_t K, const void* x, uint32_t ldx,
                          const void* w, uint32_t ldw, void* h, uint32_t ldh, void* gu, uint32_t ldgu, void* stream);

/* Linear cross entropy (xent.hip).  stats: over z, columns v0 .. v0 + n - 1
 * of the logits, the pair (max, sum of exp(z - max)) of each row and each
 * VKB_XENT_SLICE columns, to parts[slice * M + m], and the target's logit to
 * zt[m].  finish: lse and loss of S such slices.  rows: both at once, for
 * logits of at most VKB_XENT_ROW columns in all. */
#define VKB_XENT_SLICE 4096u
int vkb_launch_xent_stats(uint32_t M, uint32_t n, uint32_t v0, const float* z, int64_t ldz, const int64_t* target,
                          float* parts, float* zt, void* stream);
#define VKB_XENT_ROW 16384u
int vkb_launch_xent_rows(uint32_t M, uint32_t V, const float* z, int64_t ldz, const int64_t* target, int64_t ignore,
                         float* loss, float* lse, void* stream);
int vkb_launch_xent_finish(uint32_t M, uint32_t V, uint32_t S, const float* parts, const float* zt,
                           const int64_t* target, int64_t ignore, float* loss, float* lse, void* stream);
/* D = scal[0] * dloss * (exp(z - lse) - [v == target]), without scal by 1. */
int vkb_launch_xent_grad(int type, uint32_t M, uint32_t n, uint32_t v0, uint32_t V, const float* z, int64_t ldz,
                         const int64_t* target, int64_t ignore, const float* lse, const float* dloss,
                         vkb_scale scale, void* D, int64_t ldd, void* stream);

/* dx = D W and dw = beta dw + D^T x of a small gradient in one launch (pair.hip):
 * D M x R, W R x K, x M x K; dx of type, dw of w_type. */
typedef struct vkb_pair_scalars {
    float alpha, beta;
    const void *alpha_dev, *beta_dev;   /* fp32, in alpha's and beta's place where set */
} vkb_pair_scalars;
int vkb_pair_fits(int type, uint32_t M, uint32_t R, uint32_t K, uint32_t ldd, uint32_t ldw, uint32_t ldx);
int vkb_launch_pair(int type, int w_type, uint32_t M, uint32_t R, uint32_t K, const void* d, uint32_t ldd,
                    const void* w, uint32_t ldw, void* dx, uint32_t lddx, const vkb_pair_scalars* sx, const void* x,
                    uint32_t ldx, void* dw, uint32_t lddw, const vkb_pair_scalars* sw, void* stream);

/* The operators for up to VKB_FEW rows (few.hip), operands at any alignment.
 * forward: y = x w^T, R rows of w, fp32; or (glu) y = h = act(G) * U of R
 * columns, w of 2 R rows, and gu = [G | U] unless NULL.  K of at least 16
 * bytes.
 * backward: dw = beta * dw + D^T x (dw NULL: not) and, per slice of w's rows and
 * group of threads, the part of dx = D w (part NULL: not), vkb_few_slices
 * matrices of M x K that reduce adds up.  D (M x R) is the gated
 * projection's [dG | dU] from dh and gu, or the cross entropy's from z, fp32.
 * vkb_few_slices fills in kthreads and slice.  K of at least 16 bytes. */
#define VKB_FEW 32
/* whether rows of a forward pass go on the matrix units; R: the weight's rows (then
 * up to VKB_FEW, else up to 16) */
static inline int vkb_few_mfma(uint32_t M, uint64_t R) { return M > 8 && R >= 4096; }
#define VKB_FEW_BACK 8           /* rows of the backward pass */
typedef struct vkb_few_forward {
    const void *x, *w;
    void *y, *gu;
    int64_t ldx, ldw, ldy, ldgu;
    uint32_t M, R, K;
    int act;
} vkb_few_forward;
int vkb_launch_few_forward(int type, const vkb_few_forward* p, int glu, void* stream);
typedef struct vkb_few_backward {
    const void *x, *w;
    void* dw;
    int64_t ldx, ldw, lddw;
    float* part;
    uint32_t M, R, K;
    uint32_t kthreads, slice;
    float beta;
    const void *dh, *gu;
    int64_t lddh, ldgu;
    int act;
    const float *z, *lse, *dloss;
    int64_t ldz, ignore;
    const int64_t* target;
} vkb_few_backward;
uint32_t vkb_few_slices(int type, vkb_few_backward* p);
int vkb_launch_few_reduce(int type, const float* part, uint32_t parts, uint32_t M, uint32_t K, void* dx, int64_t lddx,
                          void* stream);
int vkb_launch_few_backward(int type, int g_type, const vkb_few_backward* p, int glu, void* stream);

/* Operators inside the pipelined GEMM kernel (nn_pipe.hpp): x M x K, w the
 * weight (2 N x K gated projection, N x K of the logits' classes), both as
 * vkb_op_plan accepts them.  tile: VKB_TILE_256 or VKB_TILE_128. */
typedef struct vkb_op_args {
    const void *x, *w;
    int64_t ldx, ldw;
    uint32_t M, N, K;
    int type, tile;
} vkb_op_args;
int vkb_launch_glu(const vkb_op_args* a, int act, void* h, int64_t ldh, void* gu, int64_t ldgu, void* stream);
/* parts: a pair for each row and each half of a tile's columns (128 or 64),
 * vkb_xent_slices of them */
uint32_t vkb_xent_slices(const vkb_op_args* a);
int vkb_launch_xent_stats_op(const vkb_op_args* a, const int64_t* target, float* parts, float* zt, void* stream);
/* D as vkb_launch_xent_grad, stored on Ms rows and Ns columns, zero past M and
 * N: at least those, at most them rounded up to 128, Ns a multiple of 8 */
int vkb_launch_xent_grad_op(const vkb_op_args* a, uint32_t Ms, uint32_t Ns, uint32_t v0, uint32_t V,
                            const int64_t* target, int64_t ignore, const float* lse, const float* dloss,
                            vkb_scale scale, void* D, int64_t ldd, void* stream);

#ifdef __cplusplus
}
#endif
