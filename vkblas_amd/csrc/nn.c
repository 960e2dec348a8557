/*
 * nn.c — host side of the operators in vkblas_nn.h: argument checks, plans,
 * workspaces and the order of launches.  No reference counterpart (see
 * vkblas_nn.h).
 *
 * A call's workspace is its stream's (engine.c): the arrival counters and
 * partials of the call's own GEMMs first, then the operator's buffers.
 */
#include <stdio.h>
#include <string.h>
#include <hip/hip_runtime_api.h>

#include "vkblas_nn.h"
#include "vkb_engine.h"
#include "vkb_launch.h"
#include "vkb_nn_launch.h"

#define DIM_MAX 0x7fffffffu
/* fp32 logits or projections that a joined call holds at a time */
#define JOIN_BYTES ((uint64_t)256 << 20)
/* the logits' gradient of a piece of the vocabulary */
#define PIECE_BYTES ((uint64_t)512 << 20)

static int known_type(vkblas_dtype_t t) {
    return t == VKBLAS_DT_F32 || t == VKBLAS_DT_F16 || t == VKBLAS_DT_BF16;
}
static size_t type_size(vkblas_dtype_t t) { return t == VKBLAS_DT_F32 ? 4 : 2; }
static int known_act(vkblas_act_t a) { return a >= VKBLAS_ACT_SILU && a <= VKBLAS_ACT_RELU; }
static int aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
static uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

/* One call: its stream, its workspace and how far it has come. */
typedef struct {
    void* stream;
    const char* what;
    vkb_prof prof;
    vkb_ws_lease ws;
    size_t gemm_bytes;           /* of the workspace, for the GEMMs' counters and partials */
    size_t used;                 /* bytes planned */
    int held;
    int written;                 /* an output's kernel is enqueued */
    vkblas_status_t st;
} op_call;

static void op_begin(op_call* c, const char* what, void* stream) {
    memset(c, 0, sizeof(*c));
    c->stream = stream;
    c->what = what;
    c->gemm_bytes = VKB_WS_HEADER;
}

/* Plan: a product of the call (its scratch), then its buffers, whose offset
 * buf() returns; room() takes the workspace. */
static void need_gemm(op_call* c, vkblas_dtype_t ab, vkblas_dtype_t ct, vkblas_op_t op_a, vkblas_op_t op_b, uint32_t M,
                      uint32_t N, uint32_t K, const void* A, uint32_t lda, const void* B, uint32_t ldb, uint32_t ldc) {
    const size_t b = vkb_gemm_scratch_bytes(ab, ct, op_a, op_b, M, N, K, lda, ldb, ldc, aligned16(A) && aligned16(B));
    if (b > c->gemm_bytes) c->gemm_bytes = b;
}
static size_t buf(op_call* c, uint64_t bytes) {
    if (!c->used) c->used = round_up(c->gemm_bytes, 256);
    const size_t at = c->used;
    c->used += round_up(bytes, 256);
    return at;
}
static vkblas_status_t room(op_call* c) {
    if (!vkb_engine_ready()) return c->st = VKBLAS_ERR_INIT;
    if (!c->used && c->gemm_bytes > VKB_WS_HEADER) c->used = c->gemm_bytes;
    if (c->used) {
        if (vkb_ws_acquire(c->stream, c->used, &c->ws) != 0) return c->st = VKBLAS_ERR_INIT;
        c->held = 1;
    }
    vkb_prof_begin(&c->prof, c->stream);
    return VKBLAS_OK;
}
static void* at(const op_call* c, size_t off) { return (char*)c->ws.ptr + off; }

/* After a launch: rc of it; out: it writes an output. */
static int step(op_call* c, int rc, int out) {
    if (rc != 0) {
        c->st = c->written ? VKBLAS_ERR_PARTIAL : VKBLAS_ERR_INIT;
        if (vkb_engine_trace()) fprintf(stderr, "[vkblas] %s: launch failed: %s\n", c->what,
                                        hipGetErrorString((hipError_t)rc));
        return 0;
    }
    if (out) c->written = 1;
    return 1;
}

/* Scalars of a product: host values, or device ones where dev is set. */
typedef struct {
    float alpha, beta;
    const float *alpha_dev, *beta_dev;
} scalars;
static scalars host_scalars(float alpha, float beta) {
    scalars s = {alpha, beta, NULL, NULL};
    return s;
}
static int product(op_call* c, vkblas_dtype_t ab, vkblas_dtype_t ct, vkblas_op_t op_a, vkblas_op_t op_b, uint32_t M,
                   uint32_t N, uint32_t K, scalars s, const void* A, uint32_t lda, const void* B, uint32_t ldb,
                   void* C, uint32_t ldc, int out) {
    const vkblas_scalar_mode_t mode = s.alpha_dev ? VKBLAS_SCALAR_DEV_F32 : VKBLAS_SCALAR_HOST;
    vkblas_status_t st;
    if (c->held)
        st = vkb_gemm_with_scratch(ab, ct, op_a, op_b, M, N, K, s.alpha, A, lda, B, ldb, s.beta, C, ldc, 1, 0, 0, 0,
                                   mode, s.alpha_dev, s.beta_dev, 0, c->stream, c->ws.ptr, c->gemm_bytes);
    else   /* no workspace held: the plan has no split */
        st = vkblas_gemm_async(ab, ct, op_a, op_b, M, N, K, s.alpha, A, lda, B, ldb, s.beta, C, ldc, 1, 0, 0, 0, mode,
                               s.alpha_dev, s.beta_dev, 0, c->stream);
    if (st != VKBLAS_OK) {
        c->st = c->written || (out && st == VKBLAS_ERR_PARTIAL) ? VKBLAS_ERR_PARTIAL : VKBLAS_ERR_INIT;
        return 0;
    }
    if (out) c->written = 1;
    return 1;
}

static vkblas_status_t op_end(op_call* c, int kernel) {
    if (c->held) vkb_ws_release(&c->ws);
    vkb_prof_end(&c->prof, c->stream, c->what, c->st == VKBLAS_OK);
    if (c->st == VKBLAS_OK) vkb_engine_ran(kernel >= VKBLAS_KERNEL_JOINED ? vkblas_last_path() : VKBLAS_PATH_NONE, kernel);
    return c->st;
}

/* ------------------------------------------- inside the pipelined kernel */

extern int vkb_launch_glu_f32(const vkb_op_args*, int, void*, int64_t, void*, int64_t, void*);
extern int vkb_launch_glu_f16(const vkb_op_args*, int, void*, int64_t, void*, int64_t, void*);
extern int vkb_launch_glu_bf16(const vkb_op_args*, int, void*, int64_t, void*, int64_t, void*);
extern int vkb_launch_xent_stats_f32(const vkb_op_args*, const int64_t*, float*, float*, void*);
extern int vkb_launch_xent_stats_f16(const vkb_op_args*, const int64_t*, float*, float*, void*);
extern int vkb_launch_xent_stats_bf16(const vkb_op_args*, const int64_t*, float*, float*, void*);
typedef int xent_grad_fn(const vkb_op_args*, uint32_t, uint32_t, const int64_t*, int64_t, const float*, const float*,
                         const float*, void*, int64_t, void*);
extern xent_grad_fn vkb_launch_xent_grad_f32, vkb_launch_xent_grad_f16, vkb_launch_xent_grad_bf16;

int vkb_launch_glu(const vkb_op_args* a, int act, void* h, int64_t ldh, void* gu, int64_t ldgu, void* stream) {
    return (a->type == VKB_T_F16 ? vkb_launch_glu_f16 : a->type == VKB_T_BF16 ? vkb_launch_glu_bf16
                                                                             : vkb_launch_glu_f32)(
        a, act, h, ldh, gu, ldgu, stream);
}
int vkb_launch_xent_stats_op(const vkb_op_args* a, const int64_t* target, float* parts, float* zt, void* stream) {
    return (a->type == VKB_T_F16 ? vkb_launch_xent_stats_f16 : a->type == VKB_T_BF16 ? vkb_launch_xent_stats_bf16
                                                                                    : vkb_launch_xent_stats_f32)(
        a, target, parts, zt, stream);
}
int vkb_launch_xent_grad_op(const vkb_op_args* a, uint32_t v0, uint32_t V, const int64_t* target, int64_t ignore,
                            const float* lse, const float* dloss, const float* scal, void* D, int64_t ldd,
                            void* stream) {
    return (a->type == VKB_T_F16 ? vkb_launch_xent_grad_f16 : a->type == VKB_T_BF16 ? vkb_launch_xent_grad_bf16
                                                                                   : vkb_launch_xent_grad_f32)(
        a, v0, V, target, ignore, lse, dloss, scal, D, ldd, stream);
}
uint32_t vkb_xent_slices(const vkb_op_args* a) {
    const uint64_t tile = vkb_tile_bn(a->tile);
    return (uint32_t)(((uint64_t)a->N + tile - 1) / tile * 2);
}

/* Whether the pipelined kernel takes x w^T with an operator at its end, and
 * on which tiles; cols: the columns that one tile of 256 holds (128 gated).
 *  - 16-byte aligned operands and leading dimensions, K in whole steps: 64 for
 *    16-bit types, from two steps on, and pairs of 32 for fp32; the bytes
 *    that a tile's rows span below 2^31 (offsets are 32-bit);
 *  - more than 64 rows: below that the decode kernels stream the weight;
 *  - 256 x 256 tiles where the planner of the plain products takes them:
 *    16-bit from more than 128 of them on, fp32 for about whole waves. */
static int op_plan(vkblas_dtype_t type, uint32_t M, uint32_t N, uint32_t K, const void* x, uint32_t ldx,
                   const void* w, uint32_t ldw, uint32_t cols, vkb_op_args* a) {
    const uint32_t vec = type == VKBLAS_DT_F32 ? 4 : 8;
    const uint64_t es = type_size(type);
    const uint64_t ld = ldx > ldw ? ldx : ldw;
    if (!aligned16(x) || !aligned16(w) || ldx % vec || ldw % vec || K % 64 || K < 128 || M <= 64 ||
        (256 * ld + K) * es >= 1ull << 31)
        return 0;
    const uint64_t t = (uint64_t)((M + 255) / 256) * ((N + cols - 1) / cols);
    a->x = x;
    a->w = w;
    a->ldx = ldx;
    a->ldw = ldw;
    a->M = M;
    a->N = N;
    a->K = K;
    a->type = type;
    a->tile = (type == VKBLAS_DT_F32 ? 8 * t >= 7 * 256 * ((t + 255) / 256) : t > 128) ? VKB_TILE_256 : VKB_TILE_128;
    return 1;
}

/* A gradient over no rows: C = beta * C. */
static vkblas_status_t empty_gradient(op_call* c, vkblas_dtype_t type, uint32_t M, uint32_t N, void* C, uint32_t ldc,
                                      float beta) {
    if (!C || (beta == 1.0f)) return VKBLAS_OK;
    if (!vkb_engine_ready()) return VKBLAS_ERR_INIT;
    step(c, vkb_launch_scale(type, M, N, C, ldc, beta, c->stream), 1);
    return c->st;
}

/* ------------------------------------------------------------- layer norm */

vkblas_status_t vkblas_layer_norm_async(vkblas_dtype_t type, vkblas_dtype_t w_type, uint32_t M, uint32_t N,
                                        const void* x, uint32_t ldx, const void* w, const void* b, float eps, void* y,
                                        uint32_t ldy, float* mean, float* rstd, void* stream) {
    if (!known_type(type) || (w_type != type && w_type != VKBLAS_DT_F32)) return VKBLAS_ERR_PARAM;
    if (N == 0 || M > DIM_MAX || N > DIM_MAX || ldx < N || ldy < N) return VKBLAS_ERR_PARAM;
    if (M == 0) return VKBLAS_OK;
    if (!x || !y) return VKBLAS_ERR_PARAM;
    op_call c;
    op_begin(&c, "layer_norm", stream);
    if (vkb_engine_trace()) fprintf(stderr, "[vkblas] layer_norm type=%d M=%u N=%u\n", (int)type, M, N);
    if (room(&c) != VKBLAS_OK) return c.st;
    step(&c, vkb_launch_layer_norm(type, w_type, M, N, x, ldx, w, b, eps, y, ldy, mean, rstd, stream), 1);
    return op_end(&c, vkb_layer_norm_long(N) ? VKBLAS_KERNEL_NORM_LONG : VKBLAS_KERNEL_NORM);
}

vkblas_status_t vkblas_layer_norm_backward_async(vkblas_dtype_t type, vkblas_dtype_t w_type, uint32_t M, uint32_t N,
                                                 const void* dy, uint32_t lddy, const void* x, uint32_t ldx,
                                                 const void* w, const float* mean, const float* rstd, void* dx,
                                                 uint32_t lddx, void* dw, void* db, vkblas_dtype_t g_type, float beta,
                                                 void* stream) {
    if (!known_type(type) || (w_type != type && w_type != VKBLAS_DT_F32)) return VKBLAS_ERR_PARAM;
    if ((dw || db) && g_type != w_type && g_type != VKBLAS_DT_F32) return VKBLAS_ERR_PARAM;
    if (N == 0 || M > DIM_MAX || N > DIM_MAX || ldx < N || lddy < N || (dx && lddx < N)) return VKBLAS_ERR_PARAM;
    op_call c;
    op_begin(&c, "layer_norm_backward", stream);
    if (M == 0) {
        if (empty_gradient(&c, g_type, 1, N, dw, N, beta) != VKBLAS_OK) return c.st;
        return empty_gradient(&c, g_type, 1, N, db, N, beta);
    }
    if (!dy || !x || !mean || !rstd) return VKBLAS_ERR_PARAM;
    if (!dx && !dw && !db) return VKBLAS_OK;
    if (vkb_engine_trace()) fprintf(stderr, "[vkblas] layer_norm_backward type=%d M=%u N=%u\n", (int)type, M, N);
    const uint32_t parts = vkb_layer_norm_parts(type, M, N);
    const int sums = dw || db;
    const size_t o_part = sums ? buf(&c, (uint64_t)parts * 2 * N * sizeof(float)) : 0;
    if (room(&c) != VKBLAS_OK) return c.st;
    float* part = sums ? (float*)at(&c, o_part) : NULL;
    if (step(&c, vkb_launch_layer_norm_backward(type, w_type, M, N, dy, lddy, x, ldx, w, mean, rstd, dx, lddx, part,
                                                stream), dx != NULL) && sums)
        step(&c, vkb_launch_layer_norm_reduce(part, parts, N, dw, db, g_type, beta, stream), 1);
    return op_end(&c, vkb_layer_norm_long(N) ? VKBLAS_KERNEL_NORM_LONG : VKBLAS_KERNEL_NORM);
}

/* ------------------------------------------------------- gated projection */

vkblas_status_t vkblas_glu_async(vkblas_dtype_t type, vkblas_act_t act, uint32_t M, uint32_t N, uint32_t K,
                                 const void* x, uint32_t ldx, const void* w, uint32_t ldw, void* h, uint32_t ldh,
                                 void* gu, uint32_t ldgu, void* stream) {
    if (!known_type(type) || !known_act(act)) return VKBLAS_ERR_PARAM;
    if (N == 0 || K == 0 || M > DIM_MAX || N > DIM_MAX / 2 || K > DIM_MAX || ldx < K || ldw < K || ldh < N ||
        (gu && ldgu < 2 * N))
        return VKBLAS_ERR_PARAM;
    if (M == 0) return VKBLAS_OK;
    if (!x || !w || !h) return VKBLAS_ERR_PARAM;
    op_call c;
    op_begin(&c, "glu", stream);
    if (vkb_engine_trace()) fprintf(stderr, "[vkblas] glu type=%d act=%d M=%u N=%u K=%u\n", (int)type, (int)act, M, N, K);
    vkb_op_args a;
    if (op_plan(type, M, N, K, x, ldx, w, ldw, 128, &a)) {
        if (room(&c) != VKBLAS_OK) return c.st;
        step(&c, vkb_launch_glu(&a, act, h, ldh, gu, ldgu, stream), 1);
        return op_end(&c, VKBLAS_KERNEL_FUSED);
    }
    /* both projections in fp32, some rows at a time, then the join; an fp32
     * gu takes them itself */
    const int direct = type == VKBLAS_DT_F32 && gu;
    uint64_t rows = direct ? M : JOIN_BYTES / ((uint64_t)8 * N);
    if (rows < 64) rows = 64;
    if (rows > M) rows = M;
    const uint32_t ldz = direct ? ldgu : (uint32_t)round_up(2 * N, 4);
    need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, (uint32_t)rows, 2 * N, K, x, ldx, w, ldw, ldz);
    const size_t es = type_size(type);
    if (M % rows)
        need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, (uint32_t)(M % rows), 2 * N, K,
                  (const char*)x + (M - M % rows) * ldx * es, ldx, w, ldw, ldz);
    const size_t o_z = direct ? 0 : buf(&c, rows * ldz * sizeof(float));
    if (room(&c) != VKBLAS_OK) return c.st;
    for (uint64_t m = 0; m < M; m += rows) {
        const uint32_t n = (uint32_t)(M - m < rows ? M - m : rows);
        float* z = direct ? (float*)gu : (float*)at(&c, o_z);
        if (!product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, n, 2 * N, K, host_scalars(1.0f, 0.0f),
                     (const char*)x + m * ldx * es, ldx, w, ldw, z, ldz, direct))
            break;
        if (!step(&c, vkb_launch_glu_join(type, act, n, N, z, ldz, (char*)h + m * ldh * es, ldh,
                                          direct || !gu ? NULL : (char*)gu + m * ldgu * es, ldgu, stream), 1))
            break;
    }
    return op_end(&c, VKBLAS_KERNEL_JOINED);
}

vkblas_status_t vkblas_glu_backward_async(vkblas_dtype_t type, vkblas_act_t act, uint32_t M, uint32_t N, uint32_t K,
                                          const void* dh, uint32_t lddh, const void* gu, uint32_t ldgu, const void* x,
                                          uint32_t ldx, const void* w, uint32_t ldw, void* dgu, uint32_t lddgu,
                                          void* dx, uint32_t lddx, void* dw, uint32_t lddw, vkblas_dtype_t dw_type,
                                          float beta, void* stream) {
    if (!known_type(type) || !known_act(act) || (dw && dw_type != type && dw_type != VKBLAS_DT_F32))
        return VKBLAS_ERR_PARAM;
    if (N == 0 || K == 0 || M > DIM_MAX || N > DIM_MAX / 2 || K > DIM_MAX || lddh < N || ldgu < 2 * N ||
        (dw && (ldx < K || lddw < K)) || (dx && (ldw < K || lddx < K)) || (dgu && lddgu < 2 * N))
        return VKBLAS_ERR_PARAM;
    op_call c;
    op_begin(&c, "glu_backward", stream);
    if (M == 0) return empty_gradient(&c, dw_type, 2 * N, K, dw, lddw, beta);
    if (!dh || !gu || (dw && !x) || (dx && !w)) return VKBLAS_ERR_PARAM;
    if (!dgu && !dx && !dw) return VKBLAS_OK;
    if (vkb_engine_trace())
        fprintf(stderr, "[vkblas] glu_backward type=%d act=%d M=%u N=%u K=%u\n", (int)type, (int)act, M, N, K);
    const uint32_t ldd = dgu ? lddgu : (uint32_t)round_up(2 * N, 8);
    if (dx) need_gemm(&c, type, type, VKBLAS_OP_N, VKBLAS_OP_N, M, K, 2 * N, dgu, ldd, w, ldw, lddx);
    if (dw) need_gemm(&c, type, dw_type, VKBLAS_OP_T, VKBLAS_OP_N, 2 * N, K, M, dgu, ldd, x, ldx, lddw);
    const size_t o_d = dgu ? 0 : buf(&c, (uint64_t)M * ldd * type_size(type));
    if (room(&c) != VKBLAS_OK) return c.st;
    void* d = dgu ? dgu : at(&c, o_d);
    if (step(&c, vkb_launch_glu_join_backward(type, act, M, N, dh, lddh, gu, ldgu, d, ldd, stream), dgu != NULL) &&
        (!dx || product(&c, type, type, VKBLAS_OP_N, VKBLAS_OP_N, M, K, 2 * N, host_scalars(1.0f, 0.0f), d, ldd, w,
                        ldw, dx, lddx, 1)) &&
        dw)
        product(&c, type, dw_type, VKBLAS_OP_T, VKBLAS_OP_N, 2 * N, K, M, host_scalars(1.0f, beta), d, ldd, x, ldx, dw,
                lddw, 1);
    return op_end(&c, VKBLAS_KERNEL_JOINED);
}

/* --------------------------------------------------- linear cross entropy */

typedef struct { uint32_t v, cols; } piece_t;

/* Columns of the vocabulary at a time, so that M of them take about `bytes`
 * at `each` bytes a logit: whole slices of 256. */
static uint32_t piece_columns(uint32_t M, uint32_t V, uint64_t bytes, uint64_t each) {
    uint64_t n = bytes / (each * M) / 256 * 256;
    if (n < 256) n = 256;
    return (uint32_t)(n < V ? n : V);
}

vkblas_status_t vkblas_linear_xent_async(vkblas_dtype_t type, uint32_t M, uint32_t V, uint32_t K, const void* x,
                                         uint32_t ldx, const void* w, uint32_t ldw, const int64_t* target,
                                         int64_t ignore_index, float* loss, float* lse, void* stream) {
    if (!known_type(type)) return VKBLAS_ERR_PARAM;
    if (V == 0 || K == 0 || M > DIM_MAX || V > DIM_MAX || K > DIM_MAX || ldx < K || ldw < K) return VKBLAS_ERR_PARAM;
    if (M == 0) return VKBLAS_OK;
    if (!x || !w || !lse || (loss && !target)) return VKBLAS_ERR_PARAM;
    if (!loss) target = NULL;
    op_call c;
    op_begin(&c, "linear_xent", stream);
    if (vkb_engine_trace()) fprintf(stderr, "[vkblas] linear_xent type=%d M=%u V=%u K=%u\n", (int)type, M, V, K);
    vkb_op_args a;
    if (op_plan(type, M, V, K, x, ldx, w, ldw, 256, &a)) {
        const uint32_t S = vkb_xent_slices(&a);
        const size_t o_p = buf(&c, (uint64_t)S * M * 2 * sizeof(float)), o_t = buf(&c, (uint64_t)M * sizeof(float));
        if (room(&c) != VKBLAS_OK) return c.st;
        float *parts = at(&c, o_p), *zt = at(&c, o_t);
        if (step(&c, vkb_launch_xent_stats_op(&a, target, parts, zt, stream), 0))
            step(&c, vkb_launch_xent_finish(M, V, S, parts, zt, target, ignore_index, loss, lse, stream), 1);
        return op_end(&c, VKBLAS_KERNEL_FUSED);
    }
    const uint32_t n = piece_columns(M, V, JOIN_BYTES, sizeof(float)), ldz = (uint32_t)round_up(n, 4);
    const uint32_t last = V % n;
    const uint32_t per = (n + VKB_XENT_SLICE - 1) / VKB_XENT_SLICE;   /* slices of a piece; the last may have fewer */
    const uint32_t S = V / n * per + (last + VKB_XENT_SLICE - 1) / VKB_XENT_SLICE;
    need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, n, K, x, ldx, w, ldw, ldz);
    if (last) need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, last, K, x, ldx, w, ldw, ldz);
    const size_t o_z = buf(&c, (uint64_t)M * ldz * sizeof(float));
    const size_t o_p = buf(&c, (uint64_t)S * M * 2 * sizeof(float));
    const size_t o_t = buf(&c, (uint64_t)M * sizeof(float));
    if (room(&c) != VKBLAS_OK) return c.st;
    float *z = at(&c, o_z), *parts = at(&c, o_p), *zt = at(&c, o_t);
    int ok = 1;
    uint32_t slice = 0;
    for (uint64_t v = 0; ok && v < V; v += n, slice += per) {
        const uint32_t cols = (uint32_t)(V - v < n ? V - v : n);
        ok = product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, cols, K, host_scalars(1.0f, 0.0f), x, ldx,
                     (const char*)w + v * ldw * type_size(type), ldw, z, ldz, 0) &&
             step(&c, vkb_launch_xent_stats(M, cols, (uint32_t)v, z, ldz, target, parts + (uint64_t)slice * M * 2, zt,
                                            stream), 0);
    }
    if (ok) step(&c, vkb_launch_xent_finish(M, V, S, parts, zt, target, ignore_index, loss, lse, stream), 1);
    return op_end(&c, VKBLAS_KERNEL_JOINED);
}

vkblas_status_t vkblas_linear_xent_backward_async(vkblas_dtype_t type, uint32_t M, uint32_t V, uint32_t K,
                                                  const void* x, uint32_t ldx, const void* w, uint32_t ldw,
                                                  const int64_t* target, int64_t ignore_index, const float* lse,
                                                  const float* dloss, void* dx, uint32_t lddx, void* dw,
                                                  uint32_t lddw, vkblas_dtype_t dw_type, float beta, void* stream) {
    if (!known_type(type) || (dw && dw_type != type && dw_type != VKBLAS_DT_F32)) return VKBLAS_ERR_PARAM;
    if (V == 0 || K == 0 || M > DIM_MAX || V > DIM_MAX || K > DIM_MAX || ldx < K || ldw < K || (dx && lddx < K) ||
        (dw && lddw < K))
        return VKBLAS_ERR_PARAM;
    op_call c;
    op_begin(&c, "linear_xent_backward", stream);
    if (M == 0) return empty_gradient(&c, dw_type, V, K, dw, lddw, beta);
    if (!x || !w || !target || !lse || !dloss) return VKBLAS_ERR_PARAM;
    if (!dx && !dw) return VKBLAS_OK;
    if (vkb_engine_trace())
        fprintf(stderr, "[vkblas] linear_xent_backward type=%d M=%u V=%u K=%u\n", (int)type, M, V, K);
    /* D of a piece of the vocabulary at a time, in type: from the pipelined
     * kernel, or over the piece's logits in fp32 (fp32: in their place).
     * Pieces are whole tiles, then the rest of the vocabulary: odd classes
     * would cost both products of a whole piece their fast kernels. */
    const int f32 = type == VKBLAS_DT_F32;
    const size_t es = type_size(type);
    vkb_op_args a;
    const int fused = op_plan(type, M, V, K, x, ldx, w, ldw, 256, &a);
    uint32_t n = piece_columns(M, V, fused ? PIECE_BYTES : JOIN_BYTES, fused ? es : sizeof(float));
    if (n == V && V > 256 && V % 128) n = V / 128 * 128;
    const uint32_t ldd = (uint32_t)round_up(n, 8);
    piece_t pieces[3];           /* the kinds of pieces: n columns, then whole tiles, then the rest */
    int kinds = 0;
    const uint32_t tail = V % n;
    pieces[kinds++] = (piece_t){0, n};
    if (tail >= 128) pieces[kinds++] = (piece_t){V - tail, tail / 128 * 128};
    if (tail % 128) pieces[kinds++] = (piece_t){V - tail % 128, tail % 128};
    /* dx adds up over the pieces in fp32: in dx itself or in the workspace */
    const int acc = dx && n < V && !f32;
    const vkblas_dtype_t xt = acc ? VKBLAS_DT_F32 : type;
    const uint32_t lda = acc ? (uint32_t)round_up(K, 4) : lddx;
    for (int i = 0; i < kinds; ++i) {
        const uint32_t cols = pieces[i].cols;
        if (!fused)
            need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, cols, K, x, ldx, w, ldw, ldd);
        if (dx) need_gemm(&c, type, xt, VKBLAS_OP_N, VKBLAS_OP_N, M, K, cols, NULL, ldd, w, ldw, lda);
        if (dw) need_gemm(&c, type, dw_type, VKBLAS_OP_T, VKBLAS_OP_N, cols, K, M, NULL, ldd, x, ldx, lddw);
    }
    const size_t o_z = fused ? 0 : buf(&c, (uint64_t)M * ldd * sizeof(float));
    const size_t o_d = f32 && !fused ? o_z : buf(&c, (uint64_t)M * ldd * es);
    const size_t o_a = acc ? buf(&c, (uint64_t)M * lda * sizeof(float)) : 0;
    const size_t o_s = buf(&c, 8 * sizeof(float));
    if (room(&c) != VKBLAS_OK) return c.st;
    float *z = at(&c, o_z), *scal = f32 ? NULL : (float*)at(&c, o_s);
    void *d = at(&c, o_d), *xo = acc ? at(&c, o_a) : dx;
    int ok = !scal || step(&c, vkb_launch_xent_scale(type, M, dloss, beta, scal, stream), 0);
    for (uint64_t v = 0; ok && v < V;) {
        const uint32_t left = (uint32_t)(V - v), cols = left >= n ? n : left >= 128 ? left / 128 * 128 : left;
        const char* wv = (const char*)w + v * ldw * es;
        if (fused) {
            a.w = wv;
            a.N = cols;
            ok = step(&c, vkb_launch_xent_grad_op(&a, (uint32_t)v, V, target, ignore_index, lse, dloss, scal, d, ldd,
                                                  stream), 0);
        } else {
            ok = product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, cols, K, host_scalars(1.0f, 0.0f), x,
                         ldx, wv, ldw, z, ldd, 0) &&
                 step(&c, vkb_launch_xent_grad(type, M, cols, (uint32_t)v, V, z, ldd, target, ignore_index, lse, dloss,
                                               scal, d, ldd, stream), 0);
        }
        const scalars sw = {1.0f, beta, scal ? scal + 1 : NULL, scal ? scal + 2 : NULL};
        const scalars sx = {1.0f, v ? 1.0f : 0.0f, scal ? scal + 1 : NULL, scal ? scal + (v ? 3 : 4) : NULL};
        if (ok && dw)
            ok = product(&c, type, dw_type, VKBLAS_OP_T, VKBLAS_OP_N, cols, K, M, sw, d, ldd, x, ldx,
                         (char*)dw + v * lddw * type_size(dw_type), lddw, 1);
        if (ok && dx)
            ok = product(&c, type, xt, VKBLAS_OP_N, VKBLAS_OP_N, M, K, cols, sx, d, ldd, wv, ldw, xo, lda, !acc);
        v += cols;
    }
    if (ok && acc)
        step(&c, vkb_launch_convert(type, M, K, xo, lda, dx, lddx, stream), 1);
    return op_end(&c, fused ? VKBLAS_KERNEL_FUSED : VKBLAS_KERNEL_JOINED);
}
