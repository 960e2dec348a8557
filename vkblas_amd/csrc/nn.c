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
    int must;                    /* a product has no plan without its partials */
    int held;
    int written;                 /* an output's kernel is enqueued */
    int path;                    /* of the last product */
    vkblas_status_t st;
} op_call;

static void op_begin(op_call* c, const char* what, void* stream) {
    memset(c, 0, sizeof(*c));
    c->stream = stream;
    c->what = what;
    c->gemm_bytes = VKB_WS_HEADER;
    c->path = VKBLAS_PATH_NONE;
}

/* Plan: a product of the call (its scratch), then its buffers, whose offset
 * buf() returns; room() takes the workspace. */
static void need_gemm(op_call* c, vkblas_dtype_t ab, vkblas_dtype_t ct, vkblas_op_t op_a, vkblas_op_t op_b, uint32_t M,
                      uint32_t N, uint32_t K, const void* A, uint32_t lda, const void* B, uint32_t ldb, uint32_t ldc) {
    int optional;
    const size_t b = vkb_gemm_scratch_bytes(ab, ct, op_a, op_b, M, N, K, lda, ldb, ldc, aligned16(A) && aligned16(B),
                                            &optional);
    if (b > c->gemm_bytes) c->gemm_bytes = b;
    if (!optional) c->must = 1;
}
static size_t buf(op_call* c, uint64_t bytes) {
    if (!c->used) c->used = round_up(c->gemm_bytes, 256);
    const size_t at = c->used;
    c->used += round_up(bytes, 256);
    return at;
}
static vkblas_status_t room(op_call* c) {
    if (!vkb_engine_ready()) return c->st = VKBLAS_ERR_INIT;
    /* wanted for nothing but K splits, the products run without it too */
    const int optional = !c->used && !c->must;
    if (!c->used && c->gemm_bytes > VKB_WS_HEADER) c->used = c->gemm_bytes;
    if (c->used) {
        c->held = vkb_ws_acquire(c->stream, c->used, &c->ws) == 0;
        if (!c->held && !optional) return c->st = VKBLAS_ERR_INIT;
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
    else   /* no workspace held: the plan has no split, or does without */
        st = vkblas_gemm_async(ab, ct, op_a, op_b, M, N, K, s.alpha, A, lda, B, ldb, s.beta, C, ldc, 1, 0, 0, 0, mode,
                               s.alpha_dev, s.beta_dev, 0, c->stream);
    if (st != VKBLAS_OK) {
        c->st = c->written || (out && st == VKBLAS_ERR_PARTIAL) ? VKBLAS_ERR_PARTIAL : VKBLAS_ERR_INIT;
        return 0;
    }
    c->path = vkblas_last_path();
    if (out) c->written = 1;
    return 1;
}

static vkblas_status_t op_end(op_call* c, int kernel) {
    if (c->held) vkb_ws_release(&c->ws);
    vkb_prof_end(&c->prof, c->stream, c->what, c->st == VKBLAS_OK);
    if (c->st == VKBLAS_OK) vkb_engine_ran(c->path, kernel);
    return c->st;
}

/* ------------------------------------------- inside the pipelined kernel */

extern int vkb_launch_glu_f32(const vkb_op_args*, int, void*, int64_t, void*, int64_t, void*);
extern int vkb_launch_glu_f16(const vkb_op_args*, int, void*, int64_t, void*, int64_t, void*);
extern int vkb_launch_glu_bf16(const vkb_op_args*, int, void*, int64_t, void*, int64_t, void*);
extern int vkb_launch_xent_stats_f32(const vkb_op_args*, const int64_t*, float*, float*, void*);
extern int vkb_launch_xent_stats_f16(const vkb_op_args*, const int64_t*, float*, float*, void*);
extern int vkb_launch_xent_stats_bf16(const vkb_op_args*, const int64_t*, float*, float*, void*);
typedef int xent_grad_fn(const vkb_op_args*, uint32_t, uint32_t, uint32_t, uint32_t, const int64_t*, int64_t,
                         const float*, const float*, vkb_scale, void*, int64_t, void*);
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
int vkb_launch_xent_grad_op(const vkb_op_args* a, uint32_t Ms, uint32_t Ns, uint32_t v0, uint32_t V,
                            const int64_t* target, int64_t ignore, const float* lse, const float* dloss,
                            vkb_scale scale, void* D, int64_t ldd, void* stream) {
    return (a->type == VKB_T_F16 ? vkb_launch_xent_grad_f16 : a->type == VKB_T_BF16 ? vkb_launch_xent_grad_bf16
                                                                                   : vkb_launch_xent_grad_f32)(
        a, Ms, Ns, v0, V, target, ignore, lse, dloss, scale, D, ldd, stream);
}
uint32_t vkb_xent_slices(const vkb_op_args* a) {
    const uint64_t tile = vkb_tile_bn(a->tile);
    return (uint32_t)(((uint64_t)a->N + tile - 1) / tile * 2);
}

/* Whether the pipelined kernel takes x w^T with an operator at its end, and
 * on which tiles; cols: the columns that one tile of 256 holds (128 gated).
 *  - 16-byte aligned operands and leading dimensions, K in whole 16-byte units;
 *    the bytes that a tile's rows span below 2^31 (offsets are 32-bit);
 *  - more than 64 rows, below which the decode kernels stream the weight, or
 *    16-bit operands with K of at most 512: then one launch instead of two or
 *    three is ahead;
 *  - enough tiles of 128 for their K: few tiles with a long K are faster as a
 *    product with K split and a pass over its result.  us, joined / here, gated
 *    projection bf16: 16 tiles K = 1024 10.8 / 9.7, 4096 21.4 / 26.8; 44 tiles 2048
 *    20.5 / 16.9; 64 tiles 512 12.0 / 7.3, 4096 25.2 / 27.2; 74 tiles 2432 22.4 / 19.9;
 *    128 tiles 4096 33.3 / 30.1; fp32: 32 tiles K = 1024 25 / 59, 128 tiles 63.8 / 62.1,
 *    K = 4096 149 / 233, 256 tiles 269 / 244;
 *  - 16-bit: the tile whose waves of workgroups (one 256 x 256 or two 128 x 128
 *    per CU) take less at the rates measured, a K step of 64 1.45 and 0.83 us and
 *    an epilogue 6 and 4 (us on 128 / 256: 2048 x 4096 x 4096 gated, one wave of 256,
 *    107 / 94; 2048 x 5120 x 4096, 1.25 waves, 146 / 160; 1000 x 16000 x 384 29 / 34);
 *    fp32: 256 x 256 only for about whole waves, as the plain products. */
static int op_plan(vkblas_dtype_t type, uint32_t M, uint32_t N, uint32_t K, const void* x, uint32_t ldx,
                   const void* w, uint32_t ldw, uint32_t cols, vkb_op_args* a) {
    const uint32_t vec = type == VKBLAS_DT_F32 ? 4 : 8;
    const uint64_t es = type_size(type);
    const uint64_t ld = ldx > ldw ? ldx : ldw;
    if (!aligned16(x) || !aligned16(w) || ldx % vec || ldw % vec || K % vec || (M <= 64 && (K > 512 || type == VKBLAS_DT_F32)) ||
        (256 * ld + K) * es >= 1ull << 31)
        return 0;
    const uint64_t t = (uint64_t)((M + 255) / 256) * ((N + cols - 1) / cols);
    const uint64_t t128 = (uint64_t)((M + 127) / 128) * ((N + cols / 2 - 1) / (cols / 2));
    int large;
    if (type == VKBLAS_DT_F32) {
        if (t128 < (K <= 2048 ? 128 : 200)) return 0;
        large = 8 * t >= 7 * 256 * ((t + 255) / 256);
    } else {
        if (t128 < 96 && K > 1024 && (K > 64 * t128 || K > 2560)) return 0;
        const double w256 = t < 1024 ? (double)((t + 255) / 256) : (double)t / 256;
        const double w128 = t128 < 2048 ? (double)((t128 + 511) / 512) : (double)t128 / 512;
        large = t > 128 && w256 * (1.45 * K / 64 + 6) <= w128 * (0.83 * K / 64 + 4);
    }
    a->x = x;
    a->w = w;
    a->ldx = ldx;
    a->ldw = ldw;
    a->M = M;
    a->N = N;
    a->K = K;
    a->type = type;
    a->tile = large ? VKB_TILE_256 : VKB_TILE_128;
    return 1;
}

/* ----------------------------------------------- operands and their copies */

/* A program's matrix (S of M x N below each other), or a copy of it in the
 * workspace, padded with zeros to Mp x Np each: what the fast kernels do not
 * take (rows off 16-byte units, sizes off whole steps) costs them 3 to 8 times
 * their time, and a copy one pass over it. */
typedef struct {
    const void* p;
    uint32_t ld, S, M, N, Mp, Np;
    int copy;
    size_t off;
} operand;

static uint32_t vec_of(vkblas_dtype_t t) { return t == VKBLAS_DT_F32 ? 4 : 8; }
static int off_units(vkblas_dtype_t t, const void* p, uint32_t ld) { return !aligned16(p) || ld % vec_of(t); }
/* Whether a 16-bit operand's K steps lie across two lines each, which loads
 * both, and K is long enough for the loads to count (us, as it is / on copies,
 * other inputs each pass: bf16 xent 4323 x 1209 x 4984 98.7 / 82.0, 4000 x 32000 x 1000
 * 285 / 262, 5886 x 79834 x 712 753 / 724, gated 4000 x 8000 x 4040 477 / 431).  The
 * copies cost 3 to 8 us: level at 4000 x 4000 x 2000 (73.4 / 73.2), behind in shorter
 * calls (1000 x 8000 x 1000 31.3 / 34.6, 4000 x 4000 x 520 32.5 / 39.0). */
static int off_lines(vkblas_dtype_t t, uint32_t K, const void* p, uint32_t ld) {
    return t != VKBLAS_DT_F32 && K >= 512 && (((uintptr_t)p | (uint64_t)ld * 2) & 127) != 0;
}

static operand as_is(const void* p, uint32_t ld, uint32_t S, uint32_t M, uint32_t N) {
    operand o = {p, ld, S, M, N, M, N, 0, 0};
    return o;
}
/* ... copied, to Mp x Np; Np in whole 16-byte units */
static void pad_to(operand* o, uint32_t Mp, uint32_t Np) {
    o->copy = 1;
    o->Mp = Mp;
    o->Np = Np;
    o->ld = Np;
    o->p = NULL;                 /* in the workspace: aligned */
}
static void place(op_call* c, operand* o, vkblas_dtype_t t) {
    if (o->copy) o->off = buf(c, (uint64_t)o->S * o->Mp * o->Np * type_size(t));
}
/* After room(): a call's copies, gathered by bring() and launched by brought()
 * together with the scalars of a cross entropy's gradient (scale, or NULL). */
typedef struct {
    vkb_pad_job job[VKB_PAD_JOBS];
    int n;
} copies;
static void bring(op_call* c, copies* j, operand* o, const void* src, uint32_t lds) {
    if (!o->copy) return;
    void* d = at(c, o->off);
    o->p = d;
    j->job[j->n++] = (vkb_pad_job){src, d, lds, o->S, o->M, o->N, o->Mp, o->Np};
}
static int brought(op_call* c, const copies* j, vkblas_dtype_t t, const vkb_scale* scale) {
    return (j->n == 0 && !scale) || step(c, vkb_launch_pad(t, j->job, j->n, scale, c->stream), 0);
}

/* A copied row's columns: rows start on whole lines (bf16 gradient of a cross
 * entropy 174 x 41152 x 2084 as 2112 columns 372 us, as 2088 417) */
static uint32_t line_k(vkblas_dtype_t t, uint32_t K) { return (uint32_t)round_up(K, K > 64 ? 64 : vec_of(t)); }
/* x (M x K) and w (S of N x K) for x w^T inside the pipelined kernel: copied
 * where they have to be and the product is worth it (us, without / with copies,
 * K = 1001: bf16 gated 300 x 500, 0.6 GFLOP, 22.7 / 15.0, 500 x 1000 25.3 / 17.0, xent
 * 300 x 1000 23.3 / 19.5; below 0.5 GFLOP small tiles take such calls in 10.8.  fp32
 * gains from about 6 GFLOP on: gated 1000 x 2000 91 / 75, xent 4000 x 4000 318 / 253; before
 * that the copies cost more: 1000 x 2000 62 / 75, 300 x 1000 24.9 / 31.2). */
static int fusable(vkblas_dtype_t type, uint32_t M, uint32_t N, uint32_t K, operand* x, operand* w, uint32_t cols,
                   vkb_op_args* a) {
    const uint32_t Kp = K % vec_of(type) ? line_k(type, K) : K;
    const int rx = Kp != K || off_units(type, x->p, x->ld) || (N >= 1000 && off_lines(type, K, x->p, x->ld));
    const int rw = Kp != K || off_units(type, w->p, w->ld) || (M >= 1000 && off_lines(type, K, w->p, w->ld));
    operand px = *x, pw = *w;
    if (rx || rw) {
        if (2.0 * M * w->S * w->M * K < 5e8) return 0;
        if (rx) pad_to(&px, x->Mp, line_k(type, K));
        if (rw) pad_to(&pw, w->Mp, line_k(type, K));
    }
    if (!op_plan(type, M, N, Kp, px.p, px.ld, pw.p, pw.ld, cols, a)) return 0;
    *x = px;
    *w = pw;
    return 1;
}
/* x and w for a joined product: copied where their rows lie off 16-byte units
 * and the product is worth it.  Returns the product's K. */
static uint32_t joinable(vkblas_dtype_t type, uint32_t M, uint32_t K, operand* x, operand* w) {
    const int off = K % vec_of(type) != 0;
    if (2.0 * M * w->S * w->M * K < 5e8) return K;
    const uint32_t Kp = off ? K <= 128 ? 128 : (uint32_t)round_up(K, 64) : K;   /* its K steps, two at least */
    if (off || off_units(type, x->p, x->ld)) pad_to(x, x->Mp, Kp);
    if (off || off_units(type, w->p, w->ld)) pad_to(w, w->Mp, Kp);
    return Kp;
}
/* the arguments with the operands where they are now */
static void bound(vkb_op_args* a, const operand* x, const operand* w) {
    a->x = x->p;
    a->w = w->p;
    a->ldx = x->ld;
    a->ldw = w->ld;
}

/* ------------------------------------------------------------- few rows */

/* Whether the one-pass kernels take a call; off: some operand's rows lie off
 * 16-byte units, which the kernels that take more rows at a time have no fast
 * form for.
 * Forward: up to `rows` rows, and 16 (VKB_FEW of many weight rows) where off (us,
 * other kernels / these: gated fp16 1 x 14336 x 4096 36.9 / 34.4, 2 x 1344 x 310 9.4 /
 * 6.3, bf16 27 x 11264 x 1658 44.7 / 23; logits bf16 5 x 107712 x 6965 883 / 410).
 * Backward: up to 8 rows, where off or the weight is so small that launches
 * count (R K elements, us: bf16 3 x 3584 x 128 15.5 / 11.2, fp16 2 x 75421 x 3456,
 * odd, 576 / 308; but 3 x 13144 x 5312 86 / 121: two passes on MFMAs, each at the
 * full rate of reads or of writes). */
static int few_forward(vkblas_dtype_t t, uint32_t M, uint64_t R, uint32_t K, uint32_t rows, int off) {
    return K >= vec_of(t) && (M <= rows || (off && (M <= 16 || (M <= VKB_FEW && vkb_few_mfma(M, R)))));
}
static int few_backward_rows(vkblas_dtype_t t, uint32_t M, uint32_t R, uint32_t K, int off) {
    return K >= vec_of(t) && M <= 8 && (off || (uint64_t)R * K <= 2u << 20);
}

/* D's two products in one pass; p: everything but the division and part. */
static vkblas_status_t few_backward(op_call* c, vkblas_dtype_t type, vkblas_dtype_t dw_type, vkb_few_backward* p,
                                    int glu, size_t o_part, uint32_t slices, void* dx, uint32_t lddx) {
    p->part = dx ? (float*)at(c, o_part) : NULL;
    if (step(c, vkb_launch_few_backward(type, p->dw ? dw_type : type, p, glu, c->stream), p->dw != NULL) && dx)
        step(c, vkb_launch_few_reduce(type, p->part, slices, p->M, p->K, dx, lddx, c->stream), 1);
    return op_end(c, VKBLAS_KERNEL_FEW);
}

/* Whether the two products of a gradient run side by side (pair.hip): where
 * both sums are short enough for four waves and no kernel for more columns is
 * ahead (us, one after the other / side by side, M R K:
 *  16-bit, M and R up to 1024: 97 384 256 13.7 / 11.1, 512 512 512 13.3 / 10.6, 1000 1000
 *   512 24.1 / 18.6; past them 1200 1000 512 26.3 / 27.6, 1000 1200 512 26.0 / 26.3; K up to
 *   1280: 512 1024 1024 21.4 / 20.5, 1280 21.0 / 23.0, 1536 20.9 / 29.8, 64 1024 4096 16.5 /
 *   34; R K up to 2 Mi: 166 3328 944 25.2 / 31.5;
 *  short K, up to 256, and M to 4096: 1547 512 64 27.3 / 20.4; past them 3000 1000 320
 *   41.3 / 42.9, 5000 1000 200 41.1 / 59.9;
 *  fp32, M and R up to 2560: 100 1000 1024 22.4 / 16.2, 103 560 2240 29.2 / 20.7, 1000 2500
 *   300 78.0 / 62.9; up to 64 rows K up to 512: 64 1000 512 14.8 / 13.9, 29 640 4456 22.8 /
 *   29.1 (64 1000 1024, 19.1 / 14.4, is given away);
 *  up to 2 GFLOP: 1000 2000 500 71.1 / 70.9, and 106.2 / 105.9 for K = 700 (long rows with a
 *   short K would still gain: bf16 3000 2000 200 54.8 / 49.6, fp32 1000 3000 300 85.8 / 76.2)). */
static int pairs(vkblas_dtype_t t, uint32_t M, uint32_t R, uint32_t K, uint32_t ldd, uint32_t ldw, uint32_t ldx) {
    const int fits = t == VKBLAS_DT_F32 ? M <= 2560 && R <= 2560 && (M > 64 || K <= 512)
                   : (M <= 1024 && R <= 1024 && (K % 8 || K <= 1280) && (uint64_t)R * K <= 2u << 20) ||
                         (M <= 4096 && R <= 2560 && K <= 256);
    return fits && 2.0 * M * R * K <= 2e9 && vkb_pair_fits(t, M, R, K, ldd, ldw, ldx);
}
static int pair(op_call* c, vkblas_dtype_t t, vkblas_dtype_t wt, uint32_t M, uint32_t R, uint32_t K, const void* d,
                uint32_t ldd, const void* w, uint32_t ldw, void* dx, uint32_t lddx, scalars sx, const void* x,
                uint32_t ldx, void* dw, uint32_t lddw, scalars sw) {
    c->path = VKBLAS_PATH_TILE64;
    const vkb_pair_scalars px = {sx.alpha, sx.beta, sx.alpha_dev, sx.beta_dev};
    const vkb_pair_scalars pw = {sw.alpha, sw.beta, sw.alpha_dev, sw.beta_dev};
    return step(c, vkb_launch_pair(t, wt, M, R, K, d, ldd, w, ldw, dx, lddx, &px, x, ldx, dw, lddw, &pw, c->stream), 1);
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
    /* Few rows all in one launch, without partial sums (us, with / this, bf16: 139 x
     * 15104 21.7 / 9.2, 500 x 4096 16.7 / 10.6, 1000 x 4096 18.6 / 18.5, 1000 x 12000
     * 28 / 29.6, 2000 x 2000 16.1 / 22.3); dw and db first where dx takes the place of
     * their operands. */
    if (M <= (N <= 4096 ? 1024u : 512u) && !vkb_layer_norm_long(N)) {
        const int apart = dx && (dw || db) && (dx == dy || dx == x);
        if (room(&c) != VKBLAS_OK) return c.st;
        if (!apart || step(&c, vkb_launch_layer_norm_few(type, w_type, M, N, dy, lddy, x, ldx, w, mean, rstd, NULL, 0, dw,
                                                         db, g_type, beta, stream), 1))
            step(&c, vkb_launch_layer_norm_few(type, w_type, M, N, dy, lddy, x, ldx, w, mean, rstd, dx, lddx,
                                               apart ? NULL : dw, apart ? NULL : db, g_type, beta, stream), 1);
        return op_end(&c, VKBLAS_KERNEL_NORM);
    }
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

/* Whether the gated projection runs on small tiles that take both halves of w
 * (glu_direct.hip); off: some operand's rows lie off 16-byte units.  Those tiles win
 * where the launches and the fill of a pipeline are most of the time (us, other
 * kernels / these, the same inputs each pass, tiles of 32 x 16 in brackets; other
 * inputs each pass: fp32 200 x 500 x 784 12.1 / 10.0, bf16 100 x 250 x 1024 10.2 / 6.9,
 * 400 x 500 x 784 11.4 / 8.6):
 *  - fp32 as a product and a pass over it: 200 x 500 x 784 11.2 / 9.0, 1000 x 60 x 96
 *    7.9 / 3.9, 1000 x 500 x 301 20.6 / 12.2; past K = 512 from K / 8 tiles on: 64 x 500
 *    x 1536 (64) 14.7 / 17.6, 400 x 250 x 2048 (208) 27.1 / 22.5; up to 16 rows the
 *    decode kernels win past K = 512: 12 x 500 x 784 7.0 / 7.8; K = 4096 32.2 / 38.0;
 *  - 16-bit against the pipelined kernel: 200 x 500 x 256 8.4 / 3.8, 100 x 250 x 1024
 *    10.1 / 6.4, 400 x 500 x 784 (416) 9.7 / 7.9, x 1024 10.7 / 10.2; 400 x 1024 x 512
 *    (832) 7.4 / 10.8; against a product and a pass: 200 x 250 x 2048 13.0 / 9.9, x 4096
 *    17.0 / 16.8; 12 x 500 x 784 6.0 / 4.8, x 2048 6.2 / 8.1;
 *  - 16-bit off 16-byte units until copies pay: 200 x 500 x 1001 14.2 / 10.9, 400 x 500
 *    x 1001 (copied) 14.9 / 19.5. */
static int glu_direct(vkblas_dtype_t t, uint32_t M, uint32_t N, uint32_t K, uint32_t ldx, uint32_t ldw, int off) {
    const uint64_t t32 = (uint64_t)((M + 31) / 32) * ((N + 15) / 16), t64 = (uint64_t)((M + 63) / 64) * ((N + 31) / 32);
    const double flops = 4.0 * M * N * K;
    if (t64 > 256 || K > 2048 || !vkb_glu_direct_fits(t, M, N, K, ldx, ldw)) return 0;
    if (t == VKBLAS_DT_F32) return flops <= 1e9 && (K <= 512 || (M > 16 && t32 >= K / 8));
    if (M <= 16) return K <= 1024 && t32 <= 256;
    return off ? flops < 5e8 : t32 <= (K < 1024 ? 512 : 256);
}

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
    operand ox = as_is(x, ldx, 1, M, K), ow = as_is(w, ldw, 2, N, K);
    const int off = K % vec_of(type) || off_units(type, x, ldx) || off_units(type, w, ldw);
    if (few_forward(type, M, 2 * (uint64_t)N, K, 4, off)) {
        if (room(&c) != VKBLAS_OK) return c.st;
        const vkb_few_forward p = {x, w, h, gu, ldx, ldw, ldh, ldgu, M, N, K, (int)act};
        step(&c, vkb_launch_few_forward(type, &p, 1, stream), 1);
        return op_end(&c, VKBLAS_KERNEL_FEW);
    }
    if (glu_direct(type, M, N, K, ldx, ldw, off)) {
        if (room(&c) != VKBLAS_OK) return c.st;
        c.path = VKBLAS_PATH_TILE64;
        step(&c, vkb_launch_glu_direct(type, act, M, N, K, x, ldx, w, ldw, h, ldh, gu, ldgu, stream), 1);
        return op_end(&c, VKBLAS_KERNEL_FUSED);
    }
    if (fusable(type, M, N, K, &ox, &ow, 128, &a)) {
        place(&c, &ox, type);
        place(&c, &ow, type);
        if (room(&c) != VKBLAS_OK) return c.st;
        copies jobs = {.n = 0};
        bring(&c, &jobs, &ox, x, ldx);
        bring(&c, &jobs, &ow, w, ldw);
        if (brought(&c, &jobs, type, NULL)) {
            bound(&a, &ox, &ow);
            step(&c, vkb_launch_glu(&a, act, h, ldh, gu, ldgu, stream), 1);
        }
        return op_end(&c, VKBLAS_KERNEL_FUSED);
    }
    /* both projections in fp32, some rows at a time, then the join; an fp32
     * gu takes them itself */
    const int direct = type == VKBLAS_DT_F32 && gu;
    const size_t es = type_size(type);
    uint64_t rows = direct ? M : JOIN_BYTES / ((uint64_t)8 * N);
    if (rows < 64) rows = 64;
    if (rows > M) rows = M;
    const uint32_t ldz = direct ? ldgu : (uint32_t)round_up(2 * N, 4);
    const uint32_t Kp = joinable(type, M, K, &ox, &ow);
    need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, (uint32_t)rows, 2 * N, Kp, ox.p, ox.ld, ow.p, ow.ld,
              ldz);
    if (M % rows)   /* (from an address that the program's x has; a copy is aligned) */
        need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, (uint32_t)(M % rows), 2 * N, Kp,
                  ox.copy ? NULL : (const char*)x + (M - M % rows) * ldx * es, ox.ld, ow.p, ow.ld, ldz);
    place(&c, &ox, type);
    place(&c, &ow, type);
    const size_t o_z = direct ? 0 : buf(&c, rows * ldz * sizeof(float));
    if (room(&c) != VKBLAS_OK) return c.st;
    copies jobs = {.n = 0};
    bring(&c, &jobs, &ox, x, ldx);
    bring(&c, &jobs, &ow, w, ldw);
    int ok = brought(&c, &jobs, type, NULL);
    for (uint64_t m = 0; ok && m < M; m += rows) {
        const uint32_t n = (uint32_t)(M - m < rows ? M - m : rows);
        float* z = direct ? (float*)gu : (float*)at(&c, o_z);
        ok = product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, n, 2 * N, Kp, host_scalars(1.0f, 0.0f),
                     (const char*)ox.p + m * ox.ld * es, ox.ld, ow.p, ow.ld, z, ldz, direct) &&
             step(&c, vkb_launch_glu_join(type, act, n, N, z, ldz, (char*)h + m * ldh * es, ldh,
                                          direct || !gu ? NULL : (char*)gu + m * ldgu * es, ldgu, stream), 1);
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
    if (!dgu && few_backward_rows(type, M, 2 * N, K,
                                  K % vec_of(type) || N % 4 || off_units(type, x, ldx) || off_units(type, w, ldw))) {
        vkb_few_backward p = {.x = x, .w = w, .dw = dw, .ldx = ldx, .ldw = ldw, .lddw = lddw, .M = M, .R = 2 * N, .K = K,
                              .beta = beta, .dh = dh, .gu = gu, .lddh = lddh, .ldgu = ldgu, .act = (int)act};
        const uint32_t slices = vkb_few_slices(type, &p);
        const size_t o_part = dx ? buf(&c, (uint64_t)slices * M * K * sizeof(float)) : 0;
        if (room(&c) != VKBLAS_OK) return c.st;
        return few_backward(&c, type, dw_type, &p, 1, o_part, slices, dx, lddx);
    }
    /* The two products as the fast kernels take them, where their work is
     * worth the copies (from 4 GFLOP each on, 2 in fp32) and the layout of [dG | dU] is
     * this call's own: K in whole 16-byte units (columns of both results), M
     * (which dw sums over) in whole pairs of K steps, and N (dx sums over both
     * halves) so that 2 N is, for an odd N from 128 rows on, else from 1024.
     * us, without / with copies, M N K: bf16 1000 1000 1001 53.6 / 45.3, 1000 2000 1001
     * 88 / 62, 1000 2003 1024 84 / 51 (300 1000 1001, 1.2 GFLOP, 34.7 / 33.7); M alone
     * off, 1001 2048 1024, 41.7 / 43.9; fp32 500 1003 1024 73 / 85, 1001 1003 1024 103 /
     * 115, 1001 1024 1024 103 / 107.  N alone: bf16 128 4003 4096 111 / 100, 300 4003
     * 2048 108 / 76, fp32 512 2003 1024 132 / 120; an even N 512 4040 2048 73 / 84,
     * 2048 4040 2048 158 / 160. */
    const size_t es = type_size(type);
    const uint32_t vec = vec_of(type), steps = type == VKBLAS_DT_F32 ? 64 : 128;
    const int big = 4.0 * M * N * K >= (type == VKBLAS_DT_F32 ? 2e9 : 4e9);
    uint32_t Mp = M, Np = N, Kp = K;
    if (big && K % vec) Kp = (uint32_t)round_up(K, vec);
    if (big && !dgu && dw && M % steps) Mp = (uint32_t)round_up(M, steps);
    if (big && !dgu && N % (steps / 2) && M >= (2 * N % vec ? 128 : 1024)) Np = (uint32_t)round_up(N, steps / 2);
    operand ox = as_is(x, ldx, 1, M, K), ow = as_is(w, ldw, 2, N, K);
    if (dw && big && (Mp != M || Kp != K || off_units(type, x, ldx))) pad_to(&ox, Mp, (uint32_t)round_up(K, vec));
    if (dx && big && (Np != N || Kp != K || off_units(type, w, ldw))) pad_to(&ow, Np, (uint32_t)round_up(K, vec));
    const uint32_t ldd = dgu ? lddgu : (uint32_t)round_up(2 * Np, 8);
    /* results of other sizes than the program's go by the workspace; a dw that
     * adds to what is there is rounded once, after that */
    const int px = dx && Kp != K, pw = dw && (Kp != K || Np != N);
    const vkblas_dtype_t wt = pw && beta != 0.0f ? VKBLAS_DT_F32 : dw_type;
    const uint32_t ldxo = px ? Kp : lddx, ldwo = pw ? Kp : lddw;
    const int both = dx && dw && !px && !pw && Mp == M && pairs(type, M, 2 * N, K, ldd, ow.ld, ox.ld);
    if (dx && !both) need_gemm(&c, type, type, VKBLAS_OP_N, VKBLAS_OP_N, M, Kp, 2 * Np, dgu, ldd, ow.p, ow.ld, ldxo);
    if (dw && !both) need_gemm(&c, type, wt, VKBLAS_OP_T, VKBLAS_OP_N, 2 * Np, Kp, Mp, dgu, ldd, ox.p, ox.ld, ldwo);
    const size_t o_d = dgu ? 0 : buf(&c, (uint64_t)Mp * ldd * es);
    place(&c, &ox, type);
    place(&c, &ow, type);
    const size_t o_x = px ? buf(&c, (uint64_t)M * Kp * es) : 0;
    const size_t o_w = pw ? buf(&c, (uint64_t)2 * Np * Kp * type_size(wt)) : 0;
    if (room(&c) != VKBLAS_OK) return c.st;
    void *d = dgu ? dgu : at(&c, o_d), *xo = px ? at(&c, o_x) : dx, *wo = pw ? at(&c, o_w) : dw;
    copies jobs = {.n = 0};
    bring(&c, &jobs, &ox, x, ldx);
    bring(&c, &jobs, &ow, w, ldw);
    int ok = step(&c, vkb_launch_glu_join_backward(type, act, M, N, dh, lddh, gu, ldgu, d, ldd, Mp, Np, stream),
                  dgu != NULL) &&
             brought(&c, &jobs, type, NULL);
    if (ok && both) {
        pair(&c, type, dw_type, M, 2 * N, K, d, ldd, ow.p, ow.ld, dx, lddx, host_scalars(1.0f, 0.0f), ox.p, ox.ld, dw, lddw,
             host_scalars(1.0f, beta));
        return op_end(&c, VKBLAS_KERNEL_JOINED);
    }
    if (ok && dx)
        ok = product(&c, type, type, VKBLAS_OP_N, VKBLAS_OP_N, M, Kp, 2 * Np, host_scalars(1.0f, 0.0f), d, ldd, ow.p,
                     ow.ld, xo, ldxo, !px);
    if (ok && dw)
        ok = product(&c, type, wt, VKBLAS_OP_T, VKBLAS_OP_N, 2 * Np, Kp, Mp, host_scalars(1.0f, pw ? 0.0f : beta), d,
                     ldd, ox.p, ox.ld, wo, ldwo, !pw);
    vkb_unpad_job out[2];
    int n = 0;
    if (px) out[n++] = (vkb_unpad_job){xo, dx, Kp, lddx, 1, M, K, M, (int)type, (int)type, 0.0f};
    if (pw) out[n++] = (vkb_unpad_job){wo, dw, Kp, lddw, 2, N, K, Np, (int)wt, (int)dw_type, beta};
    if (ok && n) step(&c, vkb_launch_unpad(out, n, stream), 1);
    return op_end(&c, VKBLAS_KERNEL_JOINED);
}

/* --------------------------------------------------- linear cross entropy */

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
    operand ox = as_is(x, ldx, 1, M, K), ow = as_is(w, ldw, 1, V, K);
    if (fusable(type, M, V, K, &ox, &ow, 256, &a)) {
        const uint32_t S = vkb_xent_slices(&a);
        place(&c, &ox, type);
        place(&c, &ow, type);
        const size_t o_p = buf(&c, (uint64_t)S * M * 2 * sizeof(float)), o_t = buf(&c, (uint64_t)M * sizeof(float));
        if (room(&c) != VKBLAS_OK) return c.st;
        float *parts = at(&c, o_p), *zt = at(&c, o_t);
        copies jobs = {.n = 0};
        bring(&c, &jobs, &ox, x, ldx);
        bring(&c, &jobs, &ow, w, ldw);
        if (brought(&c, &jobs, type, NULL)) {
            bound(&a, &ox, &ow);
            if (step(&c, vkb_launch_xent_stats_op(&a, target, parts, zt, stream), 0))
                step(&c, vkb_launch_xent_finish(M, V, S, parts, zt, target, ignore_index, loss, lse, stream), 1);
        }
        return op_end(&c, VKBLAS_KERNEL_FUSED);
    }
    const uint32_t n = piece_columns(M, V, JOIN_BYTES, sizeof(float)), ldz = (uint32_t)round_up(n, 4);
    const uint32_t last = V % n;
    const uint32_t per = (n + VKB_XENT_SLICE - 1) / VKB_XENT_SLICE;   /* slices of a piece; the last may have fewer */
    const uint32_t S = V / n * per + (last + VKB_XENT_SLICE - 1) / VKB_XENT_SLICE;
    const int rows = n == V && V <= VKB_XENT_ROW;                     /* one kernel for a row's statistics and loss */
    const int few = n == V && few_forward(type, M, V, K, 0,
                                          K % vec_of(type) || off_units(type, x, ldx) || off_units(type, w, ldw));
    const uint32_t Kp = few ? K : joinable(type, M, K, &ox, &ow);
    need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, n, Kp, ox.p, ox.ld, ow.p, ow.ld, ldz);
    if (last) need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, last, Kp, ox.p, ox.ld, ow.p, ow.ld, ldz);
    place(&c, &ox, type);
    place(&c, &ow, type);
    const size_t o_z = buf(&c, (uint64_t)M * ldz * sizeof(float));
    const size_t o_p = buf(&c, (uint64_t)S * M * 2 * sizeof(float));
    const size_t o_t = buf(&c, (uint64_t)M * sizeof(float));
    if (room(&c) != VKBLAS_OK) return c.st;
    float *z = at(&c, o_z), *parts = at(&c, o_p), *zt = at(&c, o_t);
    copies jobs = {.n = 0};
    bring(&c, &jobs, &ox, x, ldx);
    bring(&c, &jobs, &ow, w, ldw);
    int ok = brought(&c, &jobs, type, NULL);
    uint32_t slice = 0;
    for (uint64_t v = 0; ok && v < V; v += n, slice += per) {
        const uint32_t cols = (uint32_t)(V - v < n ? V - v : n);
        const vkb_few_forward fw = {x, w, z, NULL, ldx, ldw, ldz, 0, M, V, K, 0};
        ok = (few ? step(&c, vkb_launch_few_forward(type, &fw, 0, stream), 0)
                  : product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, cols, Kp, host_scalars(1.0f, 0.0f),
                            ox.p, ox.ld, (const char*)ow.p + v * ow.ld * type_size(type), ow.ld, z, ldz, 0)) &&
             (rows ? step(&c, vkb_launch_xent_rows(M, V, z, ldz, target, ignore_index, loss, lse, stream), 1)
                   : step(&c, vkb_launch_xent_stats(M, cols, (uint32_t)v, z, ldz, target,
                                                    parts + (uint64_t)slice * M * 2, zt, stream), 0));
    }
    if (ok && !rows) step(&c, vkb_launch_xent_finish(M, V, S, parts, zt, target, ignore_index, loss, lse, stream), 1);
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
    const int off = K % vec_of(type) || off_units(type, x, ldx) || off_units(type, w, ldw);
    if (few_backward_rows(type, M, V, K, off || V % 8)) {
        const uint32_t ldz = (uint32_t)round_up(V, 4);
        vkb_few_backward p = {.x = x, .w = w, .dw = dw, .ldx = ldx, .ldw = ldw, .lddw = lddw, .M = M, .R = V, .K = K,
                              .beta = beta, .lse = lse, .dloss = dloss, .ldz = ldz, .ignore = ignore_index,
                              .target = target};
        if (!off) need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, V, K, x, ldx, w, ldw, ldz);
        const uint32_t slices = vkb_few_slices(type, &p);
        const size_t o_z = buf(&c, (uint64_t)M * ldz * sizeof(float));
        const size_t o_part = dx ? buf(&c, (uint64_t)slices * M * K * sizeof(float)) : 0;
        if (room(&c) != VKBLAS_OK) return c.st;
        float* z = at(&c, o_z);
        p.z = z;
        const vkb_few_forward fw = {x, w, z, NULL, ldx, ldw, ldz, 0, M, V, K, 0};
        const int ok = off ? step(&c, vkb_launch_few_forward(type, &fw, 0, stream), 0)
                           : product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, V, K,
                                     host_scalars(1.0f, 0.0f), x, ldx, w, ldw, z, ldz, 0);
        if (!ok) return op_end(&c, VKBLAS_KERNEL_FEW);
        return few_backward(&c, type, dw_type, &p, 0, o_part, slices, dx, lddx);
    }
    /* D of a piece of the vocabulary at a time, in type: from the pipelined
     * kernel, or over the piece's logits in fp32 (fp32: in their place).
     * Where the products' work is worth it, their sums run over whole steps (us,
     * without / with, M V K: bf16, V odd, from 1 GFLOP: 500 4003 512 46.7 / 41.5, 1000
     * 8003 512 105 / 59, below it 300 2003 512 27.8 / 32.3; V in units of 8 from 40
     * GFLOP: 1000 40040 512 214 / 215, 2000 40040 1024 578 / 577, below it 500 4040 512
     * 35.7 / 41.6; fp32 from 2 GFLOP: 1000 8003 512 277 / 214, 500 8003 256 92 / 95;
     * the rows, in fp32 from 2 GFLOP: 500 8000 512 161 / 130, 1001 2000 512 104 / 104,
     * 16-bit from 10: 1000 16000 512 79 / 81, 1000 8000 512 49.7 / 51.1):
     *  - dw's over M rows padded with zeros (D's, and a copy of x);
     *  - dx's over whole tiles of classes, and the rest of the vocabulary by a
     *    padded copy of its rows of w, whose part of dw comes by the workspace;
     *    or a copied w is padded there. */
    const int f32 = type == VKBLAS_DT_F32;
    const size_t es = type_size(type);
    const double work = 2.0 * M * V * K, worth = f32 ? 2e9 : V % 8 ? 1e9 : 4e10;
    vkb_op_args a;
    operand ox = as_is(x, ldx, 1, M, K), ow = as_is(w, ldw, 1, V, K);
    const int fused = fusable(type, M, V, K, &ox, &ow, 256, &a);
    const uint32_t Kp = fused ? a.K : K, steps = f32 ? 64 : 128;
    /* Whether a copy of w, and dw by the workspace, are in whole tiles of classes: where
     * they are of another K, or small enough that the two passes cost less than a tail
     * (us, with a tail / so: bf16 4258 x 817 x 656 83 / 56, 3812 x 17898 x 96 197 / 164,
     * fp32 4994 x 522 x 564 163 / 136) */
    const int vpad = fused && (Kp != K || (V % 128 && (ow.copy || work >= worth) && (uint64_t)V * K * es <= 16u << 20));
    const int whole = fused && (work >= worth || vpad);
    uint32_t Mp = M;
    if (fused && dw && M % steps && work >= (f32 ? 2e9 : 1e10)) Mp = (uint32_t)round_up(M, steps);
    if (ox.copy || Mp != M) pad_to(&ox, Mp, line_k(type, K));
    if (vpad) pad_to(&ow, (uint32_t)round_up(V, 128), line_k(type, K));
    const uint32_t rest = whole && !vpad ? V % 128 : 0;   /* classes that the tail takes */
    uint32_t n = piece_columns(M, V, fused ? PIECE_BYTES : JOIN_BYTES, fused ? es : sizeof(float));
    const uint32_t ldd = (uint32_t)round_up(n, whole ? 128 : 8);
    /* dx adds up over several products in fp32: in dx itself or in the workspace */
    const int several = n < V || rest, acc = dx && (Kp != K || (several && !f32));
    const vkblas_dtype_t xt = acc ? VKBLAS_DT_F32 : type;
    const uint32_t ldxo = acc ? (uint32_t)round_up(Kp, 4) : lddx;
    const int pw = dw && vpad;
    const vkblas_dtype_t wt = (pw || rest) && beta != 0.0f ? VKBLAS_DT_F32 : dw_type;
    const int both = dx && dw && n == V && !rest && !acc && !pw && Mp == M && pairs(type, M, V, K, ldd, ow.ld, ox.ld);
    for (int i = 0; i < 2; ++i) {   /* a piece of n columns, and the last one */
        const uint32_t cols = i ? V % n : n;
        if (!cols) continue;
        const uint32_t main = whole ? (vpad ? (uint32_t)round_up(cols, 128) : cols / 128 * 128) : cols;
        if (!fused)
            need_gemm(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, cols, K, x, ldx, w, ldw, ldd);
        if (both) continue;
        if (dx && main) need_gemm(&c, type, xt, VKBLAS_OP_N, VKBLAS_OP_N, M, Kp, main, NULL, ldd, ow.p, ow.ld, ldxo);
        if (dw && main)
            need_gemm(&c, type, pw ? wt : dw_type, VKBLAS_OP_T, VKBLAS_OP_N, main, Kp, Mp, NULL, ldd, ox.p, ox.ld,
                      pw ? Kp : lddw);
    }
    if (rest) {
        if (dx) need_gemm(&c, type, xt, VKBLAS_OP_N, VKBLAS_OP_N, M, Kp, 128, NULL, ldd, NULL, Kp, ldxo);
        if (dw) need_gemm(&c, type, wt, VKBLAS_OP_T, VKBLAS_OP_N, 128, Kp, Mp, NULL, ldd, ox.p, ox.ld, Kp);
    }
    const size_t o_z = fused ? 0 : buf(&c, (uint64_t)M * ldd * sizeof(float));
    const size_t o_d = f32 && !fused ? o_z : buf(&c, (uint64_t)Mp * ldd * es);
    place(&c, &ox, type);
    place(&c, &ow, type);
    operand tail = as_is(NULL, Kp, 1, rest, K);
    if (rest) {
        pad_to(&tail, 128, Kp);
        place(&c, &tail, type);
    }
    const size_t o_x = acc ? buf(&c, (uint64_t)M * ldxo * sizeof(float)) : 0;
    const size_t o_w = pw || rest ? buf(&c, (pw ? round_up(n, 128) : 128) * Kp * type_size(wt)) : 0;
    const size_t o_s = buf(&c, 8 * sizeof(float));
    if (room(&c) != VKBLAS_OK) return c.st;
    float *z = at(&c, o_z), *scal = f32 ? NULL : (float*)at(&c, o_s);
    void *d = at(&c, o_d), *xo = acc ? at(&c, o_x) : dx, *wo = at(&c, o_w);
    copies jobs = {.n = 0};
    bring(&c, &jobs, &ox, x, ldx);
    bring(&c, &jobs, &ow, w, ldw);
    if (rest && dx) bring(&c, &jobs, &tail, (const char*)w + (uint64_t)(V - rest) * ldw * es, ldw);
    const vkb_scale scale = {scal, beta, !jobs.n && M <= VKB_SCALE_ROWS, M, V, dloss, target, ignore_index};
    int ok = brought(&c, &jobs, type, scal && !scale.find ? &scale : NULL);
    vkb_unpad_job out[2];        /* dw's rows still in the workspace, and dx */
    int outs = 0;
    int summed = 0;              /* dx holds a product already */
    for (uint64_t v = 0; ok && v < V;) {
        const uint32_t cols = (uint32_t)(V - v < n ? V - v : n);
        const uint32_t main = whole ? (vpad ? (uint32_t)round_up(cols, 128) : cols / 128 * 128) : cols;
        const char* wv = (const char*)ow.p + v * ow.ld * es;
        char* dwv = (char*)dw + v * lddw * (dw ? type_size(dw_type) : 0);
        if (fused) {
            bound(&a, &ox, &ow);
            a.w = wv;
            a.N = cols;
            ok = step(&c, vkb_launch_xent_grad_op(&a, Mp, (uint32_t)round_up(cols, whole ? 128 : 8), (uint32_t)v, V,
                                                  target, ignore_index, lse, dloss, scale, d, ldd, stream), 0);
        } else {
            ok = product(&c, type, VKBLAS_DT_F32, VKBLAS_OP_N, VKBLAS_OP_T, M, cols, K, host_scalars(1.0f, 0.0f), x,
                         ldx, wv, ldw, z, ldd, 0) &&
                 step(&c, vkb_launch_xent_grad(type, M, cols, (uint32_t)v, V, z, ldd, target, ignore_index, lse, dloss,
                                               scale, d, ldd, stream), 0);
        }
        if (ok && both) {
            const scalars sx = {1.0f, 0.0f, scal ? scal + 1 : NULL, scal ? scal + 4 : NULL};
            const scalars sw = {1.0f, beta, scal ? scal + 1 : NULL, scal ? scal + 2 : NULL};
            pair(&c, type, dw_type, M, V, K, d, ldd, wv, ow.ld, dx, lddx, sx, ox.p, ox.ld, dw, lddw, sw);
            break;
        }
        /* the whole tiles, then the tail */
        for (int t = 0; ok && t < 2; ++t) {
            const uint32_t rows = t ? cols - (main < cols ? main : cols) : main < cols ? main : cols;   /* of dw */
            const uint32_t sum = t ? 128 : main;
            if (!rows) continue;
            const char* dt = (const char*)d + (t ? (uint64_t)main * es : 0);
            const int by_ws = pw || t;
            if (dw) {
                const scalars sw = {1.0f, by_ws ? 0.0f : beta, scal ? scal + 1 : NULL,
                                    scal ? scal + (by_ws ? 4 : 2) : NULL};
                char* to = dwv + (t ? (uint64_t)main * lddw * type_size(dw_type) : 0);
                if (by_ws && outs) {   /* the workspace's rows make room */
                    ok = step(&c, vkb_launch_unpad(out, outs, stream), 1);
                    outs = 0;
                }
                ok = ok && product(&c, type, by_ws ? wt : dw_type, VKBLAS_OP_T, VKBLAS_OP_N, by_ws ? sum : rows, Kp, Mp, sw,
                             dt, ldd, ox.p, ox.ld, by_ws ? wo : to, by_ws ? Kp : lddw, !by_ws);
                if (by_ws)
                    out[outs++] = (vkb_unpad_job){wo, to, Kp, lddw, 1, rows, K, rows, (int)wt, (int)dw_type, beta};
            }
            if (ok && dx) {
                const scalars sx = {1.0f, summed ? 1.0f : 0.0f, scal ? scal + 1 : NULL,
                                    scal ? scal + (summed ? 3 : 4) : NULL};
                ok = product(&c, type, xt, VKBLAS_OP_N, VKBLAS_OP_N, M, Kp, sum, sx, dt, ldd, t ? tail.p : wv,
                             t ? Kp : ow.ld, xo, ldxo, !acc);
                summed = 1;
            }
        }
        v += cols;
    }
    if (acc) out[outs++] = (vkb_unpad_job){xo, dx, ldxo, lddx, 1, M, K, M, VKB_T_F32, (int)type, 0.0f};
    if (ok && outs) step(&c, vkb_launch_unpad(out, outs, stream), 1);
    return op_end(&c, fused ? VKBLAS_KERNEL_FUSED : VKBLAS_KERNEL_JOINED);
}
