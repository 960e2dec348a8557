/*
 * vkb_engine.h — internal entry of the host dispatcher (engine.c) for other
 * translation units of the library (not exported API).
 */
#pragma once
#include <stddef.h>
#include "vkblas_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

/* vkblas_gemm_async with the split-K / decode partials in the caller's
 * device buffer `scratch` of `scratch_bytes` (at least 256-byte aligned):
 * allocates nothing.  A call whose partials need more than scratch_bytes
 * returns VKBLAS_ERR_PARAM before any launch. */
__attribute__((visibility("hidden")))
vkblas_status_t vkb_gemm_with_scratch(vkblas_dtype_t ab_type, vkblas_dtype_t c_type, vkblas_op_t op_a,
                                      vkblas_op_t op_b, uint32_t M, uint32_t N, uint32_t K, float alpha,
                                      const void* A, uint32_t lda, const void* B, uint32_t ldb, float beta,
                                      void* C, uint32_t ldc, uint32_t batch, int64_t stride_a, int64_t stride_b,
                                      int64_t stride_c, vkblas_scalar_mode_t scalar_mode, const void* alpha_dev,
                                      const void* beta_dev, uint32_t split_k, void* stream, void* scratch,
                                      size_t scratch_bytes);

/* Scratch bytes with which vkb_gemm_with_scratch (split_k = 0, batch 1) runs
 * the planner's own plan, its arrival counters included; 0 where that needs
 * none.  *optional: without them vkblas_gemm_async runs a plan without a split
 * (else it fails). */
__attribute__((visibility("hidden")))
size_t vkb_gemm_scratch_bytes(vkblas_dtype_t ab_type, vkblas_dtype_t c_type, vkblas_op_t op_a, vkblas_op_t op_b,
                              uint32_t M, uint32_t N, uint32_t K, uint32_t lda, uint32_t ldb, uint32_t ldc,
                              int aligned, int* optional);

/* A workspace of the calling device and stream (engine.c, "Split-K and decode
 * partials"): held from vkb_ws_acquire (0, or -1: none, and nothing to
 * release) until vkb_ws_release, after the call's last kernel is enqueued.
 * It starts with VKB_WS_HEADER bytes of arrival counters that only GEMMs
 * touch, and must not be held across a GEMM entry point that takes its own. */
typedef struct {
    void* ptr;
    int slot;                    /* locked slot, or -1 */
    int owned;                   /* free ptr on the stream after the kernels */
    void* stream;
} vkb_ws_lease;
__attribute__((visibility("hidden"))) int vkb_ws_acquire(void* stream, size_t bytes, vkb_ws_lease* L);
__attribute__((visibility("hidden"))) void vkb_ws_release(vkb_ws_lease* L);

/* VKBLAS_PROFILE: begin before the call's first kernel, end after its last. */
typedef struct {
    int on;
    double t0, t1;
    void *e0, *e1;               /* hipEvent_t */
} vkb_prof;
__attribute__((visibility("hidden"))) void vkb_prof_begin(vkb_prof* pf, void* stream);
__attribute__((visibility("hidden"))) void vkb_prof_end(vkb_prof* pf, void* stream, const char* what, int ok);

/* A device is there; VKBLAS_TRACE is set; what vkblas_last_path / _kernel report. */
__attribute__((visibility("hidden"))) int vkb_engine_ready(void);
__attribute__((visibility("hidden"))) int vkb_engine_trace(void);
__attribute__((visibility("hidden"))) void vkb_engine_ran(int path, int kernel);

#ifdef __cplusplus
}
#endif
