// nn_pipe.hpp — launchers of the operators that run inside the pipelined GEMM
// kernel; nn_f32.hip, nn_f16.hip and nn_bf16.hip instantiate them by type.
#pragma once
#include "gemm_ops.hpp"
#include "vkb_nn_launch.h"

namespace vkb {

template <typename T, typename OP, int WT, int NST = 2>
static int launch_op(typename OP::Params p, hipStream_t st) {
    constexpr int BM = 2 * WT, BN = OP::GATED ? WT : 2 * WT;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    const uint64_t grid = (uint64_t)p.tiles_m * p.tiles_n;
    if (grid > 0xffffffffull / 256) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((gemm_pipe_kernel<T, T, true, true, WT, NST, OP>), dim3((uint32_t)grid), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}

// The tile of a->tile; 128 x 128 ones of 16-bit operands with four LDS stages
// where the grid is at most one workgroup per CU (their 144 KB allow no
// second; the loads of three K steps in flight instead of one); the kernel
// takes two steps so, or from four on.
template <typename T, typename OP>
static int launch_tiles(const vkb_op_args* a, const typename OP::Params& p, hipStream_t st) {
    if (a->tile == VKB_TILE_256) return launch_op<T, OP, 128>(p, st);
    if constexpr (sizeof(T) == 2) {
        const uint64_t cols = OP::GATED ? 64 : 128;
        const uint64_t grid = (uint64_t)((p.M + 127) / 128) * ((p.N + cols - 1) / cols);
        if (grid <= 256 && (p.K <= 128 || p.K > 192)) return launch_op<T, OP, 64, 4>(p, st);
    }
    return launch_op<T, OP, 64>(p, st);
}

template <typename T, typename P>
static P op_params(const vkb_op_args* a) {
    P p{};
    p.A = a->x;
    p.B = a->w;
    p.lda = a->ldx;
    p.ldb = a->ldw;
    p.M = a->M;
    p.N = a->N;
    p.K = a->K;
    p.batch = p.split = 1;
    p.kps = a->K;
    return p;
}

template <typename T>
static int launch_glu(const vkb_op_args* a, int act_code, void* h, int64_t ldh, void* gu, int64_t ldgu,
                      hipStream_t st) {
    GluParams p = op_params<T, GluParams>(a);
    p.h = h;
    p.ldh = ldh;
    p.gu = gu;
    p.ldgu = ldgu;
    int rc = (int)hipErrorInvalidValue;
    with_act(act_code, [&](auto act) {
        using OP = GluOp<T, decltype(act)::value>;
        rc = launch_tiles<T, OP>(a, p, st);
    });
    return rc;
}

template <typename T>
static int launch_xent_stats(const vkb_op_args* a, const int64_t* target, float* parts, float* zt, hipStream_t st) {
    XentParams p = op_params<T, XentParams>(a);
    p.target = target;
    p.parts = (float2*)parts;
    p.zt = zt;
    return launch_tiles<T, XentStatsOp<T>>(a, p, st);
}

template <typename T>
static int launch_xent_grad(const vkb_op_args* a, uint32_t Ms, uint32_t Ns, uint32_t v0, uint32_t V,
                            const int64_t* target, int64_t ignore, const float* lse, const float* dloss,
                            vkb_scale scale, void* D, int64_t ldd, hipStream_t st) {
    XentParams p = op_params<T, XentParams>(a);
    p.target = target;
    p.Ms = Ms;
    p.Ns = Ns;
    p.v0 = v0;
    p.V = V;
    p.ignore = ignore;
    p.lse = lse;
    p.dloss = dloss;
    p.scale = with_to<T>(scale);
    p.C = D;
    p.ldc = ldd;
    return launch_tiles<T, XentGradOp<T>>(a, p, st);
}

}  // namespace vkb

#define VKB_NN_TYPE(NAME, T)                                                                                         \
    extern "C" int vkb_launch_glu_##NAME(const vkb_op_args* a, int act, void* h, int64_t ldh, void* gu,              \
                                         int64_t ldgu, void* st) {                                                   \
        return vkb::launch_glu<T>(a, act, h, ldh, gu, ldgu, (hipStream_t)st);                                        \
    }                                                                                                                \
    extern "C" int vkb_launch_xent_stats_##NAME(const vkb_op_args* a, const int64_t* target, float* parts,           \
                                                float* zt, void* st) {                                               \
        return vkb::launch_xent_stats<T>(a, target, parts, zt, (hipStream_t)st);                                     \
    }                                                                                                                \
    extern "C" int vkb_launch_xent_grad_##NAME(const vkb_op_args* a, uint32_t Ms, uint32_t Ns, uint32_t v0,          \
                                               uint32_t V, const int64_t* target, int64_t ignore, const float* lse,  \
                                               const float* dloss, vkb_scale scale, void* D, int64_t ldd,            \
                                               void* st) {                                                           \
        return vkb::launch_xent_grad<T>(a, Ms, Ns, v0, V, target, ignore, lse, dloss, scale, D, ldd,                 \
                                        (hipStream_t)st);                                                            \
    }
