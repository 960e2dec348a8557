// pad.hip — copies between a program's matrices and the workspace: operands
// padded with zeros to sizes and alignments the fast GEMM kernels take, and
// results taken out again.  Bound by memory: 16 bytes a thread.
#include "nn_common.hpp"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

constexpr uint32_t THREADS = 256;

// column blocks in x, rows in y (strided: y holds at most 65535)
template <typename T>
static dim3 rows_grid(uint32_t M, uint32_t N) {
    const uint32_t per = THREADS * Elem<T>::VEC;
    return dim3((N + per - 1) / per, M < 65535u ? M : 65535u);
}

template <typename T>
__global__ __launch_bounds__(THREADS) void pad_kernel(uint32_t S, uint32_t M, uint32_t N, const T* A, int64_t lda,
                                                      T* P, uint32_t Mp, uint32_t Np) {
    constexpr int VEC = Elem<T>::VEC;
    const int64_t n = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * VEC;
    if (n >= Np) return;
    for (uint64_t r = blockIdx.y; r < (uint64_t)S * Mp; r += gridDim.y) {
        const uint32_t s = (uint32_t)(r / Mp), m = (uint32_t)(r % Mp);
        u32x4 v = {0u, 0u, 0u, 0u};
        if (m < M) v = ld_chunk(A + ((int64_t)s * M + m) * lda, n, N);
        st_chunk(P + (int64_t)r * Np, n, Np, v);
    }
}

template <typename T, typename C>
__global__ __launch_bounds__(THREADS) void unpad_kernel(uint32_t S, uint32_t M, uint32_t N, const T* P, int64_t ldp,
                                                        uint32_t Mp, C* out, int64_t ldc, float beta) {
    constexpr int VEC = Elem<C>::VEC;
    const int64_t n = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * VEC;
    if (n >= N) return;
    for (uint64_t r = blockIdx.y; r < (uint64_t)S * M; r += gridDim.y) {
        const T* src = P + ((int64_t)(r / M) * Mp + r % M) * ldp;
        C* dst = out + (int64_t)r * ldc;
        float x[VEC], o[VEC];
        if constexpr (sizeof(T) == sizeof(C)) {
            unpack<T>(ld_chunk(src, n, N), x);
        } else {
#pragma unroll
            for (int q = 0; q < VEC; q += Elem<T>::VEC) unpack<T>(ld_chunk(src, n + q, N), x + q);
        }
        if (beta != 0.0f) {
            unpack<C>(ld_chunk(dst, n, N), o);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] += beta * o[i];
        }
        st_chunk(dst, n, N, pack<C>(x));
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void scale_kernel(uint32_t M, uint32_t N, T* C, int64_t ldc, float beta) {
    for (uint32_t m = blockIdx.y; m < M; m += gridDim.y)
        for (int64_t n = (int64_t)blockIdx.x * THREADS + threadIdx.x; n < N; n += (int64_t)gridDim.x * THREADS) {
            T* c = C + (int64_t)m * ldc + n;
            *c = beta == 0.0f ? (T)0.0f : (T)(beta * (float)*c);
        }
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" int vkb_launch_pad(int type, uint32_t S, uint32_t M, uint32_t N, const void* A, int64_t lda, void* P,
                              uint32_t Mp, uint32_t Np, void* stream) {
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        const uint64_t rows = (uint64_t)S * Mp;
        hipLaunchKernelGGL((pad_kernel<T>), rows_grid<T>((uint32_t)(rows < 65535 ? rows : 65535), Np), dim3(THREADS),
                           0, (hipStream_t)stream, S, M, N, (const T*)A, lda, (T*)P, Mp, Np);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_unpad(int type, int out_type, uint32_t S, uint32_t M, uint32_t N, const void* P, int64_t ldp,
                                uint32_t Mp, void* out, int64_t ldc, float beta, void* stream) {
    bool ok = type == out_type || type == VKB_T_F32;
    ok = ok && with_type(out_type, [&](auto t) {
        using C = decltype(t);
        const uint64_t rows = (uint64_t)S * M;
        const dim3 grid = rows_grid<C>((uint32_t)(rows < 65535 ? rows : 65535), N);
        if (type == VKB_T_F32)
            hipLaunchKernelGGL((unpad_kernel<float, C>), grid, dim3(THREADS), 0, (hipStream_t)stream, S, M, N,
                               (const float*)P, ldp, Mp, (C*)out, ldc, beta);
        else
            hipLaunchKernelGGL((unpad_kernel<C, C>), grid, dim3(THREADS), 0, (hipStream_t)stream, S, M, N,
                               (const C*)P, ldp, Mp, (C*)out, ldc, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_scale(int type, uint32_t M, uint32_t N, void* C, int64_t ldc, float beta, void* stream) {
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((scale_kernel<T>), rows_grid<T>(M, N), dim3(THREADS), 0, (hipStream_t)stream, M, N, (T*)C,
                           ldc, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
