// xent.hip — softmax cross entropy on logits that a GEMM computed in pieces
// of the vocabulary: each piece's row statistics, their join into log-sum-exp
// and loss, and the logits' gradient.
//
// A row's statistics over some columns are the pair (top, s): top = max z and
// s = sum exp(z - top), and pairs join by
//   T = max top_i,  S = sum s_i exp(top_i - T),  lse = T + log S.
// Infinities follow the formula: where top is not finite the exponentials
// take 0 in its place, so an all -inf part has s = 0 and drops out of the
// join, a +inf gives s = inf and lse = inf, and a NaN reaches s and lse.
#include "nn_common.hpp"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

constexpr uint32_t THREADS = 256, WAVES = THREADS / 64;

__device__ __forceinline__ float finite_or_0(float x) { return __builtin_isinf(x) ? 0.0f : x; }

__device__ __forceinline__ float block_max(float v, float* sh) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (uint32_t i = 1; i < WAVES; ++i) r = fmaxf(r, sh[i]);
    __syncthreads();
    return r;
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (uint32_t i = 1; i < WAVES; ++i) r += sh[i];
    __syncthreads();
    return r;
}

// One workgroup per row and slice of VKB_XENT_SLICE columns, the slice in
// registers between the two reductions; rows strided over y.
__global__ __launch_bounds__(THREADS) void xent_stats_kernel(uint32_t M, uint32_t n, uint32_t v0, const float* z,
                                                             int64_t ldz, const int64_t* target, float2* parts,
                                                             float* zt) {
    constexpr int NV = VKB_XENT_SLICE / THREADS / 4;
    __shared__ float sh[WAVES];
    const int64_t c0 = (int64_t)blockIdx.x * VKB_XENT_SLICE + threadIdx.x * 4;
    for (uint32_t m = blockIdx.y; m < M; m += gridDim.y) {
        const float* row = z + (int64_t)m * ldz;
        float x[NV][4], top = -INFINITY, s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = c0 + (int64_t)i * THREADS * 4;
            unpack<float>(ld_chunk(row, c, n), x[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (c + e >= n) x[i][e] = -INFINITY;
                top = fmaxf(top, x[i][e]);
            }
        }
        top = block_max(top, sh);
        const float off = finite_or_0(top);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += fast_exp(x[i][e] - off);
        s = block_sum(s, sh);
        if (threadIdx.x == 0) {
            parts[(int64_t)blockIdx.x * M + m] = float2{top, s};
            if (target) {
                const int64_t t = target[m] - v0 - (int64_t)blockIdx.x * VKB_XENT_SLICE;
                if (t >= 0 && t < VKB_XENT_SLICE && target[m] - v0 < n) zt[m] = row[target[m] - v0];
            }
        }
    }
}

// FROWS rows per workgroup of 256, 256 / FROWS threads each: thread j of a row
// joins slices j, j + 256 / FROWS, .., eight loads in flight; then the threads'
// pairs join in LDS.
constexpr int FROWS = 8, FSLICES = THREADS / FROWS;
__global__ __launch_bounds__(THREADS) void xent_finish_kernel(uint32_t M, uint32_t V, uint32_t S, const float2* parts,
                                                              const float* zt, const int64_t* target, int64_t ignore,
                                                              float* loss, float* lse) {
    __shared__ float2 sh[FSLICES][FROWS + 1];
    const uint32_t r = threadIdx.x % FROWS, j = threadIdx.x / FROWS;
    const uint32_t m = blockIdx.x * FROWS + r;
    float top = -INFINITY, s = 0.0f;
    if (m < M)
        for (uint32_t i = j; i < S; i += 8 * FSLICES) {
            float2 p[8];
            float t = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t c = i + k * FSLICES;
                p[k] = c < S ? parts[(int64_t)c * M + m] : float2{-INFINITY, 0.0f};
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) t = fmaxf(t, p[k].x);
            const float off = finite_or_0(t);
            s *= fast_exp(top - off);
#pragma unroll
            for (int k = 0; k < 8; ++k) s += p[k].y * fast_exp(p[k].x - off);
            top = t;
        }
    sh[j][r] = float2{top, s};
    __syncthreads();
    if (j || m >= M) return;
    for (uint32_t i = 1; i < FSLICES; ++i) top = fmaxf(top, sh[i][r].x);
    const float off = finite_or_0(top);
    s = 0.0f;
    for (uint32_t i = 0; i < FSLICES; ++i) s += sh[i][r].y * fast_exp(sh[i][r].x - off);
    const float l = off + logf(s);
    lse[m] = l;
    if (loss) {
        const int64_t t = target[m];
        loss[m] = t == ignore ? 0.0f : (t >= 0 && t < V ? l - zt[m] : __builtin_nanf(""));
    }
}

// A row of at most VKB_XENT_ROW logits, in the registers of one workgroup.
constexpr uint32_t ROW_THREADS = 1024;
__global__ __launch_bounds__(ROW_THREADS) void xent_rows_kernel(uint32_t M, uint32_t V, const float* z, int64_t ldz,
                                                                const int64_t* target, int64_t ignore, float* loss,
                                                                float* lse) {
    constexpr int NV = VKB_XENT_ROW / ROW_THREADS / 4;
    __shared__ float sh[2][ROW_THREADS / 64];
    const uint32_t waves = blockDim.x / 64;
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const float* row = z + (int64_t)m * ldz;
        float x[NV][4], top = -INFINITY, s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = ((int64_t)i * blockDim.x + threadIdx.x) * 4;
            if (c + 3 < V) {
                unpack<float>(ld16_any(row + c), x[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = c + e < V ? row[c + e] : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, x[i][e]);
        top = wave_max(top);
        if ((threadIdx.x & 63) == 0) sh[0][threadIdx.x >> 6] = top;
        __syncthreads();
        for (uint32_t i = 0; i < waves; ++i) top = fmaxf(top, sh[0][i]);
        const float off = finite_or_0(top);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += fast_exp(x[i][e] - off);
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0) sh[1][threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (uint32_t i = 1; i < waves; ++i) s += sh[1][i];
            const float l = off + logf(s);
            lse[m] = l;
            if (loss) {
                const int64_t t = target[m];
                loss[m] = t == ignore ? 0.0f : (t >= 0 && t < V ? l - row[t] : __builtin_nanf(""));
            }
        }
        __syncthreads();   // the next row writes sh again
    }
}

template <typename T>
__global__ __launch_bounds__(WORK) void xent_grad_kernel(uint32_t M, uint32_t n, uint32_t v0, uint32_t V,
                                                            const float* z, int64_t ldz, const int64_t* target,
                                                            int64_t ignore, const float* lse, const float* dloss,
                                                            Scale scale, T* D, int64_t ldd) {
    constexpr int VEC = Elem<T>::VEC;
    const float sc = scale_of<T>(scale, dloss, target, M, V, ignore, blockIdx.x == 0 && threadIdx.x < 64, threadIdx.x & 63);
    for_chunks(M, (n + VEC - 1) / VEC, 0, gridDim.x, [&](uint64_t m, uint32_t k) {
        const int64_t c = (int64_t)k * VEC, t = target[m];
        const float l = lse[m];
        // the three kinds of rows: counted, ignored (all zero), target out of range (all NaN)
        const float w = t == ignore ? 0.0f : (t >= 0 && t < V ? dloss[m] * sc : __builtin_nanf(""));
        float x[VEC];
#pragma unroll
        for (int q = 0; q < VEC; q += 4) unpack<float>(ld_chunk(z + (int64_t)m * ldz, c + q, n), x + q);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float p = fast_exp(x[i] - l) - (c + i == t - v0 ? 1.0f : 0.0f);
            x[i] = t == ignore ? 0.0f : w * p;
        }
        st_chunk(D + (int64_t)m * ldd, c, n, pack<T>(x));
    });
}

}  // namespace
}  // namespace vkb

using namespace vkb;

static uint32_t rows_y(uint32_t M) { return M < 65535u ? M : 65535u; }

extern "C" int vkb_launch_xent_stats(uint32_t M, uint32_t n, uint32_t v0, const float* z, int64_t ldz,
                                     const int64_t* target, float* parts, float* zt, void* stream) {
    hipLaunchKernelGGL(xent_stats_kernel, dim3((n + VKB_XENT_SLICE - 1) / VKB_XENT_SLICE, rows_y(M)), dim3(THREADS), 0,
                       (hipStream_t)stream, M, n, v0, z, ldz, target, (float2*)parts, zt);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_xent_finish(uint32_t M, uint32_t V, uint32_t S, const float* parts, const float* zt,
                                      const int64_t* target, int64_t ignore, float* loss, float* lse, void* stream) {
    const uint64_t groups = ((uint64_t)M + FROWS - 1) / FROWS;
    if (groups > 0xffffffffull / THREADS) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(xent_finish_kernel, dim3((uint32_t)groups), dim3(THREADS), 0,
                       (hipStream_t)stream, M, V, S, (const float2*)parts, zt, target, ignore, loss, lse);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_xent_rows(uint32_t M, uint32_t V, const float* z, int64_t ldz, const int64_t* target,
                                    int64_t ignore, float* loss, float* lse, void* stream) {
    if (V > VKB_XENT_ROW) return (int)hipErrorInvalidValue;
    // whole waves for 16 values a thread
    const uint32_t threads = (V + 1023) / 1024 * 64;
    hipLaunchKernelGGL(xent_rows_kernel, dim3(M < 65536u ? M : 65536u), dim3(threads), 0, (hipStream_t)stream, M, V, z,
                       ldz, target, ignore, loss, lse);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_xent_grad(int type, uint32_t M, uint32_t n, uint32_t v0, uint32_t V, const float* z,
                                    int64_t ldz, const int64_t* target, int64_t ignore, const float* lse,
                                    const float* dloss, vkb_scale scale, void* D, int64_t ldd, void* stream) {
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((xent_grad_kernel<T>), dim3(chunk_blocks(M, chunks_of<T>(n))), dim3(WORK), 0,
                           (hipStream_t)stream, M, n, v0, V, z, ldz, target, ignore, lse, dloss, with_to<T>(scale), (T*)D, ldd);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
