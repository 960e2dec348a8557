// pad.hip — copies between a program's matrices and the workspace: operands
// padded with zeros to sizes and alignments the fast GEMM kernels take, and
// results taken out again.  Bound by memory, 16 bytes a thread; a call's copies
// are one launch (a launch of its own costs each about 4 us; 342 MB 57 us, 6 TB/s).
#include "nn_common.hpp"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

struct PadJobs {
    vkb_pad_job job[VKB_PAD_JOBS];
    uint32_t first[VKB_PAD_JOBS + 1];   // a job's first workgroup
    int n;
    // workgroup 0, where its scal is set: the loss gradients' scale, over these rows
    Scale scale;
    vkb_scale rows;
};

// Row r of matrices of M rows below each other (two at most)
__device__ __forceinline__ void split_row(uint64_t r, uint32_t M, uint32_t& s, uint32_t& m) {
    s = r >= M;
    m = (uint32_t)(r - (s ? M : 0u));
}

__device__ __forceinline__ void find_scale(const PadJobs& p) {
    __shared__ float sh[WORK / 64];
    float top = 0.0f;
    const vkb_scale& r = p.rows;
    for (uint32_t m = threadIdx.x; m < r.M; m += 4 * WORK) {
        float v[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = scale_row(r.dloss, r.target, min(m + i * WORK, r.M - 1), r.V, r.ignore);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, v[i]);
    }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x) return;
    for (uint32_t i = 1; i < WORK / 64; ++i) top = fmaxf(top, sh[i]);
    set_scale(p.scale, top);
}

template <typename T>
__global__ __launch_bounds__(WORK) void pad_kernel(PadJobs p) {
    constexpr int VEC = Elem<T>::VEC;
    if (p.scale.scal && blockIdx.x == 0) {
        find_scale(p);
        return;
    }
    int k = 0;
    while (k + 1 < p.n && blockIdx.x >= p.first[k + 1]) ++k;
    const vkb_pad_job& j = p.job[k];
    const T* A = (const T*)j.src;
    T* P = (T*)j.dst;
    for_chunks((uint64_t)j.S * j.Mp, j.Np / VEC, p.first[k], p.first[k + 1] - p.first[k], [&](uint64_t r, uint32_t c) {
        uint32_t s, m;
        split_row(r, j.Mp, s, m);
        const int64_t n = (int64_t)c * VEC;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (m < j.M) v = ld_chunk(A + ((int64_t)s * j.M + m) * j.ld, n, j.N);
        *(u32x4*)(P + (int64_t)r * j.Np + n) = v;   // the workspace's rows lie on 16-byte units
    });
}

// values of a thread (bf16 174 x 41152 x 2084, its weight's gradient: 4 76 us, 8 68)
constexpr int UNPAD_VEC = 8;

struct UnpadJobs {
    vkb_unpad_job job[2];
    uint32_t first[3];
    int n;
};

// of fp32 or of T, either side
template <typename T>
__global__ __launch_bounds__(WORK) void unpad_kernel(UnpadJobs p) {
    const int k = p.n > 1 && blockIdx.x >= p.first[1];
    const vkb_unpad_job& j = p.job[k];
    const bool sf = j.type == VKB_T_F32, df = j.out_type == VKB_T_F32;
    constexpr int VEC = UNPAD_VEC;
    for_chunks((uint64_t)j.S * j.M, (j.N + VEC - 1) / VEC, p.first[k], p.first[k + 1] - p.first[k],
               [&](uint64_t r, uint32_t c) {
        const int64_t n = (int64_t)c * VEC;
        uint32_t s, m;
        split_row(r, j.M, s, m);
        const int64_t from = ((int64_t)s * j.Mp + m) * j.ldp + n, to = (int64_t)r * j.ldc + n;
        float x[VEC] = {0.f, 0.f, 0.f, 0.f};
        const bool all = n + VEC <= j.N;
        const int have = all ? VEC : (int)(j.N - n);
        auto load = [&](const auto* q, float* out) {
            using E = std::remove_cv_t<std::remove_reference_t<decltype(*q)>>;
            typedef E ev __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));
            if (all) {
                const ev v = *(const ev*)q;
#pragma unroll
                for (int e = 0; e < VEC; ++e) out[e] = (float)v[e];
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (e < have) out[e] = (float)q[e];
            }
        };
        auto store = [&](auto* q) {
            using E = std::remove_reference_t<decltype(*q)>;
            typedef E ev __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));
            if (all) {
                ev v;
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = (E)x[e];
                *(ev*)q = v;
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (e < have) q[e] = (E)x[e];
            }
        };
        if (sf) load((const float*)j.src + from, x);
        else load((const T*)j.src + from, x);
        if (j.beta != 0.0f) {
            float o[VEC] = {0.f, 0.f, 0.f, 0.f};
            if (df) load((const float*)j.dst + to, o);
            else load((const T*)j.dst + to, o);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] += j.beta * o[e];
        }
        if (df) store((float*)j.dst + to);
        else store((T*)j.dst + to);
    });
}

template <typename T>
__global__ __launch_bounds__(WORK) void scale_kernel(uint32_t M, uint32_t N, T* C, int64_t ldc, float beta) {
    for_chunks(M, N, 0, gridDim.x, [&](uint64_t m, uint32_t n) {
        T* c = C + (int64_t)m * ldc + n;
        *c = beta == 0.0f ? (T)0.0f : (T)(beta * (float)*c);
    });
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" int vkb_launch_pad(int type, const vkb_pad_job* jobs, int n, const vkb_scale* scale, void* stream) {
    if (n < 0 || n > VKB_PAD_JOBS || (n == 0 && !scale)) return (int)hipErrorInvalidValue;
    PadJobs p{};
    p.n = n;
    if (scale) p.rows = *scale;
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        p.scale = with_to<T>(p.rows);
        uint32_t at = scale ? 1 : 0;
        for (int i = 0; i < n; ++i) {
            p.job[i] = jobs[i];
            p.first[i] = at;
            at += chunk_blocks((uint64_t)jobs[i].S * jobs[i].Mp, jobs[i].Np / Elem<T>::VEC);
        }
        p.first[n] = at;
        hipLaunchKernelGGL((pad_kernel<T>), dim3(at), dim3(WORK), 0, (hipStream_t)stream, p);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_unpad(const vkb_unpad_job* jobs, int n, void* stream) {
    if (n < 1 || n > 2) return (int)hipErrorInvalidValue;
    UnpadJobs p{};
    p.n = n;
    int type = VKB_T_F32;   // the 16-bit type among them
    uint32_t at = 0;
    for (int i = 0; i < n; ++i) {
        p.job[i] = jobs[i];
        p.first[i] = at;
        at += chunk_blocks((uint64_t)jobs[i].S * jobs[i].M, (jobs[i].N + UNPAD_VEC - 1) / UNPAD_VEC);
        if (jobs[i].type != VKB_T_F32) type = jobs[i].type;
        if (jobs[i].out_type != VKB_T_F32) type = jobs[i].out_type;
    }
    p.first[n] = at;
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((unpad_kernel<T>), dim3(at), dim3(WORK), 0, (hipStream_t)stream, p);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_scale(int type, uint32_t M, uint32_t N, void* C, int64_t ldc, float beta, void* stream) {
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((scale_kernel<T>), dim3(chunk_blocks(M, N)), dim3(WORK), 0, (hipStream_t)stream, M, N, (T*)C,
                           ldc, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
