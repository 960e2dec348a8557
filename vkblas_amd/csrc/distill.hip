// distill.hip — distillation from a teacher's top logits, beside the linear
// cross entropy's kernels (xent.hip, gemm_ops.hpp): what of it goes by rows and
// their entries.
//
// With q the teacher's softmax over a row's few entries, p the student's over
// all V classes and T the temperature,
//   loss = T^2 sum_j q_j (log q_j - z_j / T + lse),
//   D_v  = T dloss (p_v - q_v),
// so over the vocabulary both need what a cross entropy needs, log-sum-exp and
// p, and the entries come on top: their logits z_j are dot products of x's row
// with the entries' rows of w, and D's elements at the entries are written over
// by a patch once the tiles are stored.  T's factor in D is taken into dloss.
#include "nn_common.hpp"

namespace vkb {
namespace {

constexpr uint32_t TOP = VKBLAS_DISTILL_TOP, WAVES = WORK / 64;

struct Shared {
    float q[TOP];            // the teacher's logits over T, then its probabilities
    int id[TOP];             // class, or ABSENT, or BAD
    float part[WAVES];
};
constexpr int ABSENT = -1, BAD = -2;

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* sh, F join) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (uint32_t i = 1; i < WAVES; ++i) r = join(r, sh[i]);
    __syncthreads();
    return r;
}

// A row's entries into LDS: classes, and t / T less the largest.  Returns the
// log of their sum of exponentials.  counted: some entry is there and not of
// probability 0 (a NaN is not); bad: some class is past V.
template <typename TT>
__device__ __forceinline__ float teacher(uint32_t n, uint32_t V, const int64_t* top, const TT* t, float inv_t,
                                         Shared& sh, bool& counted, bool& bad) {
    float high = -INFINITY;
    int any = 0, past = 0;
    for (uint32_t j = threadIdx.x; j < n; j += WORK) {
        const int64_t c = top[j];
        const float v = c < 0 ? -INFINITY : (float)t[j] * inv_t;
        sh.id[j] = c < 0 ? ABSENT : c < V ? (int)c : BAD;
        sh.q[j] = v;
        any |= !(v == -INFINITY);
        past |= c >= (int64_t)V;
        high = fmaxf(high, v);
    }
    counted = __syncthreads_or(any) != 0;
    bad = __syncthreads_or(past) != 0;
    high = block_reduce(wave_max(high), sh.part, [](float a, float b) { return fmaxf(a, b); });
    if (high == -INFINITY) high = 0.0f;
    float s = 0.0f;
    for (uint32_t j = threadIdx.x; j < n; j += WORK) {
        sh.q[j] -= high;
        s += fast_exp(sh.q[j]);
    }
    s = block_reduce(wave_sum(s), sh.part, [](float a, float b) { return a + b; });
    return logf(s);
}

// One workgroup per row.  The waves take the entries DOTS at a time: one load of
// x's chunk for DOTS of w's rows.
constexpr uint32_t DOTS = 4;
template <typename T, typename TT>
__global__ __launch_bounds__(WORK) void rows_kernel(uint32_t M, uint32_t V, uint32_t K, const T* x, int64_t ldx,
                                                    const T* w, int64_t ldw, uint32_t n, const int64_t* top,
                                                    int64_t ldtop, const TT* t, int64_t ldt, float temp, float inv_t,
                                                    const float* lse, float* loss, float* z_top) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ Shared sh;
    __shared__ float z[TOP];
    __shared__ uint32_t list[TOP], count;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        bool counted, bad;
        const float log_s = teacher(n, V, top + (int64_t)m * ldtop, t + (int64_t)m * ldt, inv_t, sh, counted, bad);
        // the entries with a class, in order
        if (wave == 0) {
            uint32_t c = 0;
            for (uint32_t j = lane; j - lane < n; j += 64) {
                const bool in = j < n && sh.id[j] >= 0;
                const uint64_t mask = __ballot(in);
                if (in) list[c + __popcll(mask & ((1ull << lane) - 1))] = j;
                c += (uint32_t)__popcll(mask);
            }
            if (lane == 0) count = c;
        }
        __syncthreads();
        const uint32_t there = count;
        const T* xr = x + (int64_t)m * ldx;
        for (uint32_t g = wave * DOTS; g < there; g += WAVES * DOTS) {
            const T* row[DOTS];
            float acc[DOTS];
#pragma unroll
            for (uint32_t e = 0; e < DOTS; ++e) {
                row[e] = w + (int64_t)__builtin_amdgcn_readfirstlane(sh.id[list[min(g + e, there - 1)]]) * ldw;
                acc[e] = 0.0f;
            }
#pragma unroll 2
            for (int64_t k = (int64_t)lane * VEC; k < K; k += 64 * VEC) {
                float a[VEC];
                unpack<T>(ld_chunk(xr, k, K), a);
#pragma unroll
                for (uint32_t e = 0; e < DOTS; ++e) {
                    float b[VEC];
                    unpack<T>(ld_chunk(row[e], k, K), b);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[e] = __builtin_fmaf(a[i], b[i], acc[e]);
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < DOTS; ++e) {
                const float s = wave_sum(acc[e]);
                if (lane == 0 && g + e < there) z[list[g + e]] = s;
            }
        }
        __syncthreads();
        const float l = lse[m];
        float s = 0.0f;
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            const int id = sh.id[j];
            const float v = id == ABSENT ? 0.0f : id == BAD ? __builtin_nanf("") : z[j];
            z_top[(int64_t)m * n + j] = v;
            const float log_q = sh.q[j] - log_s, q = fast_exp(log_q);
            if (id != ABSENT && !(q == 0.0f)) s += q * (log_q - (v * inv_t - l));
        }
        s = block_reduce(wave_sum(s), sh.part, [](float a, float b) { return a + b; });
        if (threadIdx.x == 0) loss[m] = bad ? __builtin_nanf("") : counted ? temp * temp * s : 0.0f;
    }
}

// The backward pass's rows: q of each entry's class (both entries' where a class
// occurs twice), T dloss, and a target for D's kernels: `ignore` where the row
// is not counted, V where it is bad, else the first entry's class, whose
// element the patch writes over.
template <typename TT>
__global__ __launch_bounds__(WORK) void prepare_kernel(uint32_t M, uint32_t V, uint32_t n, const int64_t* top,
                                                       int64_t ldtop, const TT* t, int64_t ldt, float temp, float inv_t,
                                                       const float* dloss, int64_t ignore, float* q_top,
                                                       int64_t* target, float* dl) {
    __shared__ Shared sh;
    __shared__ int first[WAVES];
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        bool counted, bad;
        const float log_s = teacher(n, V, top + (int64_t)m * ldtop, t + (int64_t)m * ldt, inv_t, sh, counted, bad);
        uint32_t at = n;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            sh.q[j] = sh.id[j] == ABSENT ? 0.0f : fast_exp(sh.q[j] - log_s);
            if (sh.id[j] >= 0) at = min(at, j);
        }
        for (int d = 32; d; d >>= 1) at = min(at, (uint32_t)__shfl_xor((int)at, d));
        if ((threadIdx.x & 63) == 0) first[threadIdx.x >> 6] = (int)at;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            const int id = sh.id[j];
            float q = 0.0f;
            if (id >= 0)
                for (uint32_t i = 0; i < n; ++i) q += sh.id[i] == id ? sh.q[i] : 0.0f;
            q_top[(int64_t)m * n + j] = q;
        }
        if (threadIdx.x == 0) {
            uint32_t f = n;
            for (uint32_t i = 0; i < WAVES; ++i) f = min(f, (uint32_t)first[i]);
            target[m] = bad ? (int64_t)V : counted && f < n ? (int64_t)sh.id[f] : ignore;
            dl[m] = temp * dloss[m];
        }
        __syncthreads();
    }
}

// D at the entries whose class lies in columns v0 .. v0 + cols - 1
template <typename T>
__global__ __launch_bounds__(WORK) void patch_kernel(uint32_t M, uint32_t V, uint32_t n, const int64_t* top,
                                                     int64_t ldtop, uint32_t v0, uint32_t cols, float inv_t,
                                                     const float* lse, const float* z_top, const float* q_top,
                                                     const int64_t* target, int64_t ignore, const float* dl,
                                                     const float* scal, T* D, int64_t ldd) {
    const float sc = scal ? scal[0] : 1.0f;
    const uint64_t total = (uint64_t)M * n;
    for (uint64_t i = (uint64_t)blockIdx.x * WORK + threadIdx.x; i < total; i += (uint64_t)gridDim.x * WORK) {
        const uint64_t m = i / n;
        const int64_t id = top[(int64_t)m * ldtop + (int64_t)(i - m * n)], c = id - v0;
        if (id < 0 || c < 0 || c >= cols || target[m] == ignore || target[m] >= V) continue;
        const float p = fast_exp(z_top[i] * inv_t - lse[m]);
        D[(int64_t)m * ldd + c] = (T)(dl[m] * sc * (p - q_top[i]));
    }
}

}  // namespace
}  // namespace vkb

using namespace vkb;

static uint32_t row_blocks(uint32_t M) { return M < 65536 ? M : 65536; }

extern "C" int vkb_launch_distill_rows(int type, int t_type, const vkb_distill* d, uint32_t K, const void* x,
                                       int64_t ldx, const void* w, int64_t ldw, const float* lse, float* loss,
                                       float* z_top, void* stream) {
    const bool ok = with_type(type, [&](auto e) {
        using T = decltype(e);
        auto launch = [&](auto f) {
            using TT = decltype(f);
            hipLaunchKernelGGL((rows_kernel<T, TT>), dim3(row_blocks(d->M)), dim3(WORK), 0, (hipStream_t)stream, d->M,
                               d->V, K, (const T*)x, ldx, (const T*)w, ldw, d->n, d->top, d->ldtop, (const TT*)d->t,
                               d->ldt, d->temp, 1.0f / d->temp, lse, loss, z_top);
        };
        if (t_type == VKB_T_F32) launch(float{});
        else launch(e);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_distill_prepare(int t_type, const vkb_distill* d, const float* dloss, void* stream) {
    const bool ok = with_type(t_type, [&](auto f) {
        using TT = decltype(f);
        hipLaunchKernelGGL((prepare_kernel<TT>), dim3(row_blocks(d->M)), dim3(WORK), 0, (hipStream_t)stream, d->M, d->V,
                           d->n, d->top, d->ldtop, (const TT*)d->t, d->ldt, d->temp, 1.0f / d->temp, dloss, d->ignore,
                           d->q_top, d->target, d->dl);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_distill_patch(int type, const vkb_distill* d, uint32_t v0, uint32_t cols, const float* lse,
                                        const float* z_top, const float* scal, void* D, int64_t ldd, void* stream) {
    const bool ok = with_type(type, [&](auto e) {
        using T = decltype(e);
        hipLaunchKernelGGL((patch_kernel<T>), dim3(chunk_blocks(d->M, d->n)), dim3(WORK), 0, (hipStream_t)stream, d->M,
                           d->V, d->n, d->top, d->ldtop, v0, cols, 1.0f / d->temp, lse, z_top, d->q_top, d->target,
                           d->ignore, d->dl, scal, (T*)D, ldd);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
