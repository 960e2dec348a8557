// layer_norm.hip — layer norm of rows and its gradients.
//   mean = sum x / N, var = sum (x - mean)^2 / N, rstd = 1 / sqrt(var + eps),
//   xh = (x - mean) rstd, y = xh w + b
//   dx = rstd (g - sum g / N - xh sum(g xh) / N) with g = dy w,
//   dw = sum_m dy xh, db = sum_m dy
// Bound by memory: each row is read once into registers, between its
// statistics and its result.  A workgroup stays for many rows, so that w and b
// (and in the backward pass the running sums of dw and db) stay in registers
// too, and the next row's loads leave before the present row's reductions.
// 16-byte accesses of any alignment; columns past N are zeros that no
// statistic counts.
#include <type_traits>
#include "nn_common.hpp"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

// A row's columns over WAVES waves: thread t holds the 16-byte chunks
// t + i TPR, i < EPT / VEC.  WAVES == 1: four rows per workgroup, one per
// wave, no barrier.
template <typename T, int WAVES, int EPT>
struct RowMap {
    static constexpr int VEC = Elem<T>::VEC, NV = EPT / VEC;
    static constexpr int TPR = WAVES * 64;                   // threads per row
    static constexpr int RPB = WAVES == 1 ? 4 : 1;           // rows at a time
    static constexpr int THREADS = TPR * RPB;
    // sixteen waves leave 128 registers a thread: with 16 values, w and b are
    // read again for every row and no row is loaded ahead
    static constexpr bool LEAN = WAVES == 16 && EPT == 16;
    static_assert(EPT % VEC == 0, "whole chunks");
};

template <typename W, typename T, int WAVES, int EPT>
__device__ __forceinline__ void load_params(const W* w, int t, uint32_t N, float none, float* out) {
    using R = RowMap<T, WAVES, EPT>;
#pragma unroll
    for (int i = 0; i < R::NV; ++i) {
        const int64_t c = (int64_t)(t + i * R::TPR) * R::VEC;
        if (!w) {
#pragma unroll
            for (int e = 0; e < R::VEC; ++e) out[i * R::VEC + e] = none;
            continue;
        }
#pragma unroll
        for (int q = 0; q < R::VEC; q += Elem<W>::VEC) unpack<W>(ld_chunk(w, c + q, N), out + i * R::VEC + q);
    }
}

// Mean and sum of squares about it over a row.  Each wave forms its own mean
// and squares about that (no barrier), and the waves' join, over c_i columns
// each, as
//   mean = sum S_i / N,  M2 = sum M2_i + c_i (S_i / c_i - mean)^2:
// one barrier per row and no cancellation (the mean comes from the sums: from
// the rounded wave means it was 16 times less exact where it is near zero).
// sh is the row parity's buffer.
template <int WAVES>
__device__ __forceinline__ void join_stats(float cnt, float sum, float& mean, float& m2, float (*sh)[4], float N) {
    if constexpr (WAVES == 1) return;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        sh[wave][0] = cnt;
        sh[wave][1] = mean;
        sh[wave][2] = m2;
        sh[wave][3] = sum;
    }
    __syncthreads();
    float tot = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) tot += sh[i][3];
    mean = tot / N;
    m2 = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const float d = sh[i][1] - mean;
        m2 += sh[i][2] + sh[i][0] * d * d;
    }
}

template <typename T, typename W, int WAVES, int EPT>
__global__ __launch_bounds__((RowMap<T, WAVES, EPT>::THREADS)) void layer_norm_kernel(
    uint32_t M, uint32_t N, const T* x, int64_t ldx, const W* w, const W* b, float eps, T* y, int64_t ldy,
    float* mean_out, float* rstd_out) {
    using R = RowMap<T, WAVES, EPT>;
    constexpr int VEC = R::VEC, NV = R::NV;
    __shared__ float sh[2][WAVES][4];
    const int t = WAVES == 1 ? (threadIdx.x & 63) : threadIdx.x;
    const uint32_t sub = WAVES == 1 ? threadIdx.x >> 6 : 0;
    const uint32_t step = gridDim.x * R::RPB;
    uint32_t m = blockIdx.x * R::RPB + sub;
    u32x4 raw[NV];
    auto load_row = [&](uint32_t r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = ld_chunk(x + (int64_t)r * ldx, (int64_t)(t + i * R::TPR) * VEC, N);
    };
    float wv[EPT], bv[EPT];
    if constexpr (!R::LEAN) {
        if (m < M) load_row(m);
        load_params<W, T, WAVES, EPT>(w, t, N, 1.0f, wv);
        load_params<W, T, WAVES, EPT>(b, t, N, 0.0f, bv);
    }
    float cnt = 0.0f;   // columns of this thread, then of its wave
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t left = (int64_t)N - (int64_t)(t + i * R::TPR) * VEC;
        cnt += (float)(left < 0 ? 0 : left < VEC ? left : VEC);
    }
    cnt = wave_sum(cnt);
    for (int par = 0; m < M; m += step, par ^= 1) {
        float v[EPT], sum = 0.0f, m2 = 0.0f;
        if constexpr (R::LEAN) load_row(m);
#pragma unroll
        for (int i = 0; i < NV; ++i) unpack<T>(raw[i], v + i * VEC);
        if constexpr (!R::LEAN)
            if (m + step < M && m + step > m) load_row(m + step);
#pragma unroll
        for (int i = 0; i < EPT; ++i) sum += v[i];
        sum = wave_sum(sum);
        float mean = cnt > 0.0f ? sum / cnt : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const bool in = (int64_t)(t + i * R::TPR) * VEC + e < N;
                const float d = v[i * VEC + e] - mean;
                m2 += in ? d * d : 0.0f;
            }
        m2 = wave_sum(m2);
        join_stats<WAVES>(cnt, sum, mean, m2, sh[par], (float)N);
        const float rstd = 1.0f / sqrtf(m2 / (float)N + eps);
        if (t == 0) {
            if (mean_out) mean_out[m] = mean;
            if (rstd_out) rstd_out[m] = rstd;
        }
        if constexpr (R::LEAN) {
            load_params<W, T, WAVES, EPT>(w, t, N, 1.0f, wv);
            load_params<W, T, WAVES, EPT>(b, t, N, 0.0f, bv);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float r[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                r[e] = (v[i * VEC + e] - mean) * rstd * wv[i * VEC + e] + bv[i * VEC + e];
            st_chunk(y + (int64_t)m * ldy, (int64_t)(t + i * R::TPR) * VEC, N, pack<T>(r));
        }
        if (m + step < m) break;   // past 2^32 rows
    }
}

template <typename T, typename W, int WAVES, int EPT>
__global__ __launch_bounds__((RowMap<T, WAVES, EPT>::THREADS)) void layer_norm_backward_kernel(
    uint32_t M, uint32_t N, const T* dy, int64_t lddy, const T* x, int64_t ldx, const W* w, const float* mean,
    const float* rstd, T* dx, int64_t lddx, float* part) {
    using R = RowMap<T, WAVES, EPT>;
    constexpr int VEC = R::VEC, NV = R::NV;
    __shared__ float sh[2][WAVES][2];
    const int t = WAVES == 1 ? (threadIdx.x & 63) : threadIdx.x;
    const uint32_t sub = WAVES == 1 ? threadIdx.x >> 6 : 0;
    const uint32_t step = gridDim.x * R::RPB;
    uint32_t m = blockIdx.x * R::RPB + sub;
    u32x4 rx[NV], rd[NV];
    float mu = 0.0f, rs = 0.0f;
    auto load_row = [&](uint32_t r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(t + i * R::TPR) * VEC;
            rx[i] = ld_chunk(x + (int64_t)r * ldx, c, N);
            rd[i] = ld_chunk(dy + (int64_t)r * lddy, c, N);
        }
        mu = mean[r];
        rs = rstd[r];
    };
    float wv[EPT], dw[EPT], db[EPT];
    if constexpr (!R::LEAN) {
        if (m < M) load_row(m);
        load_params<W, T, WAVES, EPT>(w, t, N, 1.0f, wv);
    }
#pragma unroll
    for (int i = 0; i < EPT; ++i) dw[i] = db[i] = 0.0f;
    for (int par = 0; m < M; m += step, par ^= 1) {
        float xh[EPT], d[EPT], s1 = 0.0f, s2 = 0.0f;
        if constexpr (R::LEAN) {
            load_row(m);
            load_params<W, T, WAVES, EPT>(w, t, N, 1.0f, wv);
        }
        const float r = rs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unpack<T>(rx[i], xh + i * VEC);
            unpack<T>(rd[i], d + i * VEC);
        }
#pragma unroll
        for (int i = 0; i < EPT; ++i) xh[i] = (xh[i] - mu) * r;
        if constexpr (!R::LEAN)
            if (m + step < M && m + step > m) load_row(m + step);
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const float g = d[i] * wv[i];
            s1 += g;
            s2 += g * xh[i];
            dw[i] += d[i] * xh[i];
            db[i] += d[i];
        }
        if (dx) {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            if constexpr (WAVES > 1) {
                if ((threadIdx.x & 63) == 0) {
                    sh[par][threadIdx.x >> 6][0] = s1;
                    sh[par][threadIdx.x >> 6][1] = s2;
                }
                __syncthreads();
                s1 = s2 = 0.0f;
#pragma unroll
                for (int i = 0; i < WAVES; ++i) {
                    s1 += sh[par][i][0];
                    s2 += sh[par][i][1];
                }
            }
            s1 /= (float)N;
            s2 /= (float)N;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int k = i * VEC + e;
                    o[e] = r * (d[k] * wv[k] - s1 - xh[k] * s2);
                }
                st_chunk(dx + (int64_t)m * lddx, (int64_t)(t + i * R::TPR) * VEC, N, pack<T>(o));
            }
        }
        if (m + step < m) break;   // past 2^32 rows
    }
    if (part) {
        float* pw = part + (int64_t)(blockIdx.x * R::RPB + sub) * 2 * N;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int q = 0; q < VEC; q += 4) {
                const int64_t c = (int64_t)(t + i * R::TPR) * VEC + q;
                st_chunk(pw, c, N, pack<float>(dw + i * VEC + q));
                st_chunk(pw + N, c, N, pack<float>(db + i * VEC + q));
            }
    }
}

// Rows too long for a workgroup's registers (N > 16384): read once more for
// each step.
constexpr int LONG = 1024;

__device__ __forceinline__ float long_sum(float v, float* sh) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = 0.0f;
    for (int i = 0; i < LONG / 64; ++i) r += sh[i];
    __syncthreads();
    return r;
}

template <typename T, typename W>
__global__ __launch_bounds__(LONG) void layer_norm_long_kernel(uint32_t M, uint32_t N, const T* x, int64_t ldx,
                                                               const W* w, const W* b, float eps, T* y, int64_t ldy,
                                                               float* mean_out, float* rstd_out) {
    __shared__ float sh[LONG / 64];
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const T* row = x + (int64_t)m * ldx;
        float s = 0.0f, m2 = 0.0f;
        for (uint32_t n = threadIdx.x; n < N; n += LONG) s += (float)row[n];
        const float mean = long_sum(s, sh) / (float)N;
        for (uint32_t n = threadIdx.x; n < N; n += LONG) {
            const float d = (float)row[n] - mean;
            m2 += d * d;
        }
        const float rstd = 1.0f / sqrtf(long_sum(m2, sh) / (float)N + eps);
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[m] = mean;
            if (rstd_out) rstd_out[m] = rstd;
        }
        for (uint32_t n = threadIdx.x; n < N; n += LONG)
            y[(int64_t)m * ldy + n] = (T)(((float)row[n] - mean) * rstd * (w ? (float)w[n] : 1.0f) +
                                          (b ? (float)b[n] : 0.0f));
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(LONG) void layer_norm_long_dx_kernel(uint32_t M, uint32_t N, const T* dy, int64_t lddy,
                                                                  const T* x, int64_t ldx, const W* w,
                                                                  const float* mean, const float* rstd, T* dx,
                                                                  int64_t lddx) {
    __shared__ float sh[LONG / 64];
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const T *row = x + (int64_t)m * ldx, *d = dy + (int64_t)m * lddy;
        const float mu = mean[m], r = rstd[m];
        float s1 = 0.0f, s2 = 0.0f;
        for (uint32_t n = threadIdx.x; n < N; n += LONG) {
            const float g = (float)d[n] * (w ? (float)w[n] : 1.0f);
            s1 += g;
            s2 += g * (((float)row[n] - mu) * r);
        }
        s1 = long_sum(s1, sh) / (float)N;
        s2 = long_sum(s2, sh) / (float)N;
        for (uint32_t n = threadIdx.x; n < N; n += LONG) {
            const float g = (float)d[n] * (w ? (float)w[n] : 1.0f);
            dx[(int64_t)m * lddx + n] = (T)(r * (g - s1 - ((float)row[n] - mu) * r * s2));
        }
    }
}

// a thread per column, the rows over gridDim.y slices
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_long_dw_kernel(uint32_t M, uint32_t N, const T* dy, int64_t lddy,
                                                                 const T* x, int64_t ldx, const float* mean,
                                                                 const float* rstd, float* part) {
    const uint32_t n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float dw = 0.0f, db = 0.0f;
    for (uint64_t m = blockIdx.y; m < M; m += gridDim.y) {
        const float d = (float)dy[(int64_t)m * lddy + n];
        dw += d * (((float)x[(int64_t)m * ldx + n] - mean[m]) * rstd[m]);
        db += d;
    }
    part[(int64_t)blockIdx.y * 2 * N + n] = dw;
    part[(int64_t)blockIdx.y * 2 * N + N + n] = db;
}

// dw and db from the partial rows, in their order: 16 waves take 1/16 of the
// rows each for 64 columns, then the first adds the waves' sums in order
template <typename G>
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* part, uint32_t parts, uint32_t N, G* dw,
                                                                 G* db, float beta) {
    __shared__ float sh[16][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    G* out = blockIdx.y ? db : dw;
    if (!out) return;
    const uint32_t n = blockIdx.x * 64 + lane;
    const float* src = part + (blockIdx.y ? N : 0) + n;
    const uint32_t p0 = (uint32_t)((uint64_t)parts * wave / 16), p1 = (uint32_t)((uint64_t)parts * (wave + 1) / 16);
    float s = 0.0f;
    if (n < N) {
        uint32_t p = p0;
        for (; p + 8 <= p1; p += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = src[(int64_t)(p + i) * 2 * N];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; p < p1; ++p) s += src[(int64_t)p * 2 * N];
    }
    sh[wave][lane] = s;
    __syncthreads();
    if (wave || n >= N) return;
    for (int i = 1; i < 16; ++i) s += sh[i][lane];
    out[n] = (G)(beta == 0.0f ? s : s + beta * (float)out[n]);
}

// Rows are held by one wave up to 1024 columns, by four up to 4096, by
// sixteen up to LAST: 8 or 16 values a thread.
constexpr uint32_t LAST = 16384;
template <typename F>
static bool with_map(uint32_t N, F f) {
    using std::integral_constant;
    if (N <= 512) f(integral_constant<int, 1>{}, integral_constant<int, 8>{});
    else if (N <= 1024) f(integral_constant<int, 1>{}, integral_constant<int, 16>{});
    else if (N <= 2048) f(integral_constant<int, 4>{}, integral_constant<int, 8>{});
    else if (N <= 4096) f(integral_constant<int, 4>{}, integral_constant<int, 16>{});
    else if (N <= 8192) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (N <= LAST) f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
    else return false;
    return true;
}

// Workgroups for M rows of N: 16 waves per CU of 256
static uint32_t norm_blocks(uint32_t M, uint32_t waves) {
    const uint32_t rpb = waves == 1 ? 4 : 1;
    const uint64_t need = ((uint64_t)M + rpb - 1) / rpb;
    const uint64_t most = 256ull * (waves == 1 ? 4 : 16 / waves);
    return (uint32_t)(need < most ? need : most);
}

static uint32_t long_slices(uint32_t M) { return M < 64u ? M : 64u; }

// f(T{}, W{}) for the pair of element types; false: none such
template <typename F>
static bool with_types(int type, int w_type, F f) {
    return (w_type == type || w_type == VKB_T_F32) && with_type(type, [&](auto t) {
        if (w_type == VKB_T_F32) f(t, float{});
        else f(t, t);
    });
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" int vkb_launch_layer_norm(int type, int w_type, uint32_t M, uint32_t N, const void* x, int64_t ldx,
                                     const void* w, const void* b, float eps, void* y, int64_t ldy, float* mean,
                                     float* rstd, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const bool ok = with_types(type, w_type, [&](auto tt, auto tw) {
        using T = decltype(tt);
        using W = decltype(tw);
        const bool fits = with_map(N, [&](auto waves, auto ept) {
            using R = RowMap<T, waves.value, ept.value>;
            hipLaunchKernelGGL((layer_norm_kernel<T, W, waves.value, ept.value>),
                               dim3(norm_blocks(M, waves.value)), dim3(R::THREADS), 0, st, M, N, (const T*)x, ldx,
                               (const W*)w, (const W*)b, eps, (T*)y, ldy, mean, rstd);
        });
        if (!fits)
            hipLaunchKernelGGL((layer_norm_long_kernel<T, W>), dim3(M < 4096u ? M : 4096u), dim3(LONG), 0, st, M, N,
                               (const T*)x, ldx, (const W*)w, (const W*)b, eps, (T*)y, ldy, mean, rstd);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_layer_norm_long(uint32_t N) { return N > LAST; }

extern "C" uint32_t vkb_layer_norm_parts(int type, uint32_t M, uint32_t N) {
    (void)type;
    uint32_t parts = long_slices(M);
    with_map(N, [&](auto waves, auto ept) {
        parts = norm_blocks(M, waves.value) * (waves.value == 1 ? 4 : 1);
    });
    return parts;
}

extern "C" int vkb_launch_layer_norm_backward(int type, int w_type, uint32_t M, uint32_t N, const void* dy,
                                              int64_t lddy, const void* x, int64_t ldx, const void* w,
                                              const float* mean, const float* rstd, void* dx, int64_t lddx,
                                              float* part, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const bool ok = with_types(type, w_type, [&](auto tt, auto tw) {
        using T = decltype(tt);
        using W = decltype(tw);
        const bool fits = with_map(N, [&](auto waves, auto ept) {
            using R = RowMap<T, waves.value, ept.value>;
            hipLaunchKernelGGL((layer_norm_backward_kernel<T, W, waves.value, ept.value>),
                               dim3(norm_blocks(M, waves.value)), dim3(R::THREADS), 0, st, M, N, (const T*)dy, lddy,
                               (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, lddx, part);
        });
        if (fits) return;
        // the sums first: dx may be dy or x
        if (part)
            hipLaunchKernelGGL((layer_norm_long_dw_kernel<T>), dim3((N + 255) / 256, long_slices(M)), dim3(256), 0, st,
                               M, N, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, part);
        if (dx)
            hipLaunchKernelGGL((layer_norm_long_dx_kernel<T, W>), dim3(M < 4096u ? M : 4096u), dim3(LONG), 0, st, M, N,
                               (const T*)dy, lddy, (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, lddx);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_layer_norm_reduce(const float* part, uint32_t parts, uint32_t N, void* dw, void* db,
                                            int g_type, float beta, void* stream) {
    const bool ok = with_type(g_type, [&](auto t) {
        using G = decltype(t);
        hipLaunchKernelGGL((layer_norm_reduce_kernel<G>), dim3((N + 63) / 64, 2), dim3(1024), 0, (hipStream_t)stream,
                           part, parts, N, (G*)dw, (G*)db, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
