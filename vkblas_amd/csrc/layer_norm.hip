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
// statistic counts.  us (TB/s read and written; a 1 GiB copy reaches 5.2): 8192 x
// 4096 bf16 with fp32 parameters forward 24.5 (5.4), backward 33.1 (6.1) and the
// sums' join 4.8; 1003 x 997 fp32 gradients in one launch 7.7 (27.5 MiB read for the operands'
// 7.6: the rows' workgroups read them once, the columns' again, 64 bytes of a line
// each, in two L2s); one row 3.4.
#include <type_traits>
#include "nn_common.hpp"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

// How a row's columns lie in a workgroup: its threads hold the 16-byte chunks
// t + i * (threads per row), i < EPT / VEC.
//  ONE:  a wave per row, four rows per workgroup, no barrier;
//  FEW:  a workgroup of up to eight waves per row, w and b in registers;
//  MANY: up to sixteen, which leaves 128 registers a thread: w and b in LDS
//        (read from L2 for every row they were the bound: 14080 columns of
//        bf16 with fp32 parameters 196 us against 143).
// As many waves as the columns need, past four in whole rounds of the CU's
// four SIMDs: a row is about half bound by its instructions, and a fifth wave
// doubles one SIMD's (8192 x 4352 bf16 58 us with five waves).
enum { ONE, FEW, MANY };
constexpr uint32_t LAST = 16384;
template <typename T, int MAP, int EPT>
struct RowMap {
    static constexpr int VEC = Elem<T>::VEC, NV = EPT / VEC;
    static constexpr int RPB = MAP == ONE ? 4 : 1;           // rows at a time
    static constexpr int MAXW = MAP == ONE ? 1 : MAP == FEW ? 8 : 16;
    static constexpr int THREADS = MAXW * RPB * 64;          // at most
    static_assert(EPT % VEC == 0, "whole chunks");
    // waves per row of N columns
    static uint32_t waves(uint32_t N) {
        const uint32_t w = (N + 64 * EPT - 1) / (64 * EPT);
        return MAP == ONE ? 1 : w <= 4 ? w : (w + 3) / 4 * 4;
    }
};

// A thread's chunks of a row of N >= VEC columns, the same for every row, so
// that a row is loaded without a branch (one between lanes made every load wait
// for the one before it, one around a wave's load for the last row's stores:
// rows of 4832 against 4096 81 us against 37).  Chunk i is read from column
// off(i): the one at the row's end from N - VEC on, and threads past the end
// read that too; its elements before from(i) are another thread's.  whole: every
// chunk of this wave is a lane's own throughout (the same in all its lanes).
template <typename T, int NV>
struct Chunks {
    static constexpr int VEC = Elem<T>::VEC;
    int t, tpr;
    uint32_t N;
    bool whole;
    __device__ __forceinline__ Chunks(int t_, int tpr_, uint32_t N_) : t(t_), tpr(tpr_), N(N_) {
        bool all = true;
#pragma unroll
        for (int i = 0; i < NV; ++i) all = all && from(i) == 0;
        whole = __all(all);
    }
    __device__ __forceinline__ uint32_t off(int i) const { return min((uint32_t)(t + i * tpr) * VEC, N - VEC); }
    __device__ __forceinline__ int from(int i) const {
        return (int)min((uint32_t)(t + i * tpr) * VEC - off(i), (uint32_t)VEC);
    }
    // a value of t that the compiler takes for a new one: nothing derived from
    // it is kept in registers over the rows before this
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(t)); }
    __device__ __forceinline__ float count() const {
        int c = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) c += VEC - from(i);
        return (float)c;
    }
    // x[e] becomes 0 unless it is this thread's
    __device__ __forceinline__ void own(int i, float* x) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = e >= from(i) ? x[e] : 0.0f;
    }
    __device__ __forceinline__ void store(int i, T* row, u32x4 v) const {
        if (whole || from(i) == 0) {
            *(u32x4_any*)(row + off(i)) = v;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (e < from(i)) continue;
                if constexpr (sizeof(T) == 4) *(uint32_t*)(row + off(i) + e) = v[e];
                else *(uint16_t*)(row + off(i) + e) = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
            }
        }
    }
};

template <typename W, int VEC>
__device__ __forceinline__ void load_params(const W* w, uint32_t c, float none, float* out) {
    if (!w) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = none;
        return;
    }
#pragma unroll
    for (int q = 0; q < VEC; q += Elem<W>::VEC) unpack<W>(ld16_any(w + c + q), out + q);
}

// w or b of a thread's columns: registers, or this thread's own words of LDS
template <typename T, int MAP, int EPT>
struct Params {
    using R = RowMap<T, MAP, EPT>;
    float reg[MAP == MANY ? 1 : EPT];
    float4* lds;             // MANY: chunk i, quarter q of thread t at (i VEC / 4 + q) * threads + t
    int t, tpr;
    template <typename W>
    __device__ __forceinline__ void load(const W* w, float none, uint32_t N, float4* mem, int t_, int tpr_) {
        lds = mem;
        t = t_;
        tpr = tpr_;
#pragma unroll
        for (int i = 0; i < R::NV; ++i) {
            float x[R::VEC];
            load_params<W, R::VEC>(w, min((uint32_t)(t + i * tpr) * R::VEC, N - R::VEC), none, x);   // as Chunks
#pragma unroll
            for (int e = 0; e < R::VEC; ++e) {
                if constexpr (MAP != MANY) reg[i * R::VEC + e] = x[e];
            }
            if constexpr (MAP == MANY)
#pragma unroll
                for (int q = 0; q < R::VEC / 4; ++q)
                    lds[(i * (R::VEC / 4) + q) * tpr + t] = float4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
        }
    }
    // the VEC values of chunk i
    __device__ __forceinline__ void get(int i, float* x) const {
        if constexpr (MAP == MANY) {
#pragma unroll
            for (int q = 0; q < R::VEC / 4; ++q) {
                const float4 v = lds[(i * (R::VEC / 4) + q) * tpr + t];
                x[4 * q] = v.x, x[4 * q + 1] = v.y, x[4 * q + 2] = v.z, x[4 * q + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < R::VEC; ++e) x[e] = reg[i * R::VEC + e];
        }
    }
};

// Mean and sum of squares about it over a row.  Each wave forms its own mean
// and squares about that (no barrier), and the waves' join, over c_i columns
// each, as
//   mean = sum S_i / N,  M2 = sum M2_i + c_i (S_i / c_i - mean)^2:
// one barrier per row and no cancellation (the mean comes from the sums: from
// the rounded wave means it was 16 times less exact where it is near zero).
// sh is the row parity's buffer.
__device__ __forceinline__ void join_stats(float cnt, float sum, float& mean, float& m2, float4* sh, int waves,
                                           float N) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = float4{cnt, mean, m2, sum};
    __syncthreads();
    float tot = 0.0f;
    for (int i = 0; i < waves; ++i) tot += sh[i].w;
    mean = tot / N;
    m2 = 0.0f;
    for (int i = 0; i < waves; ++i) {
        const float4 v = sh[i];
        const float d = v.y - mean;
        m2 += v.z + v.x * d * d;
    }
}

template <typename T, typename W, int MAP, int EPT>
__global__ __launch_bounds__((RowMap<T, MAP, EPT>::THREADS)) void layer_norm_kernel(
    uint32_t M, uint32_t N, const T* x, int64_t ldx, const W* w, const W* b, float eps, T* y, int64_t ldy,
    float* mean_out, float* rstd_out) {
    using R = RowMap<T, MAP, EPT>;
    constexpr int VEC = R::VEC, NV = R::NV;
    __shared__ float4 sh[2][R::MAXW];
    __shared__ float4 prm[MAP == MANY ? 2 : 1][MAP == MANY ? LAST / 4 : 1];
    const int t = MAP == ONE ? (threadIdx.x & 63) : threadIdx.x, tpr = MAP == ONE ? 64 : blockDim.x;
    const uint32_t sub = MAP == ONE ? threadIdx.x >> 6 : 0;
    const uint32_t step = gridDim.x * R::RPB;
    uint32_t m = blockIdx.x * R::RPB + sub;
    const Chunks<T, NV> ch(t, tpr, N);
    const float cnt = wave_sum(ch.count());   // columns of this wave
    u32x4 raw[NV];
    auto load_row = [&](uint32_t r) {
        const T* row = x + (int64_t)r * ldx;
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = ld16_any(row + ch.off(i));
    };
    if (m < M) load_row(m);
    Params<T, MAP, EPT> wv, bv;
    wv.load(w, 1.0f, N, prm[0], t, tpr);
    bv.load(b, 0.0f, N, prm[MAP == MANY], t, tpr);
    float v[EPT];
    auto unpack_row = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i) unpack<T>(raw[i], v + i * VEC);
    };
    if (m < M) unpack_row();
    for (int par = 0; m < M; m += step, par ^= 1) {
        const bool next = m + step < M && m + step > m;   // (past 2^32 rows: none)
        if (next) load_row(m + step);
        float sum = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float own[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) own[e] = v[i * VEC + e];
            if (!ch.whole) ch.own(i, own);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += own[e];
        }
        sum = wave_sum(sum);
        float mean = cnt > 0.0f ? sum / cnt : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float d[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = v[i * VEC + e] - mean;
            if (!ch.whole) ch.own(i, d);
#pragma unroll
            for (int e = 0; e < VEC; ++e) m2 += d[e] * d[e];
        }
        m2 = wave_sum(m2);
        if constexpr (MAP != ONE) join_stats(cnt, sum, mean, m2, sh[par], tpr >> 6, (float)N);
        const float rstd = 1.0f / sqrtf(m2 / (float)N + eps);
        u32x4 out[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float r[VEC], wi[VEC], bi[VEC];
            wv.get(i, wi);
            bv.get(i, bi);
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[e] = (v[i * VEC + e] - mean) * rstd * wi[e] + bi[e];
            out[i] = pack<T>(r);
        }
        // the next row is waited for before this one's stores leave: after
        // them, its loads would be waited for together with the stores
        if (next) unpack_row();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NV; ++i) ch.store(i, y + (int64_t)m * ldy, out[i]);
        if (t == 0) {
            if (mean_out) mean_out[m] = mean;
            if (rstd_out) rstd_out[m] = rstd;
        }
        if (!next) break;
    }
}

template <typename T, typename W, int MAP, int EPT>
__global__ __launch_bounds__((RowMap<T, MAP, EPT>::THREADS)) void layer_norm_backward_kernel(
    uint32_t M, uint32_t N, const T* dy, int64_t lddy, const T* x, int64_t ldx, const W* w, const float* mean,
    const float* rstd, T* dx, int64_t lddx, float* part) {
    using R = RowMap<T, MAP, EPT>;
    constexpr int VEC = R::VEC, NV = R::NV;
    __shared__ float2 sh[2][R::MAXW];
    __shared__ float4 prm[MAP == MANY ? LAST / 4 : 1];
    const int t = MAP == ONE ? (threadIdx.x & 63) : threadIdx.x, tpr = MAP == ONE ? 64 : blockDim.x;
    const uint32_t sub = MAP == ONE ? threadIdx.x >> 6 : 0;
    const uint32_t step = gridDim.x * R::RPB;
    uint32_t m = blockIdx.x * R::RPB + sub;
    Chunks<T, NV> ch(t, tpr, N);
    u32x4 rx[NV], rd[NV];
    float mu = 0.0f, rs = 0.0f;
    auto load_row = [&](uint32_t r) {
        const T *xr = x + (int64_t)r * ldx, *dr = dy + (int64_t)r * lddy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            rx[i] = ld16_any(xr + ch.off(i));
            rd[i] = ld16_any(dr + ch.off(i));
        }
        mu = mean[r];
        rs = rstd[r];
    };
    // MANY: no registers for a row loaded ahead
    constexpr bool AHEAD = MAP != MANY;
    if (AHEAD && m < M) load_row(m);
    Params<T, MAP, EPT> wv;
    wv.load(w, 1.0f, N, prm, t, tpr);
    float dw[EPT], db[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) dw[i] = db[i] = 0.0f;
    for (int par = 0; m < M; m += step, par ^= 1) {
        const bool next = m + step < M && m + step > m;   // (past 2^32 rows: none)
        float xh[EPT], g[EPT], s1 = 0.0f, s2 = 0.0f;
        if (!AHEAD) {
            ch.fresh();
            load_row(m);
        }
        const float r = rs, mr = mu;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unpack<T>(rx[i], xh + i * VEC);
            unpack<T>(rd[i], g + i * VEC);
            if (!ch.whole) ch.own(i, g + i * VEC);   // 0: adds to no sum
        }
        if (AHEAD && next) load_row(m + step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float wi[VEC];
            wv.get(i, wi);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int k = i * VEC + e;
                xh[k] = (xh[k] - mr) * r;
                dw[k] += g[k] * xh[k];
                db[k] += g[k];
                g[k] *= wi[e];
                s1 += g[k];
                s2 += g[k] * xh[k];
            }
            if (MAP == MANY) __builtin_amdgcn_sched_barrier(0);   // one chunk's temporaries at a time
        }
        if (dx) {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            if constexpr (MAP != ONE) {
                if ((threadIdx.x & 63) == 0) sh[par][threadIdx.x >> 6] = float2{s1, s2};
                __syncthreads();
                s1 = s2 = 0.0f;
                for (int i = 0; i < tpr >> 6; ++i) {
                    s1 += sh[par][i].x;
                    s2 += sh[par][i].y;
                }
            }
            s1 /= (float)N;
            s2 /= (float)N;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = r * (g[i * VEC + e] - s1 - xh[i * VEC + e] * s2);
                ch.store(i, dx + (int64_t)m * lddx, pack<T>(o));
                if (MAP == MANY) __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!next) break;
    }
    if constexpr (MAP == ONE) {
        // the four waves' sums, in their order
        __shared__ float sums[2][EPT][64];
        for (uint32_t k = 1; k < R::RPB; ++k) {
            __syncthreads();
            if (sub == k)
#pragma unroll
                for (int i = 0; i < EPT; ++i) {
                    sums[0][i][t] = dw[i];
                    sums[1][i][t] = db[i];
                }
            __syncthreads();
            if (sub == 0)
#pragma unroll
                for (int i = 0; i < EPT; ++i) {
                    dw[i] += sums[0][i][t];
                    db[i] += sums[1][i][t];
                }
        }
        if (sub) return;
    }
    if (part) {
        float* pw = part + (int64_t)blockIdx.x * 2 * N;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float* pi = pw + ch.off(i);
#pragma unroll
            for (int q = 0; q < VEC; q += 4) {
                if (ch.from(i) <= q) {
                    *(u32x4_any*)(pi + q) = pack<float>(dw + i * VEC + q);
                    *(u32x4_any*)(pi + N + q) = pack<float>(db + i * VEC + q);
                } else {
#pragma unroll
                    for (int e = q; e < q + 4; ++e)
                        if (e >= ch.from(i)) {
                            pi[e] = dw[i * VEC + e];
                            pi[N + e] = db[i * VEC + e];
                        }
                }
                if (MAP == MANY) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
}

// Rows too long for a workgroup's registers (N > 16384), or shorter than a
// chunk: read once more for each step.
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

// A column's sum over the 1024 / COLS slices of a workgroup of COLS columns (a
// wave holds 64 / COLS slices), in a fixed tree, in the first COLS threads
template <int COLS>
__device__ __forceinline__ float join_slices(float s, float (*sh)[COLS]) {
#pragma unroll
    for (int d = COLS; d < 64; d *= 2) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) < COLS) sh[threadIdx.x >> 6][threadIdx.x & (COLS - 1)] = s;
    __syncthreads();
    s = sh[0][threadIdx.x & (COLS - 1)];
    for (int i = 1; i < 16; ++i) s += sh[i][threadIdx.x & (COLS - 1)];
    __syncthreads();
    return s;
}

template <typename G>
__device__ __forceinline__ void put_grad(G* out, float s, float beta) {
    *out = (G)(beta == 0.0f ? s : s + beta * (float)*out);
}

// dw and db from the partial rows: of a workgroup's threads per column each
// adds its share of them in order, 16 loads in flight.  32 columns read whole
// lines (4096 columns 6.7 us on 16, 4.7 on 32); up to 2048 columns 16 give twice
// the workgroups (997 columns 1.6 us less).
template <typename G, int COLS>
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* part, uint32_t parts, uint32_t N, G* dw,
                                                                 G* db, float beta) {
    constexpr uint32_t SLICES = 1024 / COLS;
    __shared__ float sh[16][COLS];
    const uint32_t slice = threadIdx.x / COLS;
    G* out = blockIdx.y ? db : dw;
    if (!out) return;
    const uint32_t n = blockIdx.x * COLS + threadIdx.x % COLS;
    const float* src = part + (blockIdx.y ? N : 0) + n;
    const uint32_t p0 = (uint32_t)((uint64_t)parts * slice / SLICES);
    const uint32_t p1 = (uint32_t)((uint64_t)parts * (slice + 1) / SLICES);
    float s = 0.0f;
    if (n < N)
        for (uint32_t p = p0; p < p1; p += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = p + i < p1 ? src[(int64_t)(p + i) * 2 * N] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += v[i];
        }
    s = join_slices<COLS>(s, sh);
    if (threadIdx.x < COLS && n < N) put_grad(out + n, s, beta);
}

// The gradients of few rows in one launch, without partial sums: the first
// workgroups take dx's rows (a wave or a workgroup each, as the maps above),
// the others 32 columns of dw and db each, from the rows themselves; or 16 where
// the walk down the rows is the longest chain of loads and twice the workgroups
// still find idle CUs.  dx must not be dy or x where both are wanted (the others
// still read them): then two launches, the columns' first.
constexpr int FEW_THREADS = 1024;

template <typename T, typename W, int MAP, int EPT>
__device__ __forceinline__ void few_dx(uint32_t M, uint32_t N, uint32_t waves, const T* dy, int64_t lddy, const T* x,
                                       int64_t ldx, const W* w, const float* mean, const float* rstd, T* dx,
                                       int64_t lddx) {
    using R = RowMap<T, MAP, EPT>;
    constexpr int VEC = R::VEC, NV = R::NV;
    __shared__ float2 sh[FEW_THREADS / 64];
    const int wave = threadIdx.x >> 6;
    const int tpr = MAP == ONE ? 64 : (int)waves * 64;
    // waves past the row's start past its last chunk (t of tpr on would be another
    // thread's next one): none is theirs, they add and store nothing
    const int t = MAP == ONE ? (int)(threadIdx.x & 63) : (int)threadIdx.x + ((int)threadIdx.x < tpr ? 0 : NV * tpr);
    const uint32_t m = MAP == ONE ? blockIdx.x * (FEW_THREADS / 64) + wave : blockIdx.x;
    if (MAP == ONE && m >= M) return;   // (no barrier there)
    const Chunks<T, NV> ch(t, tpr, N);
    const T *xr = x + (int64_t)m * ldx, *dr = dy + (int64_t)m * lddy;
    const float mu = mean[m], r = rstd[m];
    u32x4 rx[NV], rd[NV];
    float g[EPT], xh[EPT], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        rx[i] = ld16_any(xr + ch.off(i));
        rd[i] = ld16_any(dr + ch.off(i));
        load_params<W, VEC>(w, ch.off(i), 1.0f, g + i * VEC);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float d[VEC];
        unpack<T>(rx[i], xh + i * VEC);
        unpack<T>(rd[i], d);
        if (!ch.whole) ch.own(i, d);   // 0: adds to no sum
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int k = i * VEC + e;
            xh[k] = (xh[k] - mu) * r;
            g[k] *= d[e];
            s1 += g[k];
            s2 += g[k] * xh[k];
        }
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if constexpr (MAP != ONE) {
        if ((threadIdx.x & 63) == 0) sh[wave] = float2{s1, s2};
        __syncthreads();
        s1 = s2 = 0.0f;
        for (uint32_t i = 0; i < waves; ++i) {
            s1 += sh[i].x;
            s2 += sh[i].y;
        }
    }
    s1 /= (float)N;
    s2 /= (float)N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = r * (g[i * VEC + e] - s1 - xh[i * VEC + e] * s2);
        ch.store(i, dx + (int64_t)m * lddx, pack<T>(o));
    }
}

template <int COLS, typename T, typename G>
__device__ __forceinline__ void few_dw(uint32_t block, uint32_t M, uint32_t N, const T* dy, int64_t lddy, const T* x,
                                       int64_t ldx, const float* mean, const float* rstd, G* dw, G* db, float beta) {
    constexpr uint32_t SLICES = FEW_THREADS / COLS;
    __shared__ float sh[16][COLS];
    constexpr int U = 8;         // rows in flight
    const uint32_t slice = threadIdx.x / COLS;
    const uint32_t n = block * COLS + threadIdx.x % COLS;
    float sw = 0.0f, sb = 0.0f;
    if (n < N)
        for (uint32_t m = slice; m < M; m += SLICES * U) {
            float d[U], h[U];
#pragma unroll
            for (uint32_t i = 0; i < U; ++i) {
                const uint32_t r = min(m + SLICES * i, M - 1);
                d[i] = (float)dy[(int64_t)r * lddy + n];
                h[i] = ((float)x[(int64_t)r * ldx + n] - mean[r]) * rstd[r];
            }
#pragma unroll
            for (uint32_t i = 0; i < U; ++i)
                if (m + SLICES * i < M) {
                    sw += d[i] * h[i];
                    sb += d[i];
                }
        }
    sw = join_slices<COLS>(sw, sh);
    sb = join_slices<COLS>(sb, sh);
    if (threadIdx.x >= COLS || n >= N) return;
    if (dw) put_grad(dw + n, sw, beta);
    if (db) put_grad(db + n, sb, beta);
}

template <typename T, typename W, int MAP, int EPT>
__global__ __launch_bounds__(FEW_THREADS) void layer_norm_few_kernel(
    uint32_t M, uint32_t N, uint32_t waves, uint32_t dx_blocks, const T* dy, int64_t lddy, const T* x, int64_t ldx,
    const W* w, const float* mean, const float* rstd, T* dx, int64_t lddx, void* dw, void* db, bool g_f32, float beta,
    bool narrow) {
    const uint32_t block = blockIdx.x - dx_blocks;
    if (blockIdx.x < dx_blocks) {
        few_dx<T, W, MAP, EPT>(M, N, waves, dy, lddy, x, ldx, w, mean, rstd, dx, lddx);
    } else if (g_f32) {
        if (narrow) few_dw<16, T, float>(block, M, N, dy, lddy, x, ldx, mean, rstd, (float*)dw, (float*)db, beta);
        else few_dw<32, T, float>(block, M, N, dy, lddy, x, ldx, mean, rstd, (float*)dw, (float*)db, beta);
    } else {
        if (narrow) few_dw<16, T, T>(block, M, N, dy, lddy, x, ldx, mean, rstd, (T*)dw, (T*)db, beta);
        else few_dw<32, T, T>(block, M, N, dy, lddy, x, ldx, mean, rstd, (T*)dw, (T*)db, beta);
    }
}

// f(map, values a thread) for rows of N columns; false: rows shorter than a
// chunk or past a workgroup's registers
template <typename F>
static bool with_map(uint32_t N, F f) {
    using std::integral_constant;
    if (N < 8) return false;
    if (N <= 512) f(integral_constant<int, ONE>{}, integral_constant<int, 8>{});
    else if (N <= 1024) f(integral_constant<int, ONE>{}, integral_constant<int, 16>{});
    else if (N <= 2048) f(integral_constant<int, FEW>{}, integral_constant<int, 8>{});
    else if (N <= 8192) f(integral_constant<int, FEW>{}, integral_constant<int, 16>{});
    else if (N <= LAST) f(integral_constant<int, MANY>{}, integral_constant<int, 16>{});
    else return false;
    return true;
}

// Workgroups for M rows: 16 waves per CU of 256, or 8 in the backward pass,
// whose workgroups leave 8 N bytes of partial sums each.  us, bf16 with fp32
// parameters, 4 / 8 / 12 / 16 / 24 waves: 8192 x 4096 forward 50 / 31 / 28 / 27 / 28,
// backward 49 / 46 / 52 / 56 / 63.
static uint32_t norm_blocks(uint32_t M, int map, uint32_t waves, bool backward) {
    const uint32_t rpb = map == ONE ? 4 : 1;
    const uint64_t need = ((uint64_t)M + rpb - 1) / rpb;
    const uint32_t per = (backward ? 8 : 16) / (waves * rpb);
    const uint64_t most = 256ull * (per ? per : 1);
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
        const bool fits = with_map(N, [&](auto map, auto ept) {
            using R = RowMap<T, map.value, ept.value>;
            const uint32_t waves = R::waves(N);
            hipLaunchKernelGGL((layer_norm_kernel<T, W, map.value, ept.value>),
                               dim3(norm_blocks(M, map.value, waves, false)), dim3(64 * waves * R::RPB), 0, st, M, N,
                               (const T*)x, ldx, (const W*)w, (const W*)b, eps, (T*)y, ldy, mean, rstd);
        });
        if (!fits)
            hipLaunchKernelGGL((layer_norm_long_kernel<T, W>), dim3(M < 4096u ? M : 4096u), dim3(LONG), 0, st, M, N,
                               (const T*)x, ldx, (const W*)w, (const W*)b, eps, (T*)y, ldy, mean, rstd);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_layer_norm_long(uint32_t N) { return !with_map(N, [](auto, auto) {}); }

extern "C" uint32_t vkb_layer_norm_parts(int type, uint32_t M, uint32_t N) {
    (void)type;
    uint32_t parts = long_slices(M);
    with_map(N, [&](auto map, auto ept) {
        parts = norm_blocks(M, map.value, RowMap<float, map.value, ept.value>::waves(N), true);
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
        const bool fits = with_map(N, [&](auto map, auto ept) {
            using R = RowMap<T, map.value, ept.value>;
            const uint32_t waves = R::waves(N);
            hipLaunchKernelGGL((layer_norm_backward_kernel<T, W, map.value, ept.value>),
                               dim3(norm_blocks(M, map.value, waves, true)), dim3(64 * waves * R::RPB), 0, st, M, N,
                               (const T*)dy, lddy,
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
        if (N <= 2048)
            hipLaunchKernelGGL((layer_norm_reduce_kernel<G, 16>), dim3((N + 15) / 16, 2), dim3(1024), 0,
                               (hipStream_t)stream, part, parts, N, (G*)dw, (G*)db, beta);
        else
            hipLaunchKernelGGL((layer_norm_reduce_kernel<G, 32>), dim3((N + 31) / 32, 2), dim3(1024), 0,
                               (hipStream_t)stream, part, parts, N, (G*)dw, (G*)db, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_layer_norm_few(int type, int w_type, uint32_t M, uint32_t N, const void* dy, int64_t lddy,
                                         const void* x, int64_t ldx, const void* w, const float* mean,
                                         const float* rstd, void* dx, int64_t lddx, void* dw, void* db, int g_type,
                                         float beta, void* stream) {
    if ((dw || db) && g_type != type && g_type != VKB_T_F32) return (int)hipErrorInvalidValue;
    bool fits = false;
    // us, 32 / 16 columns a workgroup: fp32 500 x 512 4.9 / 3.8, 1000 x 997 8.7 / 7.1, 500 x
    // 2048 7.6 / 6.2, bf16 1000 x 1024 7.7 / 5.3; 256 x 1024 level, 139 x 2048 3.7 / 4.5, 1000
    // x 2048 11.1 / 13.5, 500 x 4096 8.7 / 10.2
    const bool narrow = M > 256 && N <= 2048 && (uint64_t)M * N <= 1u << 20;
    const bool ok = with_types(type, w_type, [&](auto tt, auto tw) {
        using T = decltype(tt);
        using W = decltype(tw);
        fits = with_map(N, [&](auto map, auto ept) {
            const uint32_t waves = RowMap<T, map.value, ept.value>::waves(N);
            const uint32_t rows = map.value == ONE ? FEW_THREADS / 64 : 1;
            const uint32_t rb = dx ? (M + rows - 1) / rows : 0, cols = narrow ? 16 : 32, cb = dw || db ? (N + cols - 1) / cols : 0;
            hipLaunchKernelGGL((layer_norm_few_kernel<T, W, map.value, ept.value>), dim3(rb + cb), dim3(FEW_THREADS), 0,
                               (hipStream_t)stream, M, N, waves, rb, (const T*)dy, lddy, (const T*)x, ldx, (const W*)w,
                               mean, rstd, (T*)dx, lddx, dw, db, g_type == VKB_T_F32, beta, narrow);
        });
    });
    return ok && fits ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
