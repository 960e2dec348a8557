// gemm_ops.hpp — operators that finish a tile of A B^T inside the pipelined
// GEMM kernel (gemm_pipe.hpp), so the product itself never reaches memory:
// the gated projection, and the logits' statistics and gradient of a linear
// cross entropy.
//
// Accumulators: with SH 0 (16-bit operands) a lane holds, of fragment (i, j)
// of its wave's WT x WT block, columns 16 j + 4 (lane / 16) + e of row
// 16 i + lane % 16; with SH 2 (fp32) register 4 q + e is column 32 j + 8 q +
// 4 (lane / 32) + e of row 32 i + lane % 32.
#pragma once
#include "gemm_pipe.hpp"
#include "nn_common.hpp"

namespace vkb {

template <int WT, int SH>
struct Frag {
    static constexpr int FR = SH == 0 ? 16 : 32, NF = WT / FR, NQ = SH == 0 ? 1 : 4;
    static __device__ __forceinline__ int row(int lane, int i) { return i * FR + (lane & (FR - 1)); }
    static __device__ __forceinline__ int col(int lane, int j, int q) {
        return j * FR + (SH == 0 ? 4 * (lane >> 4) : q * 8 + 4 * (lane >> 5));
    }
};

// Stores a wave's WT x WC block to rows row0 .. of C (leading dimension ldc),
// columns col0 .., those below M and N: f(i, j, q, x) gives four consecutive
// columns.  Through LDS, so that rows leave in 16-byte chunks of whole
// segments; non-temporal where rows lie on 16-byte units, which leaves L2 to
// the operands other tiles still read (else lines are written in parts, which
// L2 has to join).
template <typename T, int WT, int WC, int SH, int LDS, typename F>
__device__ __forceinline__ void store_block(F f, T* C, int64_t ldc, int64_t row0, int64_t col0, int64_t M, int64_t N,
                                            char* lds, int wave, int lane) {
    using G = Frag<WT, SH>;
    constexpr int STR = WC * (int)sizeof(T) + 16;            // padded: the fragments' writes fall on distinct banks
    constexpr int PASSES = 4 * WT * STR <= LDS ? 1 : 2;
    constexpr int PROWS = WT / PASSES;
    constexpr int LPR = WC * (int)sizeof(T) / 16;            // lanes per row on read-out
    constexpr int VEC = Elem<T>::VEC;
    static_assert(4 * PROWS * STR <= LDS, "staging exceeds LDS");
    char* wl = lds + wave * (PROWS * STR);
    const bool units = (((uint64_t)C | (uint64_t)(ldc * (int64_t)sizeof(T))) & 15) == 0;
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
#pragma unroll
        for (int i = 0; i < G::NF; ++i) {
            if (i * G::FR < pass * PROWS || i * G::FR >= (pass + 1) * PROWS) continue;
#pragma unroll
            for (int j = 0; j < WC / G::FR; ++j)
#pragma unroll
                for (int q = 0; q < G::NQ; ++q) {
                    float x[4];
                    f(i, j, q, x);
                    store4<T>((T*)(wl + (G::row(lane, i) - pass * PROWS) * STR + G::col(lane, j, q) * (int)sizeof(T)),
                              x, true);
                }
        }
        // a wave's LDS operations complete in order; the waits keep the
        // compiler from reordering the cross-lane accesses
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 4
        for (int it = 0; it < PROWS * LPR / 64; ++it) {
            const int r = it * (64 / LPR) + lane / LPR, c = lane % LPR;
            const u32x4 v = *(const u32x4*)(wl + r * STR + c * 16);
            const int64_t m = row0 + pass * PROWS + r, n = col0 + c * VEC;
            if (m >= M) continue;
            if (units && n + VEC <= N) __builtin_nontemporal_store(v, (u32x4*)(C + m * ldc + n));
            else st_chunk(C + m * ldc, n, N, v);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

struct GluParams : KParams {
    void *h, *gu;            // gu: null, or the projections (both halves)
    int64_t ldh, ldgu;
};

// h = act(G) * U, and G and U where kept, rounded once from fp32.  Bound by the
// matrix units at the power limit: 8192 x 11008 x 4096 bf16 1.09 ms, 1.35 PFLOP/s
// with 71% of their cycles busy (a plain library product of 8192^3 1.29 PFLOP/s).
template <typename T, int ACT>
struct GluOp {
    using Params = GluParams;
    static constexpr bool PLAIN = false, GATED = true;
    template <int WT, int SH, int LDS, typename ACC>
    static __device__ __forceinline__ void run(const Params& p, ACC& acc, char* lds, int m0, int n0, int wave,
                                               int lane) {
        constexpr int WC = WT / 2, HF = WC / Frag<WT, SH>::FR;
        const int64_t row0 = m0 + (wave >> 1) * WT, col0 = n0 + (wave & 1) * WC;
        auto store = [&](auto f, T* C, int64_t ldc) {
            store_block<T, WT, WC, SH, LDS>(f, C, ldc, row0, col0, p.M, p.N, lds, wave, lane);
        };
        store([&](int i, int j, int q, float* x) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = act<ACT>(acc[i][j][4 * q + e]) * acc[i][j + HF][4 * q + e];
        }, (T*)p.h, p.ldh);
        if (!p.gu) return;
#pragma unroll
        for (int half = 0; half < 2; ++half)
            store([&](int i, int j, int q, float* x) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[i][j + half * HF][4 * q + e];
            }, (T*)p.gu + (int64_t)half * p.N, p.ldgu);
    }
};

struct XentParams : KParams {
    const int64_t* target;   // stats: null without a loss
    int64_t v0;              // the first column's class
    // stats: (max, sum of exp) of each row and each wave's WT columns, and
    // the targets' logits
    float2* parts;
    float* zt;
    // gradient: rows and columns of D stored, zero past M and N
    uint32_t Ms, Ns;
    int64_t V, ignore;
    const float *lse, *dloss;
    Scale scale;
};

// Fragments of rows whose target lies in this wave's columns are rare: f(i, t)
// runs for them alone, t the target's column in the wave's block (or outside
// it, in the other lanes)
template <int WT, int SH, typename F>
__device__ __forceinline__ void at_targets(const XentParams& p, int64_t row0, int64_t col0, int lane, F f) {
    using G = Frag<WT, SH>;
#pragma unroll
    for (int i = 0; i < G::NF; ++i) {
        const int64_t m = row0 + G::row(lane, i);
        const int64_t t = m < p.M ? p.target[m] - p.v0 - col0 : -1;
        const bool in = t >= 0 && t < WT && col0 + t < p.N;
        if (__any(in)) f(i, in ? (int)t : -1, m);
    }
}

// Each row's statistics over a wave's columns, in the accumulators: the
// maximum, then the sum of exponentials, over the lane's columns and the lanes
// that share its row.  4096 x 128000 x 4096 bf16 3.03 ms, 1.42 PFLOP/s, the
// matrix units 72% busy; the logits would be 2 GB written and read in fp32.
template <typename T>
struct XentStatsOp {
    using Params = XentParams;
    static constexpr bool PLAIN = false, GATED = false;
    template <int WT, int SH, int LDS, typename ACC>
    static __device__ __forceinline__ void run(const Params& p, ACC& acc, char*, int m0, int n0, int wave, int lane) {
        using G = Frag<WT, SH>;
        const int64_t row0 = m0 + (wave >> 1) * WT, col0 = n0 + (wave & 1) * WT;
        if (p.target)
            at_targets<WT, SH>(p, row0, col0, lane, [&](int i, int t, int64_t m) {
#pragma unroll
                for (int j = 0; j < G::NF; ++j)
#pragma unroll
                    for (int q = 0; q < G::NQ; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (t == G::col(lane, j, q) + e) p.zt[m] = acc[i][j][4 * q + e];
            });
        const int64_t slice = (p.v0 + n0) / WT + (wave & 1);
        const int left = (int)min((int64_t)WT, p.N - col0);   // columns of this wave (none: not positive)
        auto rows = [&](auto whole) {
#pragma unroll
            for (int i = 0; i < G::NF; ++i) {
                float top = -INFINITY, s = 0.0f;
                auto at = [&](int j, int r) {
                    if constexpr (decltype(whole)::value) return acc[i][j][r];
                    else return G::col(lane, j, r / 4) + r % 4 < left ? acc[i][j][r] : -INFINITY;
                };
#pragma unroll
                for (int j = 0; j < G::NF; ++j)
#pragma unroll
                    for (int r = 0; r < 4 * G::NQ; ++r) top = fmaxf(top, at(j, r));
#pragma unroll
                for (int d = 32; d >= G::FR; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
                const float off = (__builtin_isinf(top) ? 0.0f : top) * LOG2E;
#pragma unroll
                for (int j = 0; j < G::NF; ++j)
#pragma unroll
                    for (int r = 0; r < 4 * G::NQ; ++r)
                        s += __builtin_amdgcn_exp2f(__builtin_fmaf(at(j, r), LOG2E, -off));
#pragma unroll
                for (int d = 32; d >= G::FR; d >>= 1) s += __shfl_xor(s, d);
                const int64_t m = row0 + G::row(lane, i);
                if (lane < G::FR && m < p.M) p.parts[slice * p.M + m] = float2{top, s};
                __builtin_amdgcn_sched_barrier(0);   // one row's copies of the accumulators at a time
            }
        };
        if (left == WT) rows(std::true_type{});
        else rows(std::false_type{});
    }
};

// D = scal * dloss * (exp(z - lse) - [v == target]), rounded to T (as an operand of
// two products).  4096 x 65536 x 4096 bf16 1.67 ms, 1.32 PFLOP/s.
template <typename T>
struct XentGradOp {
    using Params = XentParams;
    static constexpr bool PLAIN = false, GATED = false;
    template <int WT, int SH, int LDS, typename ACC>
    static __device__ __forceinline__ void run(const Params& p, ACC& acc, char* lds, int m0, int n0, int wave,
                                               int lane) {
        using G = Frag<WT, SH>;
        const int64_t row0 = m0 + (wave >> 1) * WT, col0 = n0 + (wave & 1) * WT;
        const float sc = scale_of<T>(p.scale, p.dloss, p.target, p.M, p.V, p.ignore,
                                     blockIdx.x == 0 && wave == 0, lane);
#pragma unroll
        for (int i = 0; i < G::NF; ++i) {
            const int64_t m = row0 + G::row(lane, i);
            const int64_t t = m < p.M ? p.target[m] : p.ignore;
            const bool skip = t == p.ignore;
            const float l = skip ? 0.0f : p.lse[m] * LOG2E;
            const float k = skip ? 0.0f : t >= 0 && t < p.V ? p.dloss[m] * sc : __builtin_nanf("");
#pragma unroll
            for (int j = 0; j < G::NF; ++j)
#pragma unroll
                for (int r = 0; r < 4 * G::NQ; ++r) {
                    const float x = k * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], LOG2E, -l));
                    acc[i][j][r] = skip ? 0.0f : x;
                }
            const int64_t tc = t - p.v0 - col0;
            const bool in = !skip && tc >= 0 && tc < WT;
            if (__any(in)) {
#pragma unroll
                for (int j = 0; j < G::NF; ++j)
#pragma unroll
                    for (int q = 0; q < G::NQ; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (in && tc == G::col(lane, j, q) + e) acc[i][j][4 * q + e] -= k;
            }
        }
        const int left = (int)min((int64_t)WT, p.N - col0);
        if (left < WT) {
#pragma unroll
            for (int j = 0; j < G::NF; ++j)
#pragma unroll
                for (int r = 0; r < 4 * G::NQ; ++r)
                    if (G::col(lane, j, r / 4) + r % 4 >= left) {
#pragma unroll
                        for (int i = 0; i < G::NF; ++i) acc[i][j][r] = 0.0f;
                    }
        }
        store_block<T, WT, WT, SH, LDS>([&](int i, int j, int q, float* x) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[i][j][4 * q + e];
        }, (T*)p.C, p.ldc, row0, col0, p.Ms, p.Ns, lds, wave, lane);
    }
};

}  // namespace vkb
