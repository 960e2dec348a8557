// glu_direct.hip — the gated projection of a small call in one launch, on
// gemm_direct.hpp's tiles:
//   [G | U] = x W^T,  h = act(G) * U
// A workgroup's tile holds NG fragments of 16 gate columns and as many of the
// same columns of the up projection, so act(G) * U takes both from the four
// waves' sums in LDS and neither goes through memory.  Bound by latency, as the
// products on these tiles: the second launch and its pass over fp32 projections
// are what it saves.  Operands and results of any element alignment.
#include "gemm_direct.hpp"
#include "nn_common.hpp"

namespace vkb {
namespace {

struct GluDirectParams {
    const void *x, *w;
    void *h, *gu;
    int64_t ldx, ldw, ldh, ldgu;
    uint32_t M, N, K, tiles_m;
};

// Columns n0 .. n0 + 16 NG - 1 of the gate, then of the up projection: the B
// operand of a tile (interface of DirectOperand<T, true, 2 NG>).
template <typename T, int NG>
struct GatedOperand {
    DirectOperand<T, true, NG> half[2];
    __device__ __forceinline__ void init(const T* w, int64_t ld, int n0, int N, int r, int g) {
        half[0].init(w, ld, n0, N, 0, r, g);
        half[1].init(w + (int64_t)N * ld, ld, n0, N, 0, r, g);
    }
    __device__ __forceinline__ void load(uint32_t (&v)[8 * NG], int k) const {
        half[0].load(*(uint32_t(*)[4 * NG])v, k);
        half[1].load(*(uint32_t(*)[4 * NG])(v + 4 * NG), k);
    }
    __device__ __forceinline__ void load_tail(uint32_t (&v)[8 * NG], int k, int nk, int g) const {
        half[0].load_tail(*(uint32_t(*)[4 * NG])v, k, nk, g);
        half[1].load_tail(*(uint32_t(*)[4 * NG])(v + 4 * NG), k, nk, g);
    }
    __device__ __forceinline__ u32x4 frag(const uint32_t (&v)[8 * NG], int i) const {
        return u32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    }
};

// four values of a row from n on, of which those below N exist
template <typename T>
__device__ __forceinline__ void st4(T* row, int n, int N, const float* x) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef t4 t4_any __attribute__((aligned(2), may_alias));
    if (n + 4 <= N) {
        t4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)x[e];
        *(t4_any*)(row + n) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < N) row[n + e] = (T)x[e];
}

template <typename T, int ACT, int MF, int NG, int U>
__global__ __launch_bounds__(256) void glu_direct_kernel(GluDirectParams p) {
    constexpr int TM = 16 * MF, TN = 16 * NG, LDR = DirectSums<MF, 2 * NG>::LDR;
    __shared__ DirectSums<MF, 2 * NG> sums;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t bid = blockIdx.x;   // neighbouring tiles on one XCD
    if ((gridDim.x & 7u) == 0) bid = (bid & 7u) * (gridDim.x >> 3) + (bid >> 3);
    const int m0 = (int)(bid % p.tiles_m) * TM, n0 = (int)(bid / p.tiles_m) * TN;
    const int M = (int)p.M, N = (int)p.N;

    DirectOperand<T, true, MF> oa;
    GatedOperand<T, NG> ob;
    oa.init((const T*)p.x, p.ldx, m0, M, 0, r, g);
    ob.init((const T*)p.w, p.ldw, n0, N, r, g);
    direct_sums<T, true, true, MF, 2 * NG, U>(oa, ob, (int)p.K, sums);

    for (int q = threadIdx.x; q < TM * TN / 4; q += 256) {
        const int ml = q / (TN / 4), nl = 4 * (q % (TN / 4)), m = m0 + ml, n = n0 + nl;
        if (m >= M || n >= N) continue;
        float z[2][4] = {};
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const floatx4 y = *(const floatx4*)&sums.wave[w][ml * LDR + half * TN + nl];
#pragma unroll
                for (int e = 0; e < 4; ++e) z[half][e] += y[e];
            }
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = act<ACT>(z[0][e]) * z[1][e];
        st4((T*)p.h + (int64_t)m * p.ldh, n, N, o);
        if (p.gu) {
            T* row = (T*)p.gu + (int64_t)m * p.ldgu;
            st4(row, n, N, z[0]);
            st4(row + N, n, N, z[1]);
        }
    }
}

static uint64_t tiles(uint32_t M, uint32_t N, uint32_t tm, uint32_t tn) {
    return (uint64_t)((M + tm - 1) / tm) * ((N + tn - 1) / tn);
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" int vkb_glu_direct_fits(int type, uint32_t M, uint32_t N, uint32_t K, uint32_t ldx, uint32_t ldw) {
    // 32-bit offsets of a tile's rows
    const uint64_t ld = ldx > ldw ? ldx : ldw;
    return (64 * ld + 64) * (type == VKB_T_F32 ? 4 : 2) < 1ull << 31 && tiles(M, N, 32, 16) < 1u << 24 && K < 1u << 30;
}

extern "C" int vkb_launch_glu_direct(int type, int act_code, uint32_t M, uint32_t N, uint32_t K, const void* x,
                                     uint32_t ldx, const void* w, uint32_t ldw, void* h, uint32_t ldh, void* gu,
                                     uint32_t ldgu, void* stream) {
    if (!M || !N || !K || !vkb_glu_direct_fits(type, M, N, K, ldx, ldw)) return (int)hipErrorInvalidValue;
    const uint64_t t64 = tiles(M, N, 64, 32);
    // (us, small / large tiles, of the large ones in brackets: fp32 1000 x 250 x 784 (128)
    // 15.9 / 20.9, 400 x 1000 x 784 (224) 28.7 / 21.0; bf16 400 x 1000 x 301 14.5 / 9.1)
    const bool large = t64 >= 144;
    const uint32_t tm = large ? 64 : 32;
    const GluDirectParams p = {x, w, h, gu, ldx, ldw, ldh, ldgu, M, N, K, (M + tm - 1) / tm};
    const uint32_t grid = (uint32_t)(large ? t64 : tiles(M, N, 32, 16));
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        with_act(act_code, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            if (large)
                hipLaunchKernelGGL((glu_direct_kernel<T, ACT, 4, 2, 4>), dim3(grid), dim3(256), 0, (hipStream_t)stream, p);
            else
                hipLaunchKernelGGL((glu_direct_kernel<T, ACT, 2, 1, 8>), dim3(grid), dim3(256), 0, (hipStream_t)stream, p);
        });
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
