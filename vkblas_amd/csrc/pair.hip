// pair.hip — the two products of a small gradient in one launch,
//   dx = D W (M x K over R) and dw = beta dw + D^T x (R x K over M),
// each on gemm_direct.hpp's tiles: the first na workgroups take dx's, the others
// dw's.  Such products are a chain of load latencies on a part of the chip, so
// side by side they take the longer one's time and one launch instead of two
// (us, with the pass that makes D, one after the other / this: M R K bf16 25 128 1088
// 16.8 / 12.7, 1535 2176 192 37.6 / 27.0, fp32 1000 2000 300 65.5 / 49.6).
#include "gemm_direct.hpp"
#include "vkb_launch.h"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

struct PairParams {
    KParams dx, dw;
    uint32_t na;
};

template <typename T, typename TW, int F, int U>
__global__ __launch_bounds__(256) void direct_pair_kernel(PairParams p) {
    __shared__ DirectSums<F, F> sums;
    if (blockIdx.x < p.na) direct_tile_run<T, T, true, false, F, F, U>(p.dx, blockIdx.x, p.na, sums);
    else direct_tile_run<T, TW, false, false, F, F, U>(p.dw, blockIdx.x - p.na, gridDim.x - p.na, sums);
}

static KParams product(const void* A, uint32_t lda, const void* B, uint32_t ldb, void* C, uint32_t ldc, uint32_t M,
                       uint32_t N, uint32_t K, const vkb_pair_scalars* s, uint32_t tile) {
    KParams p{};
    p.A = A;
    p.B = B;
    p.C = C;
    p.lda = lda;
    p.ldb = ldb;
    p.ldc = ldc;
    p.M = M;
    p.N = N;
    p.K = p.kps = K;
    p.split = p.batch = 1;
    p.alpha = s->alpha;
    p.beta = s->beta;
    p.alpha_dev = s->alpha_dev;
    p.beta_dev = s->beta_dev;
    p.scalar_mode = s->alpha_dev ? VKB_SCALAR_DEV_F32 : VKB_SCALAR_HOST;
    p.epi.cin = C;
    p.epi.ldcin = ldc;
    p.tiles_m = (M + tile - 1) / tile;
    p.tiles_n = (N + tile - 1) / tile;
    return p;
}

}  // namespace
}  // namespace vkb

using namespace vkb;

// 64 x 64 tiles where they are at least 144, in fp32 512, else 32 x 32 (us, 64 / 32:
// fp32 200 1000 784 29.2 / 22.1, 1535 2176 192 57.5 / 51.2; bf16 there 27.0 / 30.5)
static uint32_t pair_tile(int type, uint32_t M, uint32_t R, uint32_t K) {
    const uint64_t t = (uint64_t)(K + 63) / 64 * ((M + 63) / 64 + (R + 63) / 64);
    return R >= 64 && K >= 64 && t >= (type == VKB_T_F32 ? 512 : 144) ? 64 : 32;
}

extern "C" int vkb_pair_fits(int type, uint32_t M, uint32_t R, uint32_t K, uint32_t ldd, uint32_t ldw, uint32_t ldx) {
    // whole tiles across an operand that is read across, 32-bit offsets of a tile's rows
    const uint64_t ld = ldd > ldw ? (ldd > ldx ? ldd : ldx) : (ldw > ldx ? ldw : ldx);
    const uint64_t grid = (uint64_t)(K + 31) / 32 * ((M + 31) / 32 + (R + 31) / 32);
    return R >= 32 && K >= 32 && (64 * ld + 64) * (type == VKB_T_F32 ? 4 : 2) < 1ull << 31 && grid < 1u << 24;
}

extern "C" int vkb_launch_pair(int type, int w_type, uint32_t M, uint32_t R, uint32_t K, const void* d, uint32_t ldd,
                               const void* w, uint32_t ldw, void* dx, uint32_t lddx, const vkb_pair_scalars* sx,
                               const void* x, uint32_t ldx, void* dw, uint32_t lddw, const vkb_pair_scalars* sw,
                               void* stream) {
    if (!M || !vkb_pair_fits(type, M, R, K, ldd, ldw, ldx)) return (int)hipErrorInvalidValue;
    const uint32_t tile = pair_tile(type, M, R, K);
    PairParams p;
    p.dx = product(d, ldd, w, ldw, dx, lddx, M, K, R, sx, tile);
    p.dw = product(d, ldd, x, ldx, dw, lddw, R, K, M, sw, tile);
    p.na = p.dx.tiles_m * p.dx.tiles_n;
    const uint32_t grid = p.na + p.dw.tiles_m * p.dw.tiles_n;
    auto go = [&](auto t, auto tw) {
        using T = decltype(t);
        using TW = decltype(tw);
        if (tile == 64)
            hipLaunchKernelGGL((direct_pair_kernel<T, TW, 4, 4>), dim3(grid), dim3(256), 0, (hipStream_t)stream, p);
        else
            hipLaunchKernelGGL((direct_pair_kernel<T, TW, 2, 8>), dim3(grid), dim3(256), 0, (hipStream_t)stream, p);
    };
    const bool wide = w_type == VKB_T_F32;
    if (type == VKB_T_F32) go(0.0f, 0.0f);
    else if (type == VKB_T_F16 && wide) go((_Float16)0, 0.0f);
    else if (type == VKB_T_F16) go((_Float16)0, (_Float16)0);
    else if (wide) go((__bf16)0.0f, 0.0f);
    else go((__bf16)0.0f, (__bf16)0.0f);
    return (int)hipGetLastError();
}
