// few.hip — the operators for a few rows (decode and small batches): products
// bound by one pass over the weight, with what the operator does to them in
// the same pass.
//
// Forward, y = x W^T for up to 16 rows of x: a workgroup takes four rows of W,
// its four waves a quarter of K's chunks each; a lane multiplies its 16 bytes
// of every W row (non-temporal: they stream through once) with the same k of
// every x row (v_dot2 of 16-bit types, fp32 sums), the next chunk's loads in
// flight; then the sums join over lanes and waves in a fixed order.  Rows at any
// alignment.  Gated projection: the four rows are the gate's and the up
// projection's of two columns, so h leaves the same kernel.  Bound by HBM for one
// row (1 x 14336 x 4096 fp16 gated 33.8 us, 6.9 TB/s); from 9 rows on by x, which
// every four rows of W read again from L2: the second kernel, up to 32 rows.
//
// Backward, from D (M x R, R the weight's rows), which is a few values per
// weight row and computed here in fp32, not rounded:
//   dx = D W, dw = D^T x
// as one pass that reads a row of W and writes the same row of dw: a thread
// holds x's columns and dx's sums of its 16 bytes of columns for all M rows (up
// to 8), and walks down a slice of W's rows.  The slices' sums of dx join afterwards.
#include <type_traits>
#include "nn_common.hpp"
#include "vkb_nn_launch.h"

namespace vkb {
namespace {

constexpr int THREADS = 256;

// a + sum of w[i] x[i] over the two 16-bit halves
template <typename T>
__device__ __forceinline__ float dot2(uint32_t w, uint32_t x, float a) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    if constexpr (is_bf16<T>)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), __builtin_bit_cast(b2, x), a, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), __builtin_bit_cast(h2, x), a, false);
}

__device__ __forceinline__ float act_of(int code, float g) {
    return code == VKBLAS_ACT_SILU ? act<VKBLAS_ACT_SILU>(g) : code == VKBLAS_ACT_GELU ? act<VKBLAS_ACT_GELU>(g)
         : code == VKBLAS_ACT_GELU_TANH ? act<VKBLAS_ACT_GELU_TANH>(g) : act<VKBLAS_ACT_RELU>(g);
}
__device__ __forceinline__ void act_and_slope_of(int code, float g, float& a, float& da) {
    if (code == VKBLAS_ACT_SILU) act_and_slope<VKBLAS_ACT_SILU>(g, a, da);
    else if (code == VKBLAS_ACT_GELU) act_and_slope<VKBLAS_ACT_GELU>(g, a, da);
    else if (code == VKBLAS_ACT_GELU_TANH) act_and_slope<VKBLAS_ACT_GELU_TANH>(g, a, da);
    else act_and_slope<VKBLAS_ACT_RELU>(g, a, da);
}

// GLU: R = N columns of h; else R rows of W and y = z, fp32
template <typename T, int MB, bool GLU>
__global__ __launch_bounds__(THREADS) void few_forward_kernel(vkb_few_forward p) {
    constexpr int VEC = Elem<T>::VEC, RB = 4, STEP = 64 * VEC;
    __shared__ float red[4][RB][MB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t first = blockIdx.x * (GLU ? 2 : RB);
    const T* wr[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        // rows past the last are read as the last
        const uint32_t n = min(first + (GLU ? r & 1 : r), p.R - 1);
        wr[r] = (const T*)p.w + ((GLU && r >= 2 ? (int64_t)p.R : 0) + n) * p.ldw;
    }
    const T* x = (const T*)p.x;
    const uint32_t K = p.K, chunks = (K + STEP - 1) / STEP;
    float acc[RB][MB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[r][m] = 0.0f;
    u32x4 wc[RB], xc[MB];
    // lanes past K read its last chunk, and one that straddles it too: their
    // elements before k are dropped below
    auto load = [&](uint32_t c, u32x4* w, u32x4* xv) {
        const uint32_t k = min(c * STEP + lane * VEC, K - VEC);
#pragma unroll
        for (int m = 0; m < MB; ++m) xv[m] = ld16_any(x + (int64_t)min((uint32_t)m, p.M - 1) * p.ldx + k);
#pragma unroll
        for (int r = 0; r < RB; ++r) w[r] = __builtin_nontemporal_load((const u32x4_any*)(wr[r] + k));
    };
    auto drop = [&](u32x4 v, int from) {   // zeros for elements before `from`
        float f[VEC];
        unpack<T>(v, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = e < from ? 0.0f : f[e];
        return pack<T>(f);
    };
    if ((uint32_t)wave < chunks) load(wave, wc, xc);
    for (uint32_t c = wave; c < chunks; c += 4) {
        u32x4 w[RB], xv[MB];
#pragma unroll
        for (int r = 0; r < RB; ++r) w[r] = wc[r];
#pragma unroll
        for (int m = 0; m < MB; ++m) xv[m] = xc[m];
        if (c + 4 < chunks) load(c + 4, wc, xc);
        if (c * STEP + STEP > K) {   // the last chunk
            const uint32_t k = c * STEP + lane * VEC;
            const int from = (int)min(k - min(k, K - VEC), (uint32_t)VEC);
#pragma unroll
            for (int r = 0; r < RB; ++r) w[r] = drop(w[r], from);
#pragma unroll
            for (int m = 0; m < MB; ++m) xv[m] = drop(xv[m], from);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (sizeof(T) == 4)
                        acc[r][m] = __builtin_fmaf(__uint_as_float(w[r][e]), __uint_as_float(xv[m][e]), acc[r][m]);
                    else
                        acc[r][m] = dot2<T>(w[r][e], xv[m][e], acc[r][m]);
                }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const float s = wave_sum(acc[r][m]);
            if (lane == 0) red[wave][r][m] = s;
        }
    __syncthreads();
    constexpr int OUTS = GLU ? 2 : RB;
    if (threadIdx.x >= OUTS * MB) return;
    const uint32_t m = threadIdx.x / OUTS, r = threadIdx.x % OUTS, n = first + r;
    if (m >= p.M || n >= p.R) return;
    auto sum = [&](uint32_t row) { return red[0][row][m] + red[1][row][m] + red[2][row][m] + red[3][row][m]; };
    if constexpr (GLU) {
        const float g = sum(r), u = sum(r + 2);
        ((T*)p.y)[(int64_t)m * p.ldy + n] = (T)(act_of(p.act, g) * u);
        if (p.gu) {
            T* gu = (T*)p.gu + (int64_t)m * p.ldgu + n;
            gu[0] = (T)g;
            gu[p.R] = (T)u;
        }
    } else {
        ((float*)p.y)[(int64_t)m * p.ldy + n] = sum(r);
    }
}

// ... for more rows of x and many of W (vkb_few_mfma): 16 rows of W times MF fragments of 16 x rows on
// the matrix units, RF fragments of W's rows a wave (gated: one of the gate's,
// one of the up projection's).  A lane's 16 bytes of a row, at any alignment, are
// its part of a 64-byte step of k, four steps at a time and the next four in
// flight; the workgroup's waves take every fourth four steps.  us, the kernel
// above / this, cross entropy bf16: 10 x 126144 x 4502 536 / 316, 16 x 32003 x 1027 118 /
// 35, 12 x 2003 x 4101 19.6 / 24.2, 5 x 107712 x 6965 408 / 552 (rows at 2-byte
// alignment: 2.7 TB/s; at 4 bytes 3.6).
template <typename T, int MF, int RF, bool GLU>
__global__ __launch_bounds__(THREADS) void few_mfma_kernel(vkb_few_forward p) {
    constexpr int VEC = Elem<T>::VEC, U = 4, STEP = 4 * VEC * U;
    static_assert(!GLU || RF == 2, "gate and up projection");
    __shared__ floatx4 red[4][RF][MF][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const uint32_t first = blockIdx.x * (GLU ? 16 : 16 * RF);
    const T *wr[RF], *xr[MF];
    // rows past the last are read as the last
#pragma unroll
    for (int f = 0; f < RF; ++f) {
        const uint32_t n = min(first + (GLU ? 0 : 16 * f) + r, p.R - 1);
        wr[f] = (const T*)p.w + ((GLU && f ? (int64_t)p.R : 0) + n) * p.ldw;
    }
#pragma unroll
    for (int f = 0; f < MF; ++f) xr[f] = (const T*)p.x + (int64_t)min((uint32_t)(16 * f + r), p.M - 1) * p.ldx;
    const uint32_t K = p.K, steps = (K + STEP - 1) / STEP;
    floatx4 acc[RF][MF];
#pragma unroll
    for (int i = 0; i < RF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    u32x4 wn[U][RF], xn[U][MF];
    // a chunk past K is read as K's last, and one that straddles it too
    auto load = [&](uint32_t s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = min(s * STEP + (4 * u + g) * VEC, K - VEC);
#pragma unroll
            for (int f = 0; f < RF; ++f) wn[u][f] = ld16_any(wr[f] + k);
#pragma unroll
            for (int f = 0; f < MF; ++f) xn[u][f] = ld16_any(xr[f] + k);
        }
    };
    auto drop = [&](u32x4 v, int from) {   // zeros for elements before `from`
        float f[VEC];
        unpack<T>(v, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = e < from ? 0.0f : f[e];
        return pack<T>(f);
    };
    if ((uint32_t)wave < steps) load(wave);
    for (uint32_t s = wave; s < steps; s += 4) {
        u32x4 w[U][RF], x[U][MF];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int f = 0; f < RF; ++f) w[u][f] = wn[u][f];
#pragma unroll
            for (int f = 0; f < MF; ++f) x[u][f] = xn[u][f];
        }
        if (s + 4 < steps) load(s + 4);
        if (s * STEP + STEP > K) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t k = s * STEP + (4 * u + g) * VEC;
                const int from = (int)min(k - min(k, K - VEC), (uint32_t)VEC);
#pragma unroll
                for (int f = 0; f < RF; ++f) w[u][f] = drop(w[u][f], from);
#pragma unroll
                for (int f = 0; f < MF; ++f) x[u][f] = drop(x[u][f], from);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RF; ++i)
#pragma unroll
                for (int j = 0; j < MF; ++j) {
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(w[u][i][e]), __uint_as_float(x[u][j][e]), acc[i][j], 0, 0, 0);
                    } else {
                        acc[i][j] = mfma_16x16x32<T>(w[u][i], x[u][j], acc[i][j]);
                    }
                }
    }
#pragma unroll
    for (int i = 0; i < RF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j) red[wave][i][j][lane] = acc[i][j];
    __syncthreads();
    // a wave's lanes: rows n .. n + 3 of W, row m of x
    constexpr int OUTS = GLU ? MF : RF * MF;
    for (int o = wave; o < OUTS; o += 4) {
        const int i = o / MF, j = o % MF;
        const uint32_t n = first + 16 * i + 4 * g, m = 16 * j + r;
        floatx4 a = red[0][i][j][lane], b = red[0][RF - 1][j][lane];
#pragma unroll
        for (int v = 1; v < 4; ++v) {
            a += red[v][i][j][lane];
            if (GLU) b += red[v][RF - 1][j][lane];
        }
        if (m >= p.M) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (n + e >= p.R) break;
            if constexpr (GLU) {
                ((T*)p.y)[(int64_t)m * p.ldy + n + e] = (T)(act_of(p.act, a[e]) * b[e]);
                if (p.gu) {
                    T* gu = (T*)p.gu + (int64_t)m * p.ldgu + n + e;
                    gu[0] = (T)a[e];
                    gu[p.R] = (T)b[e];
                }
            } else {
                ((float*)p.y)[(int64_t)m * p.ldy + n + e] = a[e];
            }
        }
    }
}

// D[m][v] of the two operators
template <typename T, bool GLU>
__device__ __forceinline__ float few_d(const vkb_few_backward& p, uint32_t m, uint32_t v) {
    if constexpr (GLU) {
        const uint32_t N = p.R / 2, n = v < N ? v : v - N;
        const T* gu = (const T*)p.gu + (int64_t)m * p.ldgu;
        const float d = (float)((const T*)p.dh)[(int64_t)m * p.lddh + n];
        float a, da;
        act_and_slope_of(p.act, (float)gu[n], a, da);
        return v < N ? d * (float)gu[N + n] * da : d * a;
    } else {
        const int64_t t = p.target[m];
        if (t == p.ignore) return 0.0f;
        const float k = t >= 0 && t < p.R ? p.dloss[m] : __builtin_nanf("");
        return k * (fast_exp(p.z[(int64_t)m * p.ldz + v] - p.lse[m]) - (v == t ? 1.0f : 0.0f));
    }
}

template <typename T, typename G, int MB, bool GLU>
__global__ __launch_bounds__(THREADS) void few_backward_kernel(vkb_few_backward p) {
    constexpr int VC = Elem<T>::VEC;                         // columns of a thread
    constexpr int DB = 64, U = 4;                           // rows of D at a time, of W in flight
    typedef T tvec __attribute__((ext_vector_type(VC), aligned(sizeof(T))));
    typedef G gvec __attribute__((ext_vector_type(VC), aligned(sizeof(G))));
    __shared__ float D[DB][MB];
    const uint32_t kt = threadIdx.x % p.kthreads, grp = threadIdx.x / p.kthreads, groups = THREADS / p.kthreads;
    const uint32_t n = (blockIdx.x * p.kthreads + kt) * VC;
    // the row's last columns are read from K - VC on; those before n are another thread's
    const bool live = n < p.K;
    const uint32_t off = min(n, p.K - VC);
    const int from = (int)(min(n, p.K) - off);
    const bool whole = __all(!live || from == 0);   // the same in all lanes of a wave
    float x[MB][VC], dx[MB][VC];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        tvec v{};
        if (p.dw) v = *(const tvec*)((const T*)p.x + (int64_t)min((uint32_t)m, p.M - 1) * p.ldx + off);
#pragma unroll
        for (int e = 0; e < VC; ++e) {
            x[m][e] = (float)v[e];
            dx[m][e] = 0.0f;
        }
    }
    const uint32_t v0 = blockIdx.y * p.slice, v1 = min(p.R, v0 + p.slice);
    for (uint32_t v = v0; v < v1; v += DB) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < DB * MB; i += THREADS) {
            const uint32_t r = i % DB, m = i / DB;
            D[r][m] = m < p.M && v + r < v1 ? few_d<T, GLU>(p, m, v + r) : 0.0f;
        }
        __syncthreads();
        if (!live) continue;
        const uint32_t rows = min((uint32_t)DB, v1 - v);
        auto load = [&](uint32_t r0, tvec* w) {   // rows past the last are read as the last
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t r = min(r0 + u * groups, rows - 1);
                w[u] = *(const tvec*)((const T*)p.w + (int64_t)(v + r) * p.ldw + off);
            }
        };
        auto row = [&](uint32_t r, tvec w) {
            float d[MB], o[VC];
#pragma unroll
            for (int m = 0; m < MB; ++m) d[m] = D[r][m];
            if (p.part)
#pragma unroll
                for (int m = 0; m < MB; ++m)
#pragma unroll
                    for (int e = 0; e < VC; ++e) dx[m][e] = __builtin_fmaf(d[m], (float)w[e], dx[m][e]);
            if (!p.dw) return;
#pragma unroll
            for (int e = 0; e < VC; ++e) o[e] = 0.0f;
#pragma unroll
            for (int m = 0; m < MB; ++m)
                if (m < (int)p.M)   // a row past M is another's x, whose infinities would make NaN of D = 0
#pragma unroll
                    for (int e = 0; e < VC; ++e) o[e] = __builtin_fmaf(d[m], x[m][e], o[e]);
            G* out = (G*)p.dw + (int64_t)(v + r) * p.lddw + off;
            gvec g;
            if (whole) {
                if (p.beta != 0.0f) {
                    g = *(const gvec*)out;
#pragma unroll
                    for (int e = 0; e < VC; ++e) o[e] += p.beta * (float)g[e];
                }
#pragma unroll
                for (int e = 0; e < VC; ++e) g[e] = (G)o[e];
                *(gvec*)out = g;
            } else {
#pragma unroll
                for (int e = 0; e < VC; ++e)
                    if (e >= from) out[e] = (G)(p.beta != 0.0f ? o[e] + p.beta * (float)out[e] : o[e]);
            }
        };
        // the next U rows' loads leave before these rows' stores, and are not
        // waited for together with them
        tvec w[U]{}, next[U]{};
        uint32_t r0 = grp;
        if (p.part) load(r0, next);
        for (; r0 + (U - 1) * groups < rows; r0 += U * groups) {
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = next[u];
            if (p.part) load(r0 + U * groups, next);
#pragma unroll
            for (int u = 0; u < U; ++u) row(r0 + u * groups, w[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r0 + u * groups < rows) row(r0 + u * groups, next[u]);
    }
    if (!p.part || !live) return;
    float* part = p.part + (int64_t)(blockIdx.y * groups + grp) * p.M * p.K + off;
#pragma unroll
    for (int m = 0; m < MB; ++m)
        if (m < (int)p.M)
#pragma unroll
            for (int e = 0; e < VC; ++e)
                if (e >= from) part[(int64_t)m * p.K + e] = dx[m][e];
}

// dx from the parts: 16 columns of the M K per workgroup, each thread of a
// column adds 1/64 of the parts in order, 16 loads in flight, and the sums join
// in a fixed tree.  (Many parts of few columns: the split-K reduce, which gives
// a column four threads, took longer than the pass itself.)
template <typename T>
__global__ __launch_bounds__(1024) void few_reduce_kernel(const float* part, uint32_t parts, uint64_t cols, uint32_t K,
                                                          T* dx, int64_t lddx) {
    __shared__ float sh[16][16];
    const uint32_t c = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const uint64_t n = (uint64_t)blockIdx.x * 16 + c;
    const uint32_t p0 = (uint32_t)((uint64_t)parts * slice / 64), p1 = (uint32_t)((uint64_t)parts * (slice + 1) / 64);
    float s = 0.0f;
    if (n < cols)
        for (uint32_t p = p0; p < p1; p += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = p + i < p1 ? part[(uint64_t)(p + i) * cols + n] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += v[i];
        }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 63) < 16) sh[threadIdx.x >> 6][c] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || n >= cols) return;
    s = sh[0][c];
    for (int i = 1; i < 16; ++i) s += sh[i][c];
    const uint64_t m = n / K;
    dx[(int64_t)m * lddx + (int64_t)(n - m * K)] = (T)s;
}

// f(integral_constant<int, MB>) with MB >= M a power of two
template <int MOST, typename F>
static void with_rows(uint32_t M, F f) {
    using std::integral_constant;
    if (M <= 1) f(integral_constant<int, 1>{});
    else if (M <= 2) f(integral_constant<int, 2>{});
    else if (M <= 4) f(integral_constant<int, 4>{});
    else if (M <= 8) f(integral_constant<int, 8>{});
    else if constexpr (MOST > 8) f(integral_constant<int, 16>{});
}

static uint32_t backward_columns(int type) { return type == VKB_T_F32 ? 4 : 8; }

}  // namespace
}  // namespace vkb

using namespace vkb;

// One fragment of W's rows a wave where two would leave CUs without work (us,
// one / two: 16 x 32003 x 1027 bf16 41 / 34, 12 x 2003 x 4101 24 / 34).
static int few_mfma(int type, const vkb_few_forward* p, int glu, hipStream_t st) {
    const int rf = glu || p->R >= 16384 ? 2 : 1;
    const uint64_t rows = glu ? 16 : 16 * rf, grid = (p->R + rows - 1) / rows;
    if (grid > 0xffffffffull / THREADS) return (int)hipErrorInvalidValue;
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(THREADS), 0, st, *p);
        };
        if (p->M <= 16) {
            if (glu) go(few_mfma_kernel<T, 1, 2, true>);
            else if (rf == 2) go(few_mfma_kernel<T, 1, 2, false>);
            else go(few_mfma_kernel<T, 1, 1, false>);
        } else {
            if (glu) go(few_mfma_kernel<T, 2, 2, true>);
            else if (rf == 2) go(few_mfma_kernel<T, 2, 2, false>);
            else go(few_mfma_kernel<T, 2, 1, false>);
        }
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_few_forward(int type, const vkb_few_forward* p, int glu, void* stream) {
    if (p->M == 0 || (p->M > 16 && !vkb_few_mfma(p->M, glu ? 2 * (uint64_t)p->R : p->R)) || p->R == 0 || p->K < (type == VKB_T_F32 ? 4u : 8u)) return (int)hipErrorInvalidValue;
    if (vkb_few_mfma(p->M, glu ? 2 * (uint64_t)p->R : p->R)) return few_mfma(type, p, glu, (hipStream_t)stream);
    const uint64_t grid = ((uint64_t)p->R + (glu ? 1 : 3)) / (glu ? 2 : 4);
    if (grid > 0xffffffffull / THREADS) return (int)hipErrorInvalidValue;
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        with_rows<16>(p->M, [&](auto mb) {
            if (glu)
                hipLaunchKernelGGL((few_forward_kernel<T, mb.value, true>), dim3((uint32_t)grid), dim3(THREADS), 0,
                                   (hipStream_t)stream, *p);
            else
                hipLaunchKernelGGL((few_forward_kernel<T, mb.value, false>), dim3((uint32_t)grid), dim3(THREADS), 0,
                                   (hipStream_t)stream, *p);
        });
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

// How the backward kernel divides R rows of K columns: threads along K (the
// others of a workgroup take other rows), rows of a slice.  About 1024
// workgroups, and sums of dx of at most an eighth of the weight's bytes or 8 MiB.
extern "C" uint32_t vkb_few_slices(int type, vkb_few_backward* p) {
    const uint32_t chunks = (p->K + backward_columns(type) - 1) / backward_columns(type);
    p->kthreads = chunks <= 64 ? 64 : chunks <= 128 ? 128 : 256;
    const uint32_t groups = THREADS / p->kthreads;
    const uint64_t kb = (chunks + p->kthreads - 1) / p->kthreads;
    uint64_t s = (1024 + kb - 1) / kb;
    const uint64_t weight = (uint64_t)p->R * p->K * (type == VKB_T_F32 ? 4 : 2) / 8;
    const uint64_t bytes = weight > (8u << 20) ? weight : (8u << 20);
    const uint64_t most = bytes / ((uint64_t)groups * p->M * p->K * 4);
    if (s > most) s = most;
    if (s > p->R / (4 * groups)) s = p->R / (4 * groups);   // four rows in flight a thread
    if (s > 65535) s = 65535;
    if (s < 1) s = 1;
    p->slice = (uint32_t)((p->R + s - 1) / s);
    return (p->R + p->slice - 1) / p->slice * groups;
}

extern "C" int vkb_launch_few_backward(int type, int g_type, const vkb_few_backward* p, int glu, void* stream) {
    const uint32_t vc = backward_columns(type);
    if (p->M == 0 || p->M > VKB_FEW_BACK || p->R == 0 || p->K < vc || !p->kthreads || !p->slice) return (int)hipErrorInvalidValue;
    if (g_type != type && g_type != VKB_T_F32) return (int)hipErrorInvalidValue;
    const uint32_t chunks = (p->K + vc - 1) / vc;
    const dim3 grid((chunks + p->kthreads - 1) / p->kthreads, (p->R + p->slice - 1) / p->slice);
    if (grid.y > 65535) return (int)hipErrorInvalidValue;
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        with_rows<VKB_FEW_BACK>(p->M, [&](auto mb) {
            auto go = [&](auto g) {
                using G = decltype(g);
                if (glu)
                    hipLaunchKernelGGL((few_backward_kernel<T, G, mb.value, true>), grid, dim3(THREADS), 0,
                                       (hipStream_t)stream, *p);
                else
                    hipLaunchKernelGGL((few_backward_kernel<T, G, mb.value, false>), grid, dim3(THREADS), 0,
                                       (hipStream_t)stream, *p);
            };
            if (g_type == VKB_T_F32) go(float{});
            else go(t);
        });
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_few_reduce(int type, const float* part, uint32_t parts, uint32_t M, uint32_t K, void* dx,
                                     int64_t lddx, void* stream) {
    const uint64_t cols = (uint64_t)M * K, grid = (cols + 15) / 16;
    if (grid == 0 || grid > 0xffffffffull / 1024) return (int)hipErrorInvalidValue;
    const bool ok = with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((few_reduce_kernel<T>), dim3((uint32_t)grid), dim3(1024), 0, (hipStream_t)stream, part, parts,
                           cols, K, (T*)dx, lddx);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
