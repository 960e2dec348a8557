// policy.hip — clipped policy loss with a KL term on token log probabilities.
//
// A token's loss is a few operations on four or five floats, so the loss over a
// batch is a pass over its arrays and a sum.  A wave takes a unit, a part of a
// sequence, four tokens a lane at a time, and skips the arrays where no token
// of a lane's four counts: the padding behind a sequence costs its mask alone.
// A token's terms are fp32; sums are fp64, and so is logp - old, on which the
// side of a bound depends: r > 1 + clip_high exactly where logp - old >
// log(1 + clip_high).
#include "nn_common.hpp"

namespace vkb {
namespace {

// exp(d) - d - 1 without the cancellation of a small d: d^2 sum d^k / (k + 2)!
// within |d| <= 1 (the 11th term is below 2^-28 of the first)
__device__ __forceinline__ float kl_term(float d) {
    if (fabsf(d) > 1.0f) return fast_exp(d) - d - 1.0f;
    float s = 1.0f / 479001600.0f;
    s = __builtin_fmaf(s, d, 1.0f / 39916800.0f);
    s = __builtin_fmaf(s, d, 1.0f / 3628800.0f);
    s = __builtin_fmaf(s, d, 1.0f / 362880.0f);
    s = __builtin_fmaf(s, d, 1.0f / 40320.0f);
    s = __builtin_fmaf(s, d, 1.0f / 5040.0f);
    s = __builtin_fmaf(s, d, 1.0f / 720.0f);
    s = __builtin_fmaf(s, d, 1.0f / 120.0f);
    s = __builtin_fmaf(s, d, 1.0f / 24.0f);
    s = __builtin_fmaf(s, d, 1.0f / 6.0f);
    s = __builtin_fmaf(s, d, 0.5f);
    return s * d * d;
}
// 1 - exp(d), likewise
__device__ __forceinline__ float kl_slope(float d) {
    if (fabsf(d) > 1.0f) return 1.0f - fast_exp(d);
    float s = 1.0f / 39916800.0f;
    s = __builtin_fmaf(s, d, 1.0f / 3628800.0f);
    s = __builtin_fmaf(s, d, 1.0f / 362880.0f);
    s = __builtin_fmaf(s, d, 1.0f / 40320.0f);
    s = __builtin_fmaf(s, d, 1.0f / 5040.0f);
    s = __builtin_fmaf(s, d, 1.0f / 720.0f);
    s = __builtin_fmaf(s, d, 1.0f / 120.0f);
    s = __builtin_fmaf(s, d, 1.0f / 24.0f);
    s = __builtin_fmaf(s, d, 1.0f / 6.0f);
    s = __builtin_fmaf(s, d, 0.5f);
    s = __builtin_fmaf(s, d, 1.0f);
    return -s * d;
}

struct Token {
    float r, adv, d;         // ratio, advantage, ref - logp
    int side;                // 0: r A is taken, -1: the lower bound's, 1: the upper one's
};
// A NaN anywhere takes r A, which it reaches.
__device__ __forceinline__ Token token(const vkb_policy& p, float logp, float old, float ref, float adv) {
    const double diff = (double)logp - (double)old;
    Token t;
    t.r = fast_exp((float)diff);
    t.adv = adv;
    t.d = ref - logp;
    t.side = adv > 0.0f && diff > p.high ? 1 : adv < 0.0f && diff < p.low ? -1 : 0;
    return t;
}

// The tokens t .. t + 3 of sequence b that count, as bits
__device__ __forceinline__ uint32_t counted(const vkb_policy& p, int64_t b, int64_t t) {
    const int64_t left = p.T - t;
    if (left <= 0) return 0;
    uint32_t in = 0;
    if (!p.mask) in = 15;
    else {
        const uint8_t* m = p.mask + b * p.ldmask + t;
        if (left >= 4) {
            uint32_t v;
            __builtin_memcpy(&v, m, 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) in |= (v >> (8 * e) & 255 ? 1u : 0u) << e;
        } else {
            for (int e = 0; e < left; ++e) in |= (m[e] ? 1u : 0u) << e;
        }
    }
    return left >= 4 ? in : in & ((1u << left) - 1);
}
struct Four {
    float logp[4], old[4], ref[4], adv[4];
};
__device__ __forceinline__ void load4(const vkb_policy& p, int64_t b, int64_t t, Four& f) {
    unpack<float>(ld_chunk(p.logp + b * p.ldp, t, p.T), f.logp);
    unpack<float>(ld_chunk(p.old + b * p.ldo, t, p.T), f.old);
    if (p.ref) unpack<float>(ld_chunk(p.ref + b * p.ldr, t, p.T), f.ref);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) f.ref[e] = f.logp[e];
    if (p.adv_step) unpack<float>(ld_chunk(p.adv + b * p.ldadv, t, p.T), f.adv);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) f.adv[e] = p.adv[b * p.ldadv];
}

// What is summed: L, the KL term, bounds taken, ratios, tokens
constexpr int NSUM = 5;
struct Sums {
    double v[NSUM];
};
__device__ __forceinline__ Sums zero_sums() { return Sums{{0.0, 0.0, 0.0, 0.0, 0.0}}; }
// over groups of G lanes, in a fixed order
template <typename S>
__device__ __forceinline__ void lanes_sum(S& s, uint32_t G) {
    for (uint32_t d = G / 2; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < NSUM; ++i) s.v[i] += __shfl_xor(s.v[i], (int)d);
}

// A wave's sums over the tokens t0 .. t1 - 1 of sequence b
__device__ __forceinline__ Sums unit_sums(const vkb_policy& p, int64_t b, int64_t t0, int64_t t1, int lane) {
    Sums s = zero_sums();
    const bool by_kl = p.ref && p.kl != 0.0f;    // (0 * inf adds nothing)
    for (int64_t t = t0 + 4 * lane; t < t1; t += 256) {
        const uint32_t in = counted(p, b, t);
        if (!in) continue;
        Four f;
        load4(p, b, t, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!(in >> e & 1)) continue;
            const Token k = token(p, f.logp[e], f.old[e], f.ref[e], f.adv[e]);
            const float kl = p.ref ? kl_term(k.d) : 0.0f;
            const float taken = k.side ? (k.side > 0 ? p.r_high : p.r_low) : k.r;
            s.v[0] += (double)(by_kl ? p.kl * kl : 0.0f) - (double)taken * (double)k.adv;
            s.v[1] += (double)kl;
            s.v[2] += k.side ? 1.0 : 0.0;
            s.v[3] += (double)k.r;
            s.v[4] += 1.0;
        }
    }
    lanes_sum(s, 64);
    return s;
}

// The workgroup's 1024 threads over the units' sums: each sequence's by a group
// of G threads, then all sequences' by the reduction's weights.
constexpr uint32_t FIN = 1024;
template <typename GET>
__device__ __forceinline__ void finish(uint32_t B, uint32_t units, int reduce, GET get, float* stats, float* norm,
                                       double (*sh)[NSUM + 1]) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t G = 1;
    while (G < 64 && G < units) G *= 2;
    const uint32_t at = threadIdx.x / G, in = threadIdx.x % G;
    Sums total = zero_sums();
    double some = 0.0;                        // sequences with tokens
    auto sequence = [&](uint64_t b) {
        Sums s = zero_sums();
        if (b < B)
#pragma unroll 4
            for (uint32_t u = in; u < units; u += G) {
                const Sums x = get(b * units + u);
#pragma unroll
                for (int i = 0; i < NSUM; ++i) s.v[i] += x.v[i];
            }
        lanes_sum(s, G);
        return s;
    };
    for (uint64_t first = 0; first < B; first += FIN / G) {
        const Sums s = sequence(first + at);
        if (in || s.v[4] == 0.0) continue;
        const double by = reduce == VKBLAS_REDUCE_SEQUENCES ? 1.0 / s.v[4] : 1.0;
#pragma unroll
        for (int i = 0; i < NSUM; ++i) total.v[i] += s.v[i] * by;
        some += 1.0;
    }
    lanes_sum(total, 64);
#pragma unroll
    for (int d = 32; d; d >>= 1) some += __shfl_xor(some, d);
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < NSUM; ++i) sh[wave][i] = total.v[i];
        sh[wave][NSUM] = some;
    }
    __syncthreads();
    total = zero_sums();
    some = 0.0;
    for (uint32_t w = 0; w < FIN / 64; ++w) {
#pragma unroll
        for (int i = 0; i < NSUM; ++i) total.v[i] += sh[w][i];
        some += sh[w][NSUM];
    }
    const double weight = some == 0.0 ? 0.0 : reduce == VKBLAS_REDUCE_SUM ? 1.0
                        : reduce == VKBLAS_REDUCE_TOKENS ? 1.0 / total.v[4] : 1.0 / some;
    if (threadIdx.x < 4) stats[threadIdx.x] = (float)(total.v[threadIdx.x] * weight);
    for (uint64_t first = 0; first < B; first += FIN / G) {
        double n = 0.0;
        if (first + at < B)
            for (uint32_t u = in; u < units; u += G) n += get((first + at) * units + u).v[4];
        for (uint32_t d = G / 2; d; d >>= 1) n += __shfl_xor(n, (int)d);
        if (in == 0 && first + at < B)
            norm[first + at] = (float)(n == 0.0 ? 0.0 : reduce == VKBLAS_REDUCE_SEQUENCES ? weight / n : weight);
    }
}

__global__ __launch_bounds__(WORK) void unit_kernel(vkb_policy p, Sums* part) {
    const uint64_t unit = (uint64_t)blockIdx.x * (WORK / 64) + (threadIdx.x >> 6);
    if (unit >= (uint64_t)p.B * p.units) return;
    const int64_t b = (int64_t)(unit / p.units), t0 = (int64_t)(unit % p.units) * p.unit;
    const Sums s = unit_sums(p, b, t0, min(t0 + p.unit, (int64_t)p.T), threadIdx.x & 63);
    if ((threadIdx.x & 63) == 0) part[unit] = s;
}
__global__ __launch_bounds__(FIN) void finish_kernel(vkb_policy p, int reduce, const Sums* part, float* stats,
                                                     float* norm) {
    __shared__ double sh[FIN / 64][NSUM + 1];
    finish(p.B, p.units, reduce, [&](uint64_t u) { return part[u]; }, stats, norm, sh);
}
// A small call: the units' sums in LDS
constexpr uint32_t SMALL = VKBLAS_POLICY_SMALL / 256;
__global__ __launch_bounds__(FIN) void small_kernel(vkb_policy p, int reduce, float* stats, float* norm) {
    __shared__ double sh[FIN / 64][NSUM + 1];
    __shared__ Sums part[SMALL];
    const uint32_t n = p.B * p.units;
    for (uint32_t unit = threadIdx.x >> 6; unit < n; unit += FIN / 64) {
        const int64_t t0 = (int64_t)(unit % p.units) * p.unit;
        const Sums s = unit_sums(p, unit / p.units, t0, min(t0 + p.unit, (int64_t)p.T), threadIdx.x & 63);
        if ((threadIdx.x & 63) == 0) part[unit] = s;
    }
    __syncthreads();
    finish(p.B, p.units, reduce, [&](uint64_t u) { return part[u]; }, stats, norm, sh);
}

__global__ __launch_bounds__(WORK) void grad_kernel(vkb_policy p, const float* norm, const float* dloss, float* dlogp,
                                                    int64_t lddp) {
    const float dl = dloss[0];
    const bool by_kl = p.ref && p.kl != 0.0f;
    for_chunks(p.B, (p.T + 3) / 4, 0, gridDim.x, [&](uint64_t b, uint32_t k) {
        const int64_t t = (int64_t)k * 4;
        const uint32_t in = counted(p, b, t);
        float g[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (in) {
            Four f;
            load4(p, b, t, f);
            const float by = dl * norm[b];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const Token x = token(p, f.logp[e], f.old[e], f.ref[e], f.adv[e]);
                float s = x.side ? 0.0f : -x.adv * x.r;
                if (by_kl) s += p.kl * kl_slope(x.d);
                g[e] = in >> e & 1 ? by * s : 0.0f;
            }
        }
        st_chunk(dlogp + (int64_t)b * lddp, t, p.T, pack<float>(g));
    });
}

}  // namespace
}  // namespace vkb

using namespace vkb;

// Units of 256 tokens (a wave's four a lane) or as many as leave 16 waves a CU
extern "C" void vkb_policy_units(vkb_policy* p) {
    uint64_t n = ((uint64_t)p->B * p->T + 4095) / 4096;
    n = (n + 255) / 256 * 256;
    if (n > p->T) n = p->T;
    p->unit = (uint32_t)((n + 255) / 256 * 256);
    p->units = (uint32_t)(((uint64_t)p->T + p->unit - 1) / p->unit);
}
static bool small(const vkb_policy* p) { return (uint64_t)p->B * (((uint64_t)p->T + 255) / 256) <= SMALL; }
extern "C" size_t vkb_policy_part_bytes(const vkb_policy* p) {
    return small(p) ? 0 : (size_t)p->B * p->units * sizeof(Sums);
}

extern "C" int vkb_launch_policy(const vkb_policy* p, int reduce, void* part, float* stats, float* norm, void* stream) {
    if (!part) {
        if (!small(p)) return (int)hipErrorInvalidValue;
        hipLaunchKernelGGL(small_kernel, dim3(1), dim3(FIN), 0, (hipStream_t)stream, *p, reduce, stats, norm);
        return (int)hipGetLastError();
    }
    const uint64_t blocks = ((uint64_t)p->B * p->units + WORK / 64 - 1) / (WORK / 64);
    if (blocks > 0xffffffffull / WORK) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(unit_kernel, dim3((uint32_t)blocks), dim3(WORK), 0, (hipStream_t)stream, *p, (Sums*)part);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(FIN), 0, (hipStream_t)stream, *p, reduce, (const Sums*)part, stats,
                       norm);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_policy_grad(const vkb_policy* p, const float* norm, const float* dloss, float* dlogp,
                                      int64_t lddp, void* stream) {
    hipLaunchKernelGGL(grad_kernel, dim3(chunk_blocks(p->B, (p->T + 3) / 4)), dim3(WORK), 0, (hipStream_t)stream, *p,
                       norm, dloss, dlogp, lddp);
    return (int)hipGetLastError();
}
