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
    float r, d;              // ratio, ref - logp
    int side;                // 0: r A is taken, -1: the lower bound's, 1: the upper one's
};
// A NaN anywhere takes r A, which it reaches.
__device__ __forceinline__ Token token(const vkb_policy& p, float logp, float old, float ref, float adv) {
    const double diff = (double)logp - (double)old;
    Token t;
    t.r = fast_exp(logp - old);
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
// WHOLE: all four are of the sequence
template <bool WHOLE>
__device__ __forceinline__ void load4(const vkb_policy& p, int64_t b, int64_t t, Four& f) {
    auto get = [&](const float* row, float* x) {
        unpack<float>(WHOLE ? ld16_any(row + t) : ld_chunk(row, t, p.T), x);
    };
    get(p.logp + b * p.ldp, f.logp);
    get(p.old + b * p.ldo, f.old);
    if (p.ref) get(p.ref + b * p.ldr, f.ref);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) f.ref[e] = f.logp[e];
    if (p.adv_step) get(p.adv + b * p.ldadv, f.adv);
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

// A wave's sum in a fixed order, in every lane: the steps of wave_reduce, on
// both halves of a double
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    v = dpp_add<0x143, 0xc>(v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A wave's sums over the tokens of sequence b from t0 + 4 lane on, four every
// `step`, below t1; the masks of AHEAD rounds are read before their arrays.
// Tokens that do not count become ones whose terms are 0.  Four tokens are added
// in fp32, as good as the terms themselves, and their sum in fp64.
constexpr int AHEAD = 2;
__device__ __forceinline__ Sums token_sums(const vkb_policy& p, int64_t b, int64_t t0, int64_t t1, int64_t step, int lane) {
    Sums s = zero_sums();
    uint32_t tokens = 0, sides = 0;
    const bool by_kl = p.ref && p.kl != 0.0f;    // (0 * inf adds nothing)
    auto add = [&](uint32_t in, const Four& f) {
        float loss = 0.0f, kls = 0.0f, rs = 0.0f;
        tokens += __popc(in);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool is = in >> e & 1;
            const float adv = is ? f.adv[e] : 0.0f;
            const Token k = token(p, is ? f.logp[e] : 0.0f, is ? f.old[e] : 0.0f, is ? f.ref[e] : 0.0f, adv);
            const float kl = p.ref ? kl_term(k.d) : 0.0f;
            const float taken = k.side ? (k.side > 0 ? p.r_high : p.r_low) : k.r;
            loss += (by_kl ? p.kl * kl : 0.0f) - taken * adv;
            kls += kl;
            sides += k.side ? 1u : 0u;
            rs += is ? k.r : 0.0f;
        }
        s.v[0] += (double)loss;
        s.v[1] += (double)kls;
        s.v[3] += (double)rs;
    };
    auto rounds = [&](auto whole, int64_t t) {
        uint32_t in[AHEAD];
        Four f[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) in[i] = t + step * i < t1 ? counted(p, b, t + step * i) : 0;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (in[i]) load4<decltype(whole)::value>(p, b, t + step * i, f[i]);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (in[i]) add(in[i], f[i]);
    };
    for (int64_t t = t0; t < t1; t += step * AHEAD)
        if (t + step * (AHEAD - 1) + 256 <= t1) rounds(std::true_type{}, t + 4 * lane);
        else rounds(std::false_type{}, t + 4 * lane);
    s.v[2] = (double)sides;
    s.v[4] = (double)tokens;
#pragma unroll
    for (int i = 0; i < NSUM; ++i) s.v[i] = wave_sum(s.v[i]);
    return s;
}

// The workgroup over the units' sums (part: NSUM arrays of `count`): each
// sequence's by a group of lanes, as many as B leaves of the threads, then all
// sequences' by the reduction's weights.
constexpr uint32_t FIN = 1024;
struct Shared {
    double waves[NSUM + 1][FIN / 64], tokens[FIN];       // tokens: of the first FIN sequences
};
__device__ __forceinline__ void finish(uint32_t B, uint32_t units, int reduce, const double* part, uint64_t count,
                                       float* stats, float* norm, Shared& sh) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, threads = blockDim.x;
    uint32_t G = 1;
    while (G < 64 && G < units && 2 * G * B <= threads) G *= 2;
    const uint32_t at = threadIdx.x / G, in = threadIdx.x % G;
    double total[NSUM + 1] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};             // the last: sequences with tokens
    for (uint64_t b = at; b < B; b += threads / G) {
        double s[NSUM] = {0.0, 0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
        for (uint32_t u = in; u < units; u += G)
#pragma unroll
            for (int i = 0; i < NSUM; ++i) s[i] += part[i * count + b * units + u];
        for (uint32_t d = G / 2; d; d >>= 1)
#pragma unroll
            for (int i = 0; i < NSUM; ++i) s[i] += __shfl_xor(s[i], (int)d);
        if (in == 0 && b < FIN) sh.tokens[b] = s[4];
        if (in || s[4] == 0.0) continue;
        const double by = reduce == VKBLAS_REDUCE_SEQUENCES ? 1.0 / s[4] : 1.0;
#pragma unroll
        for (int i = 0; i < NSUM; ++i) total[i] += s[i] * by;
        total[NSUM] += 1.0;
    }
#pragma unroll
    for (int i = 0; i <= NSUM; ++i) {
        total[i] = wave_sum(total[i]);
        if (lane == 0) sh.waves[i][wave] = total[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i <= NSUM; ++i) total[i] = wave_sum(lane < threads / 64 ? sh.waves[i][lane] : 0.0);
    const double some = total[NSUM];
    const double weight = some == 0.0 ? 0.0 : reduce == VKBLAS_REDUCE_SUM ? 1.0
                        : reduce == VKBLAS_REDUCE_TOKENS ? 1.0 / total[4] : 1.0 / some;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (threadIdx.x == (uint32_t)i) stats[i] = (float)(total[i] * weight);
    for (uint64_t b = threadIdx.x; b < B; b += threads) {
        double n = 0.0;
        if (b < FIN) n = sh.tokens[b];
        else
            for (uint32_t u = 0; u < units; ++u) n += part[4 * count + b * units + u];
        norm[b] = (float)(n == 0.0 ? 0.0 : reduce == VKBLAS_REDUCE_SEQUENCES ? weight / n : weight);
    }
}

// Units of a wave (sequences of up to 256 tokens) or of a workgroup's four
template <bool SHORT>
__global__ __launch_bounds__(WORK) void unit_kernel(vkb_policy p, double* part) {
    constexpr uint32_t WAVES = WORK / 64;
    __shared__ double sh[WAVES][NSUM];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t count = (uint64_t)p.B * p.units, step = (uint64_t)gridDim.x * (SHORT ? WAVES : 1);
    for (uint64_t unit = SHORT ? (uint64_t)blockIdx.x * WAVES + wave : blockIdx.x; unit < count; unit += step) {
        const int64_t b = (int64_t)(unit / p.units), t0 = (int64_t)(unit % p.units) * p.unit;
        const int64_t t1 = min(t0 + p.unit, (int64_t)p.T);
        Sums s = token_sums(p, b, SHORT ? t0 : t0 + 256 * wave, t1, SHORT ? 256 : 256 * WAVES, lane);
        if (!SHORT) {
            __syncthreads();                 // the unit before is read
#pragma unroll
            for (int i = 0; i < NSUM; ++i)
                if (lane == 0) sh[wave][i] = s.v[i];
            __syncthreads();
            if (wave) continue;
#pragma unroll
            for (int i = 0; i < NSUM; ++i)
                for (uint32_t w = 1; w < WAVES; ++w) s.v[i] += sh[w][i];
        }
#pragma unroll
        for (int i = 0; i < NSUM; ++i)
            if (lane == (uint32_t)i) part[i * count + unit] = s.v[i];
    }
}
__global__ __launch_bounds__(FIN) void finish_kernel(vkb_policy p, int reduce, const double* part, float* stats,
                                                     float* norm) {
    __shared__ Shared sh;
    finish(p.B, p.units, reduce, part, (uint64_t)p.B * p.units, stats, norm, sh);
}
// A small call: units of 256 tokens, their sums in LDS
constexpr uint32_t SMALL = VKBLAS_POLICY_SMALL / 256;
__global__ __launch_bounds__(FIN) void small_kernel(vkb_policy p, int reduce, float* stats, float* norm) {
    __shared__ Shared sh;
    __shared__ double part[NSUM * SMALL];
    const uint32_t units = (p.T + 255) / 256, n = p.B * units, unit = threadIdx.x >> 6;
    const int64_t t0 = (int64_t)(unit % units) * 256;
    const Sums s = token_sums(p, unit / units, t0, min(t0 + 256, (int64_t)p.T), 256, threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < NSUM; ++i)
        if ((threadIdx.x & 63) == i) part[i * n + unit] = s.v[i];
    __syncthreads();
    finish(p.B, units, reduce, part, n, stats, norm, sh);
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
            load4<false>(p, b, t, f);
            const float by = dl * norm[b];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const Token x = token(p, f.logp[e], f.old[e], f.ref[e], f.adv[e]);
                float s = x.side ? 0.0f : -f.adv[e] * x.r;
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

// A unit: a wave's 256 tokens, or 1024 times as many as leave 2048 workgroups
extern "C" void vkb_policy_units(vkb_policy* p) {
    if (p->T <= 256) {
        p->unit = 256;
        p->units = 1;
        return;
    }
    const uint64_t n = ((uint64_t)p->B * p->T + 2047) / 2048;
    const uint64_t unit = n < p->T ? (n + 1023) / 1024 * 1024 : ((uint64_t)p->T + 1023) / 1024 * 1024;
    p->unit = (uint32_t)unit;
    p->units = (uint32_t)(((uint64_t)p->T + unit - 1) / unit);
}
// One wave each for up to 16 units of 256
static uint64_t small_units(const vkb_policy* p) { return (uint64_t)p->B * (((uint64_t)p->T + 255) / 256); }
extern "C" size_t vkb_policy_part_bytes(const vkb_policy* p) {
    return small_units(p) <= SMALL ? 0 : (size_t)p->B * p->units * sizeof(Sums);   // as NSUM arrays
}

extern "C" int vkb_launch_policy(const vkb_policy* p, int reduce, void* part, float* stats, float* norm, void* stream) {
    if (!part) {
        static_assert(SMALL <= FIN / 64, "a wave for each unit");
        if (small_units(p) > SMALL) return (int)hipErrorInvalidValue;
        hipLaunchKernelGGL(small_kernel, dim3(1), dim3(64 * (uint32_t)small_units(p)), 0, (hipStream_t)stream, *p, reduce,
                           stats, norm);
        return (int)hipGetLastError();
    }
    const uint64_t count = (uint64_t)p->B * p->units, blocks = p->T <= 256 ? (count + WORK / 64 - 1) / (WORK / 64) : count;
    const dim3 grid((uint32_t)(blocks < 1u << 20 ? blocks : 1u << 20));
    if (p->T <= 256)
        hipLaunchKernelGGL((unit_kernel<true>), grid, dim3(WORK), 0, (hipStream_t)stream, *p, (double*)part);
    else
        hipLaunchKernelGGL((unit_kernel<false>), grid, dim3(WORK), 0, (hipStream_t)stream, *p, (double*)part);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(FIN), 0, (hipStream_t)stream, *p, reduce, (const double*)part, stats,
                       norm);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_policy_grad(const vkb_policy* p, const float* norm, const float* dloss, float* dlogp,
                                      int64_t lddp, void* stream) {
    hipLaunchKernelGGL(grad_kernel, dim3(chunk_blocks(p->B, (p->T + 3) / 4)), dim3(WORK), 0, (hipStream_t)stream, *p,
                       norm, dloss, dlogp, lddp);
    return (int)hipGetLastError();
}
