// policy.hip — clipped policy loss with a KL term on token log probabilities.
//
// A token's loss is a few operations on four or five floats, so the loss over a
// batch is a pass over its arrays and a sum, bound by the reads: 8 bytes a token,
// 1 with a mask, 4 each with a reference and with its own advantage.  A workgroup takes a unit, a sequence or a part of one (a wave where
// there are many short sequences), four tokens a lane at a time, and skips the
// arrays where no token of a lane's four counts: the padding behind a sequence
// costs its mask alone.  A token's terms and the sum of a lane's four are fp32, the
// sums of those fp64, and so is logp - old, on which the side of a bound depends: r >
// 1 + clip_high exactly where logp - old > log(1 + clip_high).
//
// 1024 sequences of 8192 tokens, half of them padding: 20.8 us (3.6 TB/s of the
// bytes that it reads) and 5.8 for the finish, one workgroup over 2048 units; the
// gradient, which writes the padding's zeros too, 20 us (5.4 TB/s).  A call of up to
// 16 units of 256 tokens is one workgroup, 7.2 us with its launch.
#include "nn_common.hpp"

namespace vkb {
namespace {

// exp(d) - d - 1 without the cancellation of a small d: d^2 sum d^k / (k + 2)!
// within |d| <= 1 (the terms left out are below 2^-30 of the sum)
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
// 1 - exp(d), likewise (below 2^-28)
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
    float by;                // what A is multiplied by where r A is taken
    int side;                // 0: r A is taken, -1: the lower bound's, 1: the upper one's
};
// A NaN anywhere takes r A, which it reaches.  r of finite numbers may be past fp32's
// range, and an advantage of 0 times it is 0 all the same: logp - old, which is finite
// where they are, stands in for it.
__device__ __forceinline__ Token token(const vkb_policy& p, float logp, float old, float ref, float adv) {
    const double diff = (double)logp - (double)old;
    Token t;
    t.r = fast_exp(logp - old);
    t.d = ref - logp;
    t.by = adv == 0.0f ? logp - old : t.r;
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

// A count's, likewise
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    v = dpp_add<0x143, 0xc>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// A lane's sums over the tokens of sequence b from t0 + 4 lane on, four every
// `step`, below t1; the masks of AHEAD rounds are read before their arrays.
// Tokens that do not count become ones whose terms are 0.  Four tokens are added
// in fp32, as good as the terms themselves, and their sum in fp64.
constexpr int AHEAD = 2;
__device__ __forceinline__ Sums lane_sums(const vkb_policy& p, int64_t b, int64_t t0, int64_t t1, int64_t step,
                                          int lane) {
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
            const float taken = k.side ? (k.side > 0 ? p.r_high : p.r_low) : k.by;
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
    return s;
}
// ... a wave's
__device__ __forceinline__ Sums token_sums(const vkb_policy& p, int64_t b, int64_t t0, int64_t t1, int64_t step,
                                           int lane) {
    Sums s = lane_sums(p, b, t0, t1, step, lane);
#pragma unroll
    for (int i = 0; i < NSUM; ++i) s.v[i] = wave_sum(s.v[i]);
    return s;
}

// What sequences sum to, by the reduction's weights, and those that have tokens
struct Total {
    double v[NSUM + 1];
};
__device__ __forceinline__ void add_sequence(Total& t, const double* s, int reduce) {
    if (s[4] == 0.0) return;
    const double by = reduce == VKBLAS_REDUCE_SEQUENCES ? 1.0 / s[4] : 1.0;
#pragma unroll
    for (int i = 0; i < NSUM; ++i) t.v[i] += s[i] * by;
    t.v[NSUM] += 1.0;
}
// The threads' totals joined: stats (write), and the batch's weight
constexpr uint32_t FIN = 1024;
__device__ __forceinline__ double settle(Total t, int reduce, bool write, float* stats, double (*sh)[FIN / 64]) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i <= NSUM; ++i) {
        t.v[i] = wave_sum(t.v[i]);
        if (lane == 0) sh[i][wave] = t.v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i <= NSUM; ++i) t.v[i] = wave_sum(lane < blockDim.x / 64 ? sh[i][lane] : 0.0);
    const double some = t.v[NSUM];
    const double weight = some == 0.0 ? 0.0 : reduce == VKBLAS_REDUCE_SUM ? 1.0
                        : reduce == VKBLAS_REDUCE_TOKENS ? 1.0 / t.v[4] : 1.0 / some;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (write && threadIdx.x == (uint32_t)i) stats[i] = (float)(t.v[i] * weight);
    return weight;
}
__device__ __forceinline__ float norm_of(double tokens, double weight, int reduce) {
    return (float)(tokens == 0.0 ? 0.0 : reduce == VKBLAS_REDUCE_SEQUENCES ? weight / tokens : weight);
}

// The workgroup over the units' sums (part: NSUM arrays of `count`): each
// sequence's by a group of lanes, as many as B leaves of the threads.
struct Shared {
    double waves[NSUM + 1][FIN / 64], tokens[FIN];       // tokens: of the first FIN sequences
};
__device__ __forceinline__ void finish(uint32_t B, uint32_t units, int reduce, const double* part, uint64_t count,
                                       float* stats, float* norm, Shared& sh) {
    const uint32_t threads = blockDim.x;
    uint32_t G = 1;
    while (G < 64 && G < units && 2 * G * B <= threads) G *= 2;
    const uint32_t at = threadIdx.x / G, in = threadIdx.x % G;
    Total total = {};
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
        if (in == 0) add_sequence(total, s, reduce);
    }
    const double weight = settle(total, reduce, true, stats, sh.waves);
    for (uint64_t b = threadIdx.x; b < B; b += threads) {
        double n = 0.0;
        if (b < FIN) n = sh.tokens[b];
        else
            for (uint32_t u = 0; u < units; ++u) n += part[4 * count + b * units + u];
        norm[b] = norm_of(n, weight, reduce);
    }
}

// Sequences of several units, one a workgroup
constexpr uint32_t WAVES = WORK / 64;
__global__ __launch_bounds__(WORK) void unit_kernel(vkb_policy p, double* part) {
    __shared__ double sh[WAVES][NSUM];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t count = (uint64_t)p.B * p.units;
    for (uint64_t unit = blockIdx.x; unit < count; unit += gridDim.x) {
        const int64_t b = (int64_t)(unit / p.units), t0 = (int64_t)(unit % p.units) * p.unit;
        Sums s = token_sums(p, b, t0 + 256 * wave, min(t0 + p.unit, (int64_t)p.T), 256 * WAVES, lane);
        __syncthreads();                     // the unit before is read
#pragma unroll
        for (int i = 0; i < NSUM; ++i)
            if (lane == 0) sh[wave][i] = s.v[i];
        __syncthreads();
        if (wave) continue;
#pragma unroll
        for (int i = 0; i < NSUM; ++i)
            for (uint32_t w = 1; w < WAVES; ++w) s.v[i] += sh[w][i];
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

// Sequences of one unit: a wave's (WAVE) or a workgroup's
// own.  Their tokens are counted, and each lane adds its sums by the
// reduction's weight: lanes and waves are joined once for all of a workgroup's
// sequences, and the finish reads as many totals as there are workgroups
// (part: NSUM + 1 arrays of those, then each sequence's tokens).  Against each
// sequence's five sums to memory and one workgroup over them (us): 65536 x 128
// 115 -> 53, 16384 x 1024 71 -> 49, 8192 x 256 22 -> 16.  What is left at many short
// sequences is arithmetic, a wave's whatever its lanes hold.
template <bool WAVE>
__global__ __launch_bounds__(WORK) void whole_kernel(vkb_policy p, int reduce, double* part) {
    __shared__ double totals[WAVES][NSUM + 1];
    __shared__ uint32_t counts[2][WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double* tokens = part + (NSUM + 1) * (uint64_t)gridDim.x;
    Total total = {};
    uint32_t turn = 0;
    for (uint64_t b = WAVE ? (uint64_t)blockIdx.x * WAVES + wave : blockIdx.x; b < p.B;
         b += (uint64_t)gridDim.x * (WAVE ? WAVES : 1)) {
        const Sums s = lane_sums(p, (int64_t)b, WAVE ? 0 : 256 * wave, p.T, WAVE ? 256 : 256 * WAVES, lane);
        uint32_t n = wave_sum((uint32_t)s.v[4]);
        if (!WAVE) {
            if (lane == 0) counts[turn][wave] = n;
            __syncthreads();             // (one a sequence: the next one's counts go to the other half)
            n = 0;
            for (uint32_t w = 0; w < WAVES; ++w) n += counts[turn][w];
            turn ^= 1;
        }
        const bool first = lane == 0 && (WAVE || wave == 0);
        if (first) tokens[b] = (double)n;
        if (n == 0) continue;
        const double by = reduce == VKBLAS_REDUCE_SEQUENCES ? 1.0 / (double)n : 1.0;
#pragma unroll
        for (int i = 0; i < NSUM; ++i) total.v[i] += s.v[i] * by;
        total.v[NSUM] += first ? 1.0 : 0.0;
    }
#pragma unroll
    for (int i = 0; i <= NSUM; ++i) {
        total.v[i] = wave_sum(total.v[i]);
        if (lane == 0) totals[wave][i] = total.v[i];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i <= NSUM; ++i) {
        for (uint32_t w = 1; w < WAVES; ++w) total.v[i] += totals[w][i];
        if (lane == (uint32_t)i) part[i * (uint64_t)gridDim.x + blockIdx.x] = total.v[i];
    }
}
// Every workgroup adds the `count` totals, and writes its part of norm
__global__ __launch_bounds__(FIN) void whole_finish_kernel(uint32_t B, int reduce, const double* part, uint32_t count,
                                                           float* stats, float* norm) {
    __shared__ double sh[NSUM + 1][FIN / 64];
    Total total = {};
#pragma unroll 2
    for (uint32_t j = threadIdx.x; j < count; j += FIN)
#pragma unroll
        for (int i = 0; i <= NSUM; ++i) total.v[i] += part[(uint64_t)i * count + j];
    const double weight = settle(total, reduce, blockIdx.x == 0, stats, sh);
    const double* tokens = part + (NSUM + 1) * (uint64_t)count;
    for (uint64_t b = (uint64_t)blockIdx.x * FIN + threadIdx.x; b < B; b += (uint64_t)gridDim.x * FIN)
        norm[b] = norm_of(tokens[b], weight, reduce);
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

// Four tokens a thread; dlogp is written whole, so the floor counts 4 bytes a
// token more
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
                float s = x.side ? 0.0f : -f.adv[e] * x.by;
                if (by_kl) s += p.kl * kl_slope(x.d);
                // 0 times a slope past fp32's range is 0: its arguments, finite where the inputs are, stand in
                if (by == 0.0f && !__builtin_isfinite(s))
                    s = (x.side ? 0.0f : f.adv[e] + (f.logp[e] - f.old[e])) + (by_kl ? x.d : 0.0f);
                g[e] = in >> e & 1 ? by * s : 0.0f;
            }
        }
        st_chunk(dlogp + (int64_t)b * lddp, t, p.T, pack<float>(g));
    });
}

}  // namespace
}  // namespace vkb

using namespace vkb;

// A unit: sequences of up to 256 tokens, or 1024 tokens times as many as leave 2048
// workgroups
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
// Whether sequences of one unit are a wave's: up to 256 tokens leave a workgroup's
// others nothing, and up to 1024 are so where there are waves enough (us, a
// workgroup / a wave each: 1024 x 1000 12.0 / 14.3, 2048 x 512 15.2 / 11.7, 2048 x 1024
// 16.4 / 15.3, 16384 x 300 48 / 25, 16384 x 1024 61 / 49; 4096 x 4096 47 / 49).
static bool by_wave(const vkb_policy* p) { return p->T <= 256 || (p->T <= 1024 && p->B >= 2048); }
// Workgroups of sequences of one unit (us for 512 / 1024 / 2048 / 4096 of them:
// 65536 x 128 81 / 52 / 52 / 53, 4096 x 4096 73 / 49 / 48 / 47)
constexpr uint32_t WHOLE_BLOCKS = 2048;
static uint32_t whole_blocks(const vkb_policy* p) {
    const uint32_t n = by_wave(p) ? (p->B + WAVES - 1) / WAVES : p->B;
    return n < WHOLE_BLOCKS ? n : WHOLE_BLOCKS;
}
extern "C" size_t vkb_policy_part_bytes(const vkb_policy* p) {
    if (small_units(p) <= SMALL) return 0;
    if (p->units == 1) return ((size_t)whole_blocks(p) * (NSUM + 1) + p->B) * sizeof(double);
    return (size_t)p->B * p->units * sizeof(Sums);   // as NSUM arrays
}

extern "C" int vkb_launch_policy(const vkb_policy* p, int reduce, void* part, float* stats, float* norm, void* stream) {
    if (!part) {
        static_assert(SMALL <= FIN / 64, "a wave for each unit");
        if (small_units(p) > SMALL) return (int)hipErrorInvalidValue;
        hipLaunchKernelGGL(small_kernel, dim3(1), dim3(64 * (uint32_t)small_units(p)), 0, (hipStream_t)stream, *p,
                           reduce, stats, norm);
        return (int)hipGetLastError();
    }
    const bool whole = p->units == 1;
    const uint32_t blocks = whole_blocks(p);
    const uint64_t count = (uint64_t)p->B * p->units;
    if (whole && by_wave(p))
        hipLaunchKernelGGL((whole_kernel<true>), dim3(blocks), dim3(WORK), 0, (hipStream_t)stream, *p, reduce,
                           (double*)part);
    else if (whole)
        hipLaunchKernelGGL((whole_kernel<false>), dim3(blocks), dim3(WORK), 0, (hipStream_t)stream, *p, reduce,
                           (double*)part);
    else
        hipLaunchKernelGGL(unit_kernel, dim3((uint32_t)(count < 1u << 20 ? count : 1u << 20)), dim3(WORK), 0,
                           (hipStream_t)stream, *p, (double*)part);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    const uint32_t n = (uint32_t)(((uint64_t)p->B + FIN - 1) / FIN);
    if (whole)
        hipLaunchKernelGGL(whole_finish_kernel, dim3(n < 64 ? n : 64), dim3(FIN), 0, (hipStream_t)stream, p->B, reduce,
                           (const double*)part, blocks, stats, norm);
    else
        hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(FIN), 0, (hipStream_t)stream, *p, reduce, (const double*)part,
                           stats, norm);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_policy_grad(const vkb_policy* p, const float* norm, const float* dloss, float* dlogp,
                                      int64_t lddp, void* stream) {
    hipLaunchKernelGGL(grad_kernel, dim3(chunk_blocks(p->B, (p->T + 3) / 4)), dim3(WORK), 0, (hipStream_t)stream, *p,
                       norm, dloss, dlogp, lddp);
    return (int)hipGetLastError();
}
