// nn_common.hpp — what the kernels of vkblas_nn.h share: 16-byte accesses of
// any element alignment, reductions over a wave, the activations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gemm_mfma.hpp"
#include "vkb_launch.h"
#include "vkb_nn_launch.h"
#include "vkblas_nn.h"

namespace vkb {

// VEC = 16 / sizeof(T) values of a row from n on, of which only those below N
// exist; the others read as zero.  The address has its element's alignment.
template <typename T>
__device__ __forceinline__ u32x4 ld_chunk(const T* row, int64_t n, int64_t N) {
    constexpr int VEC = Elem<T>::VEC;
    if (n + VEC <= N) return ld16_any(row + n);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n < N) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (n + i >= N) break;
            if constexpr (sizeof(T) == 4) v[i] = *(const uint32_t*)(row + n + i);
            else v[i / 2] |= (uint32_t)*(const uint16_t*)(row + n + i) << (16 * (i & 1));
        }
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void unpack(u32x4 v, float* x) {
    constexpr int VEC = Elem<T>::VEC;
    typedef T tvec __attribute__((ext_vector_type(VEC)));
    const tvec t = __builtin_bit_cast(tvec, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = (float)t[i];
}

template <typename T>
__device__ __forceinline__ u32x4 pack(const float* x) {
    constexpr int VEC = Elem<T>::VEC;
    typedef T tvec __attribute__((ext_vector_type(VEC)));
    tvec t;
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (T)x[i];
    return __builtin_bit_cast(u32x4, t);
}

template <typename T>
__device__ __forceinline__ void st_chunk(T* row, int64_t n, int64_t N, u32x4 v) {
    constexpr int VEC = Elem<T>::VEC;
    if (n + VEC <= N) {
        *(u32x4_any*)(row + n) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if (n + i >= N) break;
        if constexpr (sizeof(T) == 4) *(uint32_t*)(row + n + i) = v[i];
        else *(uint16_t*)(row + n + i) = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
    }
}

// Reductions over a wave in a fixed order, the result in every lane: four
// shifts within each row of 16 lanes, the last lanes of rows 0 and 2 to rows 1
// and 3, then that of row 1 to rows 2 and 3.  As DPP operands of the additions
// (about 8 instructions; through LDS permutes they were a third of a layer
// norm row's instructions).
template <int CTRL, int ROWS, typename F>
__device__ __forceinline__ float dpp_step(float v, float none, F f) {
    const int o = __builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xf, false);
    return f(v, __int_as_float(o));
}
template <typename F>
__device__ __forceinline__ float wave_reduce(float v, float none, F f) {
    v = dpp_step<0x111, 0xf>(v, none, f);
    v = dpp_step<0x112, 0xf>(v, none, f);
    v = dpp_step<0x114, 0xf>(v, none, f);
    v = dpp_step<0x118, 0xf>(v, none, f);
    v = dpp_step<0x142, 0xa>(v, none, f);
    v = dpp_step<0x143, 0xc>(v, none, f);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, 0.0f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

// The factor of a cross entropy's D, and where it and its inverse go
// (vkb_launch_pad in vkb_nn_launch.h; to: fp16's 2^13).
struct Scale {
    float* scal;
    float beta, to;
    int find;
};
template <typename T>
static inline Scale with_to(vkb_scale s) {
    return Scale{s.scal, s.beta, sizeof(T) == 2 && !is_bf16<T> ? 8192.0f : 1.0f, s.find};
}
// By the largest itself, not a power of two near it: equal loss gradients (a
// mean's) then round the target's p - 1 near -1 almost exactly, where any other
// factor puts one and the same error on every row.
// Held where it and its inverse are normal fp32 numbers (of 2^-13 the smallest,
// 1e-33, of 1 the largest, 8e37); what lies past that still fits the type.
__device__ __forceinline__ float scale_top(float top) { return fminf(fmaxf(top, 1e-33f), 8e37f); }
__device__ __forceinline__ float scale_by(const Scale& s, float top) { return s.to / scale_top(top); }
__device__ __forceinline__ void set_scale(const Scale& s, float top) {
    s.scal[0] = scale_by(s, top);
    s.scal[1] = scale_top(top) / s.to;
    s.scal[2] = s.beta;
    s.scal[3] = 1.0f;
    s.scal[4] = 0.0f;
}
// What a row adds to the search for the largest: |dloss| where it counts and is
// finite, else 0.
__device__ __forceinline__ float scale_row(const float* dloss, const int64_t* target, uint32_t m, int64_t V,
                                           int64_t ignore) {
    const float d = fabsf(dloss[m]);
    const int64_t t = target[m];
    return t != ignore && t >= 0 && t < V && d < INFINITY ? d : 0.0f;
}
// The factor in every lane: read, or found by this wave over all M rows (the
// wave with `write` leaves it for the products that follow).  fp32: none.
template <typename T>
__device__ __forceinline__ float scale_of(const Scale& s, const float* dloss, const int64_t* target, uint32_t M,
                                          int64_t V, int64_t ignore, bool write, int lane) {
    if (sizeof(T) == 4 || !s.scal) return 1.0f;
    if (!s.find) return s.scal[0];
    float top = 0.0f;
    for (uint32_t m = 0; m < M; m += 256) {
        float v[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = scale_row(dloss, target, min(m + 64 * i + lane, M - 1), V, ignore);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, v[i]);
    }
    top = wave_max(top);
    if (write && lane == 0) set_scale(s, top);
    return scale_by(s, top);
}

constexpr float LOG2E = 1.4426950408889634f;

// exp(x) by the hardware's 2^x: relative error about |x| 2^-24 from rounding
// x log2(e), plus one unit of the result
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-x)); }

constexpr float GELU_C = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float GELU_A = 0.044715f;

template <int ACT>
__device__ __forceinline__ float act(float g) {
    if constexpr (ACT == VKBLAS_ACT_SILU) return g * sigmoid(g);
    // (1 + tanh y) / 2 = 1 / (1 + exp(-2 y))
    if constexpr (ACT == VKBLAS_ACT_GELU_TANH) return g * sigmoid(2.0f * GELU_C * (g + GELU_A * g * g * g));
    if constexpr (ACT == VKBLAS_ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.7071067811865476f));
    return g > 0.0f ? g : (g != g ? g : 0.0f);   // max(g, 0), a NaN stays
}

// act(g) and its derivative
template <int ACT>
__device__ __forceinline__ void act_and_slope(float g, float& a, float& da) {
    if constexpr (ACT == VKBLAS_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        da = s + a * (1.0f - s);
    } else if constexpr (ACT == VKBLAS_ACT_GELU_TANH) {
        const float s = sigmoid(2.0f * GELU_C * (g + GELU_A * g * g * g));
        a = g * s;
        da = s + a * (1.0f - s) * (2.0f * GELU_C * (1.0f + 3.0f * GELU_A * g * g));
    } else if constexpr (ACT == VKBLAS_ACT_GELU) {
        const float p = 0.5f * (1.0f + erff(g * 0.7071067811865476f));
        a = g * p;
        da = p + g * (0.3989422804014327f * fast_exp(-0.5f * g * g));
    } else {
        a = act<ACT>(g);
        da = g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
    }
}

// f(row, 16-byte chunk of the row) for rows of `chunks` chunks each, over the
// workgroups first .. first + blocks - 1 of WORK threads
constexpr uint32_t WORK = 256;
template <typename F>
__device__ __forceinline__ void for_chunks(uint64_t rows, uint32_t chunks, uint32_t first, uint32_t blocks, F f) {
    const uint64_t total = rows * chunks;
    const uint32_t step = blocks * WORK, start = (blockIdx.x - first) * WORK + threadIdx.x;
    if (total + step <= 0xffffffffull) {
        for (uint32_t i = start; i < (uint32_t)total; i += step) {
            const uint32_t r = i / chunks;
            f((uint64_t)r, i - r * chunks);
        }
    } else {
        for (uint64_t i = start; i < total; i += step) {
            const uint64_t r = i / chunks;
            f(r, (uint32_t)(i - r * chunks));
        }
    }
}
// ... its workgroups: one chunk a thread, up to 32 per CU of 256
static inline uint32_t chunk_blocks(uint64_t rows, uint32_t chunks) {
    const uint64_t b = (rows * chunks + WORK - 1) / WORK;
    return (uint32_t)(b < 8192 ? b : 8192);
}
template <typename T>
static inline uint32_t chunks_of(uint32_t N) { return (N + Elem<T>::VEC - 1) / Elem<T>::VEC; }

// f(integral_constant<int, ACT>) for the activation's code; false: unknown
template <typename F>
static inline bool with_act(int code, F f) {
    switch (code) {
        case VKBLAS_ACT_SILU: f(std::integral_constant<int, VKBLAS_ACT_SILU>{}); return true;
        case VKBLAS_ACT_GELU: f(std::integral_constant<int, VKBLAS_ACT_GELU>{}); return true;
        case VKBLAS_ACT_GELU_TANH: f(std::integral_constant<int, VKBLAS_ACT_GELU_TANH>{}); return true;
        case VKBLAS_ACT_RELU: f(std::integral_constant<int, VKBLAS_ACT_RELU>{}); return true;
        default: return false;
    }
}

// f(T{}) for the element type's code; false: unknown
template <typename F>
static inline bool with_type(int code, F f) {
    switch (code) {
        case VKB_T_F32: f(float{}); return true;
        case VKB_T_F16: f((_Float16)0); return true;
        case VKB_T_BF16: f((__bf16)0.0f); return true;
        default: return false;
    }
}

}  // namespace vkb
