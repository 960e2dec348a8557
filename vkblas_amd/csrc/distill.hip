// distill.hip — distillation from a teacher's top logits, beside the linear
// cross entropy's kernels (xent.hip, gemm_ops.hpp): what of it goes by rows and
// their entries.
//
// With q the teacher's softmax over a row's few entries, p the student's over
// all V classes and T the temperature,
//   loss = T^2 sum_j q_j (log q_j - z_j / T + lse),
//   D_v  = T dloss (p_v - q_v),
// so over the vocabulary both need what a cross entropy needs, log-sum-exp and
// p, and the entries come on top: their logits z_j are dot products of x's row
// with the entries' rows of w, and D's elements at the entries are written over
// by a patch once the tiles are stored.  T's factor in D is taken into dloss.
#include "nn_common.hpp"

namespace vkb {
namespace {

constexpr uint32_t TOP = VKBLAS_DISTILL_TOP, WAVES = WORK / 64;

constexpr int ABSENT = -1, BAD = -2;
struct Shared {
    float q[TOP];            // the teacher's logits, then over T, then its probabilities
    int id[TOP];             // class, or ABSENT, or BAD
    float high[WAVES], sum[WAVES];
    uint32_t flags[WAVES];
};

// A row's entries into LDS: classes, and t / T less the largest (the difference
// first: t of the type's lowest value over a T below 1 is no -inf).  Returns the
// log of their sum of exponentials.  counted: some entry is there and not of
// probability 0 (a NaN is not); bad: some class is past V.
template <typename TT>
__device__ __forceinline__ float teacher(uint32_t n, uint32_t V, const int64_t* top, const TT* t, float inv_t,
                                         Shared& sh, bool& counted, bool& bad) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float high = -INFINITY;
    bool any = false, past = false;
    for (uint32_t j = threadIdx.x; j < n; j += WORK) {
        const int64_t c = top[j];
        const float v = c < 0 ? -INFINITY : (float)t[j];
        sh.id[j] = c < 0 ? ABSENT : c < V ? (int)c : BAD;
        sh.q[j] = v;
        any |= !(v == -INFINITY);
        past |= c >= (int64_t)V;
        high = fmaxf(high, v);
    }
    high = wave_max(high);
    const uint32_t f = (__any(any) ? 1u : 0u) | (__any(past) ? 2u : 0u);
    if (lane == 0) {
        sh.high[wave] = high;
        sh.flags[wave] = f;
    }
    __syncthreads();
    uint32_t flags = 0;
    for (uint32_t w = 0; w < WAVES; ++w) {
        high = fmaxf(high, sh.high[w]);
        flags |= sh.flags[w];
    }
    counted = flags & 1;
    bad = flags & 2;
    if (high == -INFINITY) high = 0.0f;
    float s = 0.0f;
    for (uint32_t j = threadIdx.x; j < n; j += WORK) {
        sh.q[j] = (sh.q[j] - high) * inv_t;
        s += fast_exp(sh.q[j]);
    }
    s = wave_sum(s);
    if (lane == 0) sh.sum[wave] = s;
    __syncthreads();
    s = 0.0f;
    for (uint32_t w = 0; w < WAVES; ++w) s += sh.sum[w];
    return logf(s);
}

// A row's pair (top, s) as xent.hip's, of logits times inv_t = c2 / log2(e); the
// threads' join: its log-sum-exp, in every thread
struct Pair {
    float top = -INFINITY, s = 0.0f;
};
__device__ __forceinline__ float finite_or_0(float x) { return __builtin_isinf(x) ? 0.0f : x; }
__device__ __forceinline__ float block_lse(Pair p, float inv_t, float2* sh) {
    const float c2 = inv_t * LOG2E;
    float top = wave_max(p.top), off = finite_or_0(top);
    float s = wave_sum(p.s * __builtin_amdgcn_exp2f((p.top - off) * c2));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = float2{top, s};
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; ++w) top = fmaxf(top, sh[w].x);
    off = finite_or_0(top);
    s = 0.0f;
    for (uint32_t w = 0; w < WAVES; ++w) s += sh[w].y * __builtin_amdgcn_exp2f((sh[w].x - off) * c2);
    return off * inv_t + logf(s);
}
// ... of S pairs of a row, `stride` apart
__device__ __forceinline__ Pair join_parts(const float2* parts, uint64_t stride, uint32_t S, float c2) {
    Pair p;
    for (uint32_t i = threadIdx.x; i < S; i += 4 * WORK) {
        float2 x[4];
        float t = p.top;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            x[k] = i + k * WORK < S ? parts[(i + k * WORK) * stride] : float2{-INFINITY, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) t = fmaxf(t, x[k].x);
        const float off = finite_or_0(t);
        p.s *= __builtin_amdgcn_exp2f((p.top - off) * c2);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) p.s += x[k].y * __builtin_amdgcn_exp2f((x[k].x - off) * c2);
        p.top = t;
    }
    return p;
}
// ... of a row of V logits
__device__ __forceinline__ Pair join_logits(const float* z, uint32_t V, float c2) {
    Pair p;
    for (int64_t c = 4 * threadIdx.x; c < V; c += 16 * WORK) {
        float x[4][4], t = p.top;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t at = c + 4 * k * WORK;
            if (at + 4 <= V) unpack<float>(ld16_any(z + at), x[k]);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) x[k][e] = at + e < V ? z[at + e] : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) t = fmaxf(t, x[k][e]);
        const float off = finite_or_0(t);
        p.s *= __builtin_amdgcn_exp2f((p.top - off) * c2);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) p.s += __builtin_amdgcn_exp2f((x[k][e] - off) * c2);
        p.top = t;
    }
    return p;
}

// Where the tiles of the logits leave those at the entries: each row's entries by
// slices of `width` classes, in counting order (which entry of a slice goes first
// is no matter: each has a place of its own in z_top).  M stride + M n small numbers
// to write; bound by a row's chain of five passes over LDS.
template <uint32_t SLICES>
__global__ __launch_bounds__(WORK) void table_kernel(uint32_t M, uint32_t V, uint32_t n, const int64_t* top,
                                                     int64_t ldtop, uint32_t width, uint32_t stride, uint32_t* list,
                                                     uint16_t* offs) {
    constexpr uint32_t EACH = SLICES / WORK;
    __shared__ uint32_t count[SLICES], waves[WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < SLICES; i += WORK) count[i] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            const int64_t c = top[(int64_t)m * ldtop + j];
            if (c >= 0 && c < V) atomicAdd(&count[(uint32_t)c / width], 1u);
        }
        __syncthreads();
        // the places before each slice: a thread's EACH, the lanes' before it, the waves' before those
        uint32_t own[EACH], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            own[i] = sum;
            sum += count[threadIdx.x * EACH + i];
        }
        uint32_t before = sum;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t x = (uint32_t)__shfl_up((int)before, d);
            before += lane >= (uint32_t)d ? x : 0;
        }
        if (lane == 63) waves[wave] = before;
        before -= sum;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) before += waves[w];
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            const uint32_t s = threadIdx.x * EACH + i;
            count[s] = before + own[i];
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < stride; i += WORK) offs[m * stride + i] = (uint16_t)count[i];
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            const int64_t c = top[(int64_t)m * ldtop + j];
            if (c < 0 || c >= V) continue;
            const uint32_t s = (uint32_t)c / width;
            list[m * n + atomicAdd(&count[s], 1u)] = j * width + ((uint32_t)c - s * width);
        }
    }
}

// One workgroup per row.  Its log-sum-exp comes from lse, from the parts that
// tiles or slices left (then lse is written) or, with neither, from the logits.
// The logits at the entries are there (given), read where the row is, or computed, the
// waves on DOTS entries at a time: one load of x's chunk for DOTS of w's rows.
// Those rows of w are the kernel's bytes: 4096 rows of 64 entries, K = 4096 and 128000
// classes in bf16, 165 us for 2.1 GB, half of it from HBM (6.4 TB/s).
constexpr uint32_t DOTS = 8;
template <typename T, typename TT>
__global__ __launch_bounds__(WORK) void rows_kernel(uint32_t M, uint32_t V, uint32_t K, const T* x, int64_t ldx,
                                                    const T* w, int64_t ldw, uint32_t n, const int64_t* top,
                                                    int64_t ldtop, const TT* t, int64_t ldt, float temp, float inv_t,
                                                    const float* logits, int64_t ldz, const float2* parts, uint32_t S,
                                                    int have_lse, int given, float* lse, float* loss,
                                                    float* z_top) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ Shared sh;
    __shared__ float z[TOP], sums[WAVES];
    __shared__ float2 pairs[WAVES];
    __shared__ uint32_t list[TOP], count;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        bool counted, bad;
        const float log_s = teacher(n, V, top + (int64_t)m * ldtop, t + (int64_t)m * ldt, inv_t, sh, counted, bad);
        // the entries with a class, in order
        if (wave == 0) {
            uint32_t c = 0;
            for (uint32_t j = lane; j - lane < n; j += 64) {
                const bool in = j < n && sh.id[j] >= 0;
                const uint64_t mask = __ballot(in);
                if (in) list[c + __popcll(mask & ((1ull << lane) - 1))] = j;
                c += (uint32_t)__popcll(mask);
            }
            if (lane == 0) count = c;
        }
        __syncthreads();
        const uint32_t there = logits || given ? 0 : count;
        const T* xr = x + (int64_t)m * ldx;
        for (uint32_t g = wave * DOTS; g < there; g += WAVES * DOTS) {
            const T* row[DOTS];
            float acc[DOTS];
#pragma unroll
            for (uint32_t e = 0; e < DOTS; ++e) {
                row[e] = w + (int64_t)__builtin_amdgcn_readfirstlane(sh.id[list[min(g + e, there - 1)]]) * ldw;
                acc[e] = 0.0f;
            }
#pragma unroll 1      // (two rounds of loads cost a wave per SIMD: 38 -> 51 us at 1000 rows of 200 entries, K = 1024)
            for (int64_t k = (int64_t)lane * VEC; k < K; k += 64 * VEC) {
                float a[VEC];
                unpack<T>(ld_chunk(xr, k, K), a);
#pragma unroll
                for (uint32_t e = 0; e < DOTS; ++e) {
                    float b[VEC];
                    unpack<T>(ld_chunk(row[e], k, K), b);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[e] = __builtin_fmaf(a[i], b[i], acc[e]);
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < DOTS; ++e) {
                const float s = wave_sum(acc[e]);
                if (lane == 0 && g + e < there) z[list[g + e]] = s;
            }
        }
        float l;
        if (have_lse) l = lse[m];
        else
            l = block_lse(S ? join_parts(parts + m, M, S, inv_t * LOG2E)
                            : join_logits(logits + (int64_t)m * ldz, V, inv_t * LOG2E), inv_t, pairs);
        if (!have_lse && threadIdx.x == 0) lse[m] = l;
        __syncthreads();
        float s = 0.0f;
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            const int id = sh.id[j];
            const float v = id == ABSENT ? 0.0f : id == BAD ? __builtin_nanf("")
                          : given ? z_top[(int64_t)m * n + j] : logits ? logits[(int64_t)m * ldz + id] : z[j];
            z_top[(int64_t)m * n + j] = v;
            const float log_q = sh.q[j] - log_s, q = fast_exp(log_q);
            if (id != ABSENT && !(q == 0.0f)) s += q * (log_q - (v * inv_t - l));
        }
        s = wave_sum(s);
        if (lane == 0) sums[wave] = s;
        __syncthreads();      // (the next row's entries are written past this)
        if (threadIdx.x == 0) {
            for (uint32_t i = 1; i < WAVES; ++i) s += sums[i];
            loss[m] = bad ? __builtin_nanf("") : counted ? temp * temp * s : 0.0f;
        }
    }
}

// The backward pass's rows: q of each entry's class (where a class occurs twice
// both entries' at the first, -1 at the other: one of them patches D), T dloss,
// and a target for D's kernels: `ignore` where the row is not counted, V where it
// is bad, else the first entry's class, whose element the patch writes over.
// Classes that occur twice are found by a hash of the row's in LDS (us at 4096 rows, by
// comparing each pair of entries / so: 64 entries 10.2 / 9.7, 256 24 / 12, 1024 245 / 41;
// 64 entries with the 24 KB that 1024 need 16).
template <typename TT, uint32_t CAP>
__global__ __launch_bounds__(WORK) void prepare_kernel(uint32_t M, uint32_t V, uint32_t n, const int64_t* top,
                                                       int64_t ldtop, const TT* t, int64_t ldt, float temp, float inv_t,
                                                       const float* dloss, int64_t ignore, float* q_top,
                                                       int64_t* target, float* dl) {
    __shared__ Shared sh;
    __shared__ int first[WAVES], key[2 * CAP];           // key: a place's class, or ABSENT
    __shared__ uint32_t leader[2 * CAP], times[2 * CAP];
    uint32_t bits = 6;
    while (1u << bits < 2 * n) ++bits;
    const uint32_t places = 1u << bits;
    for (uint64_t m = blockIdx.x; m < M; m += gridDim.x) {
        for (uint32_t i = threadIdx.x; i < places; i += WORK) {
            key[i] = ABSENT;
            leader[i] = n;
            times[i] = 0;
        }
        bool counted, bad;
        const float log_s = teacher(n, V, top + (int64_t)m * ldtop, t + (int64_t)m * ldt, inv_t, sh, counted, bad);
        int at = (int)n;
        for (uint32_t j = threadIdx.x; j < n; j += WORK) {
            sh.q[j] = sh.id[j] == ABSENT ? 0.0f : fast_exp(sh.q[j] - log_s);
            if (sh.id[j] >= 0) at = min(at, (int)j);
        }
        for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d));
        if ((threadIdx.x & 63) == 0) first[threadIdx.x >> 6] = at;
        uint32_t place[CAP / WORK];
#pragma unroll
        for (uint32_t l = 0; l < CAP / WORK; ++l) {
            const uint32_t j = l * WORK + threadIdx.x;
            const int id = j < n ? sh.id[j] : ABSENT;
            place[l] = places;
            if (id < 0) continue;
            uint32_t h = (uint32_t)id * 2654435761u >> (32 - bits);
            for (;; h = (h + 1) & (places - 1)) {        // (at most half of the places are taken)
                const int there = atomicCAS(&key[h], ABSENT, id);
                if (there == ABSENT || there == id) break;
            }
            atomicMin(&leader[h], j);
            atomicAdd(&times[h], 1u);
            place[l] = h;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t l = 0; l < CAP / WORK; ++l) {
            const uint32_t j = l * WORK + threadIdx.x, h = place[l];
            if (j >= n) continue;
            float q = sh.q[j];
            if (h < places && times[h] > 1) {
                if (leader[h] != j) q = -1.0f;
                else
                    for (uint32_t i = j + 1; i < n; ++i) q += sh.id[i] == sh.id[j] ? sh.q[i] : 0.0f;
            }
            q_top[(int64_t)m * n + j] = q;
        }
        if (threadIdx.x == 0) {
            for (uint32_t i = 0; i < WAVES; ++i) at = min(at, first[i]);
            target[m] = bad ? (int64_t)V : counted && at < (int)n ? (int64_t)sh.id[at] : ignore;
            dl[m] = temp * dloss[m];
        }
        __syncthreads();
    }
}

// D in place at the entries, after the kernels that write p of every class: 5 us for
// 4096 rows of 64, each entry's 2 or 4 bytes by themselves.
// The entries whose class lies in columns v0 .. v0 + cols - 1
template <typename T>
__global__ __launch_bounds__(WORK) void patch_kernel(uint32_t M, uint32_t V, uint32_t n, const int64_t* top,
                                                     int64_t ldtop, uint32_t v0, uint32_t cols, float inv_t,
                                                     const float* lse, const float* z_top, const float* q_top,
                                                     const int64_t* target, int64_t ignore, const float* dl,
                                                     const float* scal, T* D, int64_t ldd) {
    const float sc = scal ? scal[0] : 1.0f;
    const uint64_t total = (uint64_t)M * n;
    for (uint64_t i = (uint64_t)blockIdx.x * WORK + threadIdx.x; i < total; i += (uint64_t)gridDim.x * WORK) {
        const uint64_t m = i / n;
        const int64_t id = top[(int64_t)m * ldtop + (int64_t)(i - m * n)], c = id - v0;
        const float q = q_top[i];
        if (id < 0 || c < 0 || c >= cols || q < 0.0f || target[m] == ignore || target[m] >= V) continue;
        const float p = fast_exp(z_top[i] * inv_t - lse[m]);
        D[(int64_t)m * ldd + c] = (T)(dl[m] * sc * (p - q));
    }
}

}  // namespace
}  // namespace vkb

using namespace vkb;

static uint32_t row_blocks(uint32_t M) { return M < 65536 ? M : 65536; }

extern "C" int vkb_launch_distill_rows(int type, int t_type, const vkb_distill* d, uint32_t K, const void* x,
                                       int64_t ldx, const void* w, int64_t ldw, const vkb_distill_rows* r,
                                       void* stream) {
    const bool ok = with_type(type, [&](auto e) {
        using T = decltype(e);
        auto launch = [&](auto f) {
            using TT = decltype(f);
            hipLaunchKernelGGL((rows_kernel<T, TT>), dim3(row_blocks(d->M)), dim3(WORK), 0, (hipStream_t)stream, d->M,
                               d->V, K, (const T*)x, ldx, (const T*)w, ldw, d->n, d->top, d->ldtop, (const TT*)d->t,
                               d->ldt, d->temp, 1.0f / d->temp, r->z, r->ldz, (const float2*)r->parts, r->S,
                               r->have_lse, r->given, r->lse, r->loss, r->z_top);
        };
        if (t_type == VKB_T_F32) launch(float{});
        else launch(e);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_distill_table(const vkb_distill* d, const vkb_distill_table* t, void* stream) {
    if (t->stride > VKB_DISTILL_SLICES + 1) return (int)hipErrorInvalidValue;
    if (t->stride <= 1024)
        hipLaunchKernelGGL(table_kernel<1024>, dim3(row_blocks(d->M)), dim3(WORK), 0, (hipStream_t)stream, d->M, d->V,
                           d->n, d->top, d->ldtop, t->width, t->stride, t->list, t->offs);
    else
        hipLaunchKernelGGL((table_kernel<VKB_DISTILL_SLICES + WORK>), dim3(row_blocks(d->M)), dim3(WORK), 0,
                           (hipStream_t)stream, d->M, d->V, d->n, d->top, d->ldtop, t->width, t->stride, t->list,
                           t->offs);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_distill_prepare(int t_type, const vkb_distill* d, const float* dloss, void* stream) {
    if (d->n > TOP) return (int)hipErrorInvalidValue;
    const bool ok = with_type(t_type, [&](auto f) {
        using TT = decltype(f);
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(row_blocks(d->M)), dim3(WORK), 0, (hipStream_t)stream, d->M, d->V, d->n,
                               d->top, d->ldtop, (const TT*)d->t, d->ldt, d->temp, 1.0f / d->temp, dloss, d->ignore,
                               d->q_top, d->target, d->dl);
        };
        if (d->n <= WORK) launch(prepare_kernel<TT, WORK>);
        else launch(prepare_kernel<TT, TOP>);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_distill_patch(int type, const vkb_distill* d, uint32_t v0, uint32_t cols, const float* lse,
                                        const float* z_top, const float* scal, void* D, int64_t ldd, void* stream) {
    const bool ok = with_type(type, [&](auto e) {
        using T = decltype(e);
        hipLaunchKernelGGL((patch_kernel<T>), dim3(chunk_blocks(d->M, d->n)), dim3(WORK), 0, (hipStream_t)stream, d->M,
                           d->V, d->n, d->top, d->ldtop, v0, cols, 1.0f / d->temp, lse, z_top, d->q_top, d->target,
                           d->ignore, d->dl, scal, (T*)D, ldd);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}
