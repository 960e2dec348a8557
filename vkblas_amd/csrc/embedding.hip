// embedding.hip — the tokens' embedding and its gradient.
//
// y[m] = s w[ids[m]] is a copy of rows.  The gradient is the sum of each
// token's rows of dy, over a vocabulary of which a batch meets a small part, a
// few tokens hundreds of times.  Atomic additions would make its bits depend on
// their order and serialise on the frequent tokens, so tokens are grouped
// first: (id, m) pairs sorted by id, then m, in the workspace.
//
//  - Sort: runs of RUN pairs by counting (a pair's place is the number of pairs
//    before it: RUN comparisons each, no passes that depend on each other), then
//    merges of up to WAYS runs at a time (a pair's place is its own index plus
//    binary searches in the other runs, all in flight at once).
//  - Sums: the sorted pairs in chunks of equal length, so that frequent tokens
//    are spread over the chip.  A wave sums a chunk's rows over its columns; a
//    token that ends inside goes to dw, a part that began before the chunk or
//    goes on after it to the workspace.
//  - Join: a token of several chunks adds their parts in order.
// Rows of dw without a token are zeroed beside the sort (beta = 0), left alone
// (beta = 1), or scaled by a pass that searches each row's id.
#include "nn_common.hpp"

namespace vkb {
namespace {

constexpr uint32_t RUN = VKB_EMBED_RUN, WAYS = VKB_EMBED_WAYS;

template <typename T, typename W>
__global__ __launch_bounds__(WORK) void lookup_kernel(uint32_t M, uint32_t V, uint32_t N, const int64_t* ids,
                                                      int64_t pad, const W* w, int64_t ldw, float scale, T* y,
                                                      int64_t ldy) {
    constexpr int VEC = Elem<T>::VEC;
    for_chunks(M, (N + VEC - 1) / VEC, 0, gridDim.x, [&](uint64_t m, uint32_t k) {
        const int64_t c = (int64_t)k * VEC, id = ids[m];
        const bool in = id != pad && id >= 0 && id < V;
        const float none = id == pad ? 0.0f : __builtin_nanf("");
        float x[VEC];
        if (in) {
            const W* row = w + id * ldw;
#pragma unroll
            for (int q = 0; q < VEC; q += Elem<W>::VEC) unpack<W>(ld_chunk(row, c + q, N), x + q);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = in ? scale * x[i] : none;
        st_chunk(y + (int64_t)m * ldy, c, N, pack<T>(x));
    });
}

// What an id is sorted by: itself, or V (behind all others) where its row adds
// nothing.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t pad, uint32_t V) {
    return id != pad && id >= 0 && id < V ? (uint32_t)id : V;
}

// RTOK tokens of a run per workgroup, 16 groups of threads on a part of the
// run's keys each.  A pair before the token's counts where its key is at most
// the token's, one after it where it is less.
constexpr uint32_t RTOK = 16, RGROUPS = WORK / RTOK;
template <typename W>
__global__ __launch_bounds__(WORK) void rank_kernel(uint32_t M, uint32_t V, const int64_t* ids, int64_t pad,
                                                    uint32_t* key, uint32_t* order, uint32_t rank_blocks, uint32_t N,
                                                    W* dw, int64_t lddw) {
    if (blockIdx.x >= rank_blocks) {      // dw = 0
        constexpr int VEC = Elem<W>::VEC;
        for_chunks(V, (N + VEC - 1) / VEC, rank_blocks, gridDim.x - rank_blocks, [&](uint64_t v, uint32_t k) {
            st_chunk(dw + (int64_t)v * lddw, (int64_t)k * VEC, N, u32x4{0u, 0u, 0u, 0u});
        });
        return;
    }
    __shared__ __attribute__((aligned(16))) uint32_t keys[RUN];
    __shared__ uint32_t count[WORK];
    const uint32_t tok = threadIdx.x % RTOK, g = threadIdx.x / RTOK;
    for (uint64_t first = (uint64_t)blockIdx.x * RTOK; first < M; first += (uint64_t)rank_blocks * RTOK) {
        const uint64_t run = first / RUN * RUN;
        const uint32_t n = (uint32_t)min((uint64_t)RUN, M - run), whole = (n + 3) / 4 * 4;
        for (uint32_t i = threadIdx.x; i < whole; i += WORK) keys[i] = i < n ? sort_key(ids[run + i], pad, V) : ~0u;
        __syncthreads();
        const uint32_t me = (uint32_t)(first - run) + tok;
        const uint32_t mine = me < n ? keys[me] : 0;
        // groups take quads of keys in turn: neighbouring ones read neighbouring banks
        uint32_t below = 0;
#pragma unroll 4
        for (uint32_t i = 4 * g; i < whole; i += 4 * RGROUPS) {
            const u32x4 k = *(const u32x4*)(keys + i);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) below += k[e] < mine + (i + e < me ? 1u : 0u);
        }
        count[threadIdx.x] = below;
        __syncthreads();
        if (threadIdx.x < RTOK && me < n) {
            uint32_t at = 0;
#pragma unroll
            for (uint32_t i = 0; i < RGROUPS; ++i) at += count[i * RTOK + tok];
            key[run + at] = mine;
            order[run + at] = (uint32_t)(run + me);
        }
    }
}

// Groups of WAYS sorted runs of `len` pairs into one.  The earlier run's pair
// goes first among equal keys, so pairs stay in the order of m.
__global__ __launch_bounds__(WORK) void merge_kernel(uint32_t M, uint64_t len, uint32_t steps, const uint32_t* key_in,
                                                     const uint32_t* order_in, uint32_t* key, uint32_t* order) {
    const uint64_t i = (uint64_t)blockIdx.x * WORK + threadIdx.x;
    if (i >= M) return;
    const uint64_t group = i / (len * WAYS) * (len * WAYS);
    const uint32_t own = (uint32_t)((i - group) / len), k = key_in[i];
    uint32_t lo[WAYS], hi[WAYS];
    uint64_t at = i - (group + own * len);
#pragma unroll
    for (uint32_t r = 0; r < WAYS; ++r) {
        const uint64_t start = group + r * len;
        lo[r] = 0;
        hi[r] = r != own && start < M ? (uint32_t)min(len, M - start) : 0u;
    }
    for (uint32_t s = 0; s < steps; ++s) {
        uint32_t x[WAYS];
#pragma unroll
        for (uint32_t r = 0; r < WAYS; ++r)
            x[r] = lo[r] < hi[r] ? key_in[group + r * len + (lo[r] + hi[r]) / 2] : 0u;
#pragma unroll
        for (uint32_t r = 0; r < WAYS; ++r)
            if (lo[r] < hi[r]) {
                const uint32_t mid = (lo[r] + hi[r]) / 2;
                if (r < own ? x[r] <= k : x[r] < k) lo[r] = mid + 1;
                else hi[r] = mid;
            }
    }
#pragma unroll
    for (uint32_t r = 0; r < WAYS; ++r) at += lo[r];
    key[group + at] = k;
    order[group + at] = order_in[i];
}

// dw = beta * dw on the rows that no token has
template <typename W>
__global__ __launch_bounds__(WORK) void scale_others_kernel(uint32_t M, uint32_t V, uint32_t N, const uint32_t* key,
                                                            W* dw, int64_t lddw, float beta) {
    constexpr int VEC = Elem<W>::VEC;
    for (uint64_t v = blockIdx.x; v < V; v += gridDim.x) {
        uint32_t lo = 0, hi = M;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (key[mid] < v) lo = mid + 1;
            else hi = mid;
        }
        if (lo < M && key[lo] == v) continue;
        W* row = dw + (int64_t)v * lddw;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < N; c += (int64_t)WORK * VEC) {
            float x[VEC];
            unpack<W>(ld_chunk(row, c, N), x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] *= beta;
            st_chunk(row, c, N, pack<W>(x));
        }
    }
}

struct SumParams {
    uint32_t M, V, N, chunk, chunks, blocks;    // blocks: of columns
    const uint32_t *key, *order;
    const void* dy;
    int64_t lddy;
    void* dw;
    int64_t lddw;
    float scale, beta;
    float* part;             // chunks x 2 x N: what began before a chunk, what goes on after it
};

// dw's columns c .. of a token: its sum, scaled, and what was there
template <typename T, typename W>
__device__ __forceinline__ void put(const SumParams& p, uint32_t v, int64_t c, const float* acc) {
    constexpr int VEC = Elem<T>::VEC, WV = Elem<W>::VEC;
    W* row = (W*)p.dw + (int64_t)v * p.lddw;
#pragma unroll
    for (int q = 0; q < VEC; q += WV) {
        if (c + q >= p.N) break;
        float x[WV];
        if (p.beta != 0.0f) {
            unpack<W>(ld_chunk(row, c + q, p.N), x);
#pragma unroll
            for (int i = 0; i < WV; ++i) x[i] = p.beta * x[i] + p.scale * acc[q + i];
        } else {
#pragma unroll
            for (int i = 0; i < WV; ++i) x[i] = p.scale * acc[q + i];
        }
        st_chunk(row, c + q, p.N, pack<W>(x));
    }
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// A wave: one chunk, 64 x 16 bytes of its rows' columns, SROWS rows in flight.
constexpr uint32_t SROWS = 8;
template <typename T, typename W>
__global__ __launch_bounds__(WORK) void sum_kernel(SumParams p) {
    constexpr int VEC = Elem<T>::VEC;
    const uint64_t unit = (uint64_t)blockIdx.x * (WORK / 64) + uniform(threadIdx.x >> 6);
    const uint32_t chunk = (uint32_t)(unit / p.blocks), block = (uint32_t)(unit % p.blocks);
    if (chunk >= p.chunks) return;
    const int64_t c = ((int64_t)block * 64 + (threadIdx.x & 63)) * VEC;
    const uint32_t p0 = chunk * p.chunk, p1 = p0 + min(p.chunk, p.M - p0);
    const uint32_t before = p0 ? uniform(p.key[p0 - 1]) : ~0u, after = p1 < p.M ? uniform(p.key[p1]) : ~0u;
    float acc[VEC];
    uint32_t now = uniform(p.key[p0]);
    bool began = now == before;
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    };
    // the token `now` ends here, or goes on in the next chunk
    auto done = [&](bool on) {
        if (c >= p.N) return;
        if (!began && !on) {
            put<T, W>(p, now, c, acc);
            return;
        }
        float* part = p.part + ((int64_t)chunk * 2 + (began ? 0 : 1)) * p.N;
#pragma unroll
        for (int q = 0; q < VEC; q += 4)
            if (c + q < p.N) st_chunk(part, c + q, p.N, pack<float>(acc + q));
    };
    clear();
    // 64 pairs at a time in the lanes
    for (uint32_t base = p0; base < p1 && now < p.V; base += 64) {
        const uint32_t n = min(64u, p1 - base), mine = base + min(threadIdx.x & 63, n - 1);
        const uint32_t keys = p.key[mine], rows = p.order[mine];
        for (uint32_t i = 0; i < n; i += SROWS) {
            u32x4 x[SROWS];
#pragma unroll
            for (uint32_t r = 0; r < SROWS; ++r) {
                const uint32_t m = (uint32_t)__builtin_amdgcn_readlane((int)rows, (int)min(i + r, n - 1));
                x[r] = ld_chunk((const T*)p.dy + (int64_t)m * p.lddy, c, p.N);
            }
#pragma unroll
            for (uint32_t r = 0; r < SROWS; ++r) {
                if (i + r >= n || now >= p.V) continue;
                const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)keys, (int)(i + r));
                if (k != now) {
                    done(false);
                    clear();
                    now = k;
                    began = false;
                    if (now >= p.V) continue;
                }
                float f[VEC];
                unpack<T>(x[r], f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += f[e];
            }
        }
    }
    if (now < p.V) done(now == after);
}

// A token that begins in a chunk and goes on: that chunk's part and those of
// the chunks it fills, the waves on a quarter each, in order.
template <typename T, typename W>
__global__ __launch_bounds__(WORK) void join_kernel(SumParams p) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ float sh[WORK / 64 - 1][64][VEC + 1];
    const uint32_t chunk = blockIdx.y, block = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const uint32_t p0 = chunk * p.chunk, p1 = p0 + p.chunk;      // the last chunk is not here
    const uint32_t k = p.key[p1 - 1];
    if (k >= p.V || p.key[p1] != k || (p0 && p.key[p0] == k && p.key[p0 - 1] == k)) return;
    // the last chunk whose first key is k: keys are sorted
    uint32_t lo = chunk + 1, hi = p.chunks - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (p.key[mid * p.chunk] == k) lo = mid;
        else hi = mid - 1;
    }
    const uint32_t parts = lo - chunk + 1, each = (parts + 3) / 4;
    const uint32_t a = min(wave * each, parts), b = min(a + each, parts);
    const int64_t c = ((int64_t)block * 64 + lane) * VEC;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    // part i: the tail of the first chunk, then the heads of the others
    auto row = [&](uint32_t i) { return p.part + ((int64_t)(chunk + i) * 2 + (i ? 0 : 1)) * p.N; };
    if (c < p.N)
        for (uint32_t i = a; i < b; i += 4) {
            u32x4 x[4][VEC / 4];
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
                for (int q = 0; q < VEC; q += 4) x[r][q / 4] = ld_chunk(row(min(i + r, b - 1)), c + q, p.N);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                if (i + r >= b) continue;
#pragma unroll
                for (int q = 0; q < VEC; q += 4) {
                    float f[4];
                    unpack<float>(x[r][q / 4], f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[q + e] += f[e];
                }
            }
        }
    if (wave) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) sh[wave - 1][lane][i] = acc[i];
    }
    __syncthreads();
    if (wave || c >= p.N) return;
#pragma unroll
    for (int w = 0; w < (int)WORK / 64 - 1; ++w)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += sh[w][lane][i];
    put<T, W>(p, k, c, acc);
}

// f(T{}, W{}) for a type and one that is it or fp32
template <typename F>
bool with_types(int type, int other, F f) {
    return with_type(type, [&](auto t) {
        if (other == VKB_T_F32) f(t, float{});
        else f(t, t);
    });
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" int vkb_launch_embedding(int type, int w_type, uint32_t M, uint32_t V, uint32_t N, const int64_t* ids,
                                    int64_t pad, const void* w, int64_t ldw, float scale, void* y, int64_t ldy,
                                    void* stream) {
    const bool ok = with_types(type, w_type, [&](auto t, auto o) {
        using T = decltype(t);
        using W = decltype(o);
        hipLaunchKernelGGL((lookup_kernel<T, W>), dim3(chunk_blocks(M, chunks_of<T>(N))), dim3(WORK), 0,
                           (hipStream_t)stream, M, V, N, ids, pad, (const W*)w, ldw, scale, (T*)y, ldy);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_rank(uint32_t M, uint32_t V, const int64_t* ids, int64_t pad, uint32_t* key,
                                         uint32_t* order, int w_type, uint32_t N, void* dw, int64_t lddw,
                                         void* stream) {
    const uint32_t tiles = (uint32_t)(((uint64_t)M + RTOK - 1) / RTOK), ranks = tiles < 65536 ? tiles : 65536;
    const bool ok = with_type(w_type, [&](auto t) {
        using W = decltype(t);
        const uint32_t fill = dw ? chunk_blocks(V, chunks_of<W>(N)) : 0;
        hipLaunchKernelGGL((rank_kernel<W>), dim3(ranks + fill), dim3(WORK), 0, (hipStream_t)stream, M, V, ids, pad,
                           key, order, ranks, N, (W*)dw, lddw);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_merge(uint32_t M, uint64_t len, const uint32_t* key_in, const uint32_t* order_in,
                                          uint32_t* key, uint32_t* order, void* stream) {
    // a search over n places takes as many steps as n has binary digits
    const uint64_t n = len < M ? len : M;
    const uint32_t steps = 64 - (uint32_t)__builtin_clzll(n);
    hipLaunchKernelGGL(merge_kernel, dim3((M + WORK - 1) / WORK), dim3(WORK), 0, (hipStream_t)stream, M, len, steps,
                       key_in, order_in, key, order);
    return (int)hipGetLastError();
}

extern "C" int vkb_launch_embedding_scale(int w_type, uint32_t M, uint32_t V, uint32_t N, const uint32_t* key, void* dw,
                                          int64_t lddw, float beta, void* stream) {
    const bool ok = with_type(w_type, [&](auto t) {
        using W = decltype(t);
        hipLaunchKernelGGL((scale_others_kernel<W>), dim3(V < 8192 ? V : 8192), dim3(WORK), 0, (hipStream_t)stream,
                           M, V, N, key, (W*)dw, lddw, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_sums(int type, int w_type, const vkb_embedding_sums* a, void* stream) {
    const uint32_t cols = 64 * (type == VKB_T_F32 ? 4 : 8);
    SumParams p{a->M, a->V, a->N, a->chunk, a->chunks, (a->N + cols - 1) / cols, a->key, a->order, a->dy, a->lddy,
                a->dw, a->lddw, a->scale, a->beta, a->part};
    const uint64_t units = (uint64_t)p.chunks * p.blocks;
    if (units > 0xffffffffull / WORK) return (int)hipErrorInvalidValue;
    int rc = (int)hipErrorInvalidValue;
    with_types(type, w_type, [&](auto t, auto o) {
        using T = decltype(t);
        using W = decltype(o);
        hipLaunchKernelGGL((sum_kernel<T, W>), dim3((uint32_t)((units + 3) / 4)), dim3(WORK), 0, (hipStream_t)stream,
                           p);
        rc = (int)hipGetLastError();
        if (rc != 0 || p.chunks == 1) return;
        hipLaunchKernelGGL((join_kernel<T, W>), dim3(p.blocks, p.chunks - 1), dim3(WORK), 0, (hipStream_t)stream, p);
        rc = (int)hipGetLastError();
    });
    return rc;
}
