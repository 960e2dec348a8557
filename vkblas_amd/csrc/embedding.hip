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
// dw is zeroed beside the first step of the sort (beta = 0), or its rows without
// a token are scaled by a pass that searches their ids (not for beta = 1).
//
// Few tokens and a small dw take one launch without a workspace: each workgroup
// looks all ids over for those of its own rows of dw.
#include "nn_common.hpp"

namespace vkb {
namespace {

constexpr uint32_t RUN = VKB_EMBED_RUN, WAYS = VKB_EMBED_WAYS;

// Bound by its reads and writes: fp32 to bf16 16384 x 4096, 403 MB, 45 us (164 MB of
// the 268 that it reads come from HBM, a frequent token's row out of the caches: 6.6
// TB/s).  One chunk a thread, many short
// workgroups: 8192 in strides 47 us.
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
//
// The workgroups from ranks on zero dw, 16 bytes a thread: stores are fastest
// from many short workgroups (1 GiB of zeros: 4 KB each 6.8 TB/s, 8 KB 6.1, 512 KB 5.7,
// 8192 workgroups in strides 4.6; rows with tokens left out, which takes a look at
// a map of them, 4.6 beside the sums).  Beside 1 GB of them, 150 us, the ranks cost
// nothing.  Runs of 1024 / 2048: 16384 tokens and 65 MB of zeros 11.8 / 14.5 us, and
// their merge 4.1 / 4.0; 65536 and 33 MB 14.7 / 20.2, and 13.4 / 9.7.
constexpr uint32_t RTOK = 16, RGROUPS = WORK / RTOK;
template <typename W>
__global__ __launch_bounds__(WORK) void rank_kernel(uint32_t M, uint32_t V, const int64_t* ids, int64_t pad,
                                                    uint32_t* key, uint32_t* order, uint32_t ranks, uint32_t N, W* dw,
                                                    int64_t lddw) {
    if (blockIdx.x >= ranks) {
        constexpr int VEC = Elem<W>::VEC;
        for_chunks(V, (N + VEC - 1) / VEC, ranks, gridDim.x - ranks, [&](uint64_t v, uint32_t k) {
            st_chunk(dw + (int64_t)v * lddw, (int64_t)k * VEC, N, u32x4{0u, 0u, 0u, 0u});
        });
        return;
    }
    __shared__ __attribute__((aligned(16))) uint32_t keys[RUN];
    __shared__ uint32_t count[WORK];
    const uint32_t tok = threadIdx.x % RTOK, g = threadIdx.x / RTOK;
    for (uint64_t first = (uint64_t)blockIdx.x * RTOK; first < M; first += (uint64_t)ranks * RTOK) {
        const uint64_t run = first / RUN * RUN;
        const uint32_t n = (uint32_t)min((uint64_t)RUN, M - run), whole = (n + 3) / 4 * 4;
        int64_t id[RUN / WORK];               // all loads in flight
#pragma unroll
        for (uint32_t l = 0; l < RUN / WORK; ++l)
            if (l * WORK < n) id[l] = ids[run + min(l * WORK + threadIdx.x, n - 1)];
#pragma unroll
        for (uint32_t l = 0; l < RUN / WORK; ++l) {
            const uint32_t i = l * WORK + threadIdx.x;
            if (i < whole) keys[i] = i < n ? sort_key(id[l], pad, V) : ~0u;
        }
        __syncthreads();
        const uint32_t me = (uint32_t)(first - run) + tok;
        const uint32_t mine = me < n ? keys[me] : 0;
        // groups take quads of keys in turn: neighbouring ones read neighbouring banks.  The workgroup's tokens
        // are 4 quads, so a quad of another place is before or after all of them.
        const uint32_t here = (uint32_t)(first - run);
        uint32_t below = 0;
#pragma unroll 4
        for (uint32_t i = 4 * g; i < whole; i += 4 * RGROUPS) {
            const u32x4 k = *(const u32x4*)(keys + i);
            const uint32_t bound = mine + (i < here ? 1u : 0u);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) below += k[e] < bound;
        }
        // equal keys before the token among its neighbours
        if (g == 0)
            for (uint32_t i = here; i < me && i < n; ++i) below += keys[i] == mine;
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

// Groups of sorted runs into one.  The earlier run's pair goes first among equal
// keys, so pairs stay in the order of m.
//
// Runs of RUN: a search is a chain of reads, so it runs in LDS, where a group's
// keys fit (S = 1, WAYS runs), or the last of each S of them (S = 4, S WAYS
// runs): then the S keys at the place found there are read and counted.
// Searches count the keys below a bound, which for earlier runs is past the
// pair's own key; SEARCHES of them run side by side, and MGROUPS waves share the
// runs of 64 pairs (with one wave for all of them, runs of 2048, 16384 pairs took 6.0 us,
// not 4.0, and 65536 pairs 18, not 9.7: the LDS leaves a CU few workgroups, so few waves
// to hide the searches' chains).
constexpr uint32_t MGROUPS = 4, MTHREADS = MGROUPS * WORK;
template <uint32_t S>
__global__ __launch_bounds__(MTHREADS) void merge_runs_kernel(uint32_t M, const uint32_t* key_in,
                                                              const uint32_t* order_in, uint32_t* key,
                                                              uint32_t* order) {
    constexpr uint32_t GROUP = RUN * WAYS * S, LEN = RUN / S;      // pairs of a group, keys of a run in LDS
    constexpr uint32_t SEARCHES = S == 1 ? 4 : 8;
    __shared__ uint32_t places[MGROUPS - 1][WORK];
    __shared__ __attribute__((aligned(16))) uint32_t keys[LEN * WAYS * S];
    for (uint64_t first = (uint64_t)blockIdx.x * WORK; first < M; first += (uint64_t)gridDim.x * WORK) {
        const uint64_t group = first / GROUP * GROUP;
        const uint32_t n = (uint32_t)min((uint64_t)GROUP, M - group), runs = (n + RUN - 1) / RUN;
        // whole runs, the last one filled up with keys above all others; LOADS in flight
        constexpr uint32_t LOADS = 4;
        for (uint32_t q0 = 0; q0 < runs * (RUN / 4); q0 += LOADS * MTHREADS) {
            u32x4 x[LOADS];
#pragma unroll
            for (uint32_t l = 0; l < LOADS; ++l) {
                const uint32_t i = 4 * (q0 + l * MTHREADS + threadIdx.x);
                if (i + 4 <= n) x[l] = *(const u32x4*)(key_in + group + i);
                else
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) x[l][e] = i + e < n ? key_in[group + i + e] : ~0u;
            }
#pragma unroll
            for (uint32_t l = 0; l < LOADS; ++l) {
                const uint32_t q = q0 + l * MTHREADS + threadIdx.x;
                if (q >= runs * (RUN / 4)) continue;
                if constexpr (S == 1) *(u32x4*)(keys + 4 * q) = x[l];
                else keys[q] = x[l][3];
            }
        }
        __syncthreads();
        const uint32_t share = threadIdx.x / WORK, pair = threadIdx.x % WORK;
        const uint32_t i = min((uint32_t)(first - group) + pair, n - 1);
        const uint32_t own = i / RUN, k = key_in[group + i], o = order_in[group + i];
        uint32_t at = 0;
        for (uint32_t r0 = share * SEARCHES; r0 < runs; r0 += MGROUPS * SEARCHES) {
            uint32_t pos[SEARCHES];
#pragma unroll
            for (uint32_t r = 0; r < SEARCHES; ++r) pos[r] = 0;
#pragma unroll
            for (uint32_t step = LEN / 2; step; step /= 2)
#pragma unroll
                for (uint32_t r = 0; r < SEARCHES; ++r) {
                    const uint32_t* run = keys + min(r0 + r, runs - 1) * LEN;
                    pos[r] += run[pos[r] + step - 1] < k + (r0 + r < own ? 1u : 0u) ? step : 0u;
                }
#pragma unroll
            for (uint32_t r = 0; r < SEARCHES; ++r) {
                const uint32_t run = min(r0 + r, runs - 1), bound = k + (run < own ? 1u : 0u);
                pos[r] += keys[run * LEN + pos[r]] < bound ? 1u : 0u;
            }
            if constexpr (S == 4) {
                u32x4 x[SEARCHES];
#pragma unroll
                for (uint32_t r = 0; r < SEARCHES; ++r) {
                    const uint32_t j = 4 * (min(r0 + r, runs - 1) * LEN + min(pos[r], LEN - 1));
                    if (j + 4 <= n) x[r] = *(const u32x4*)(key_in + group + j);
                    else
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) x[r][e] = j + e < n ? key_in[group + j + e] : ~0u;
                }
#pragma unroll
                for (uint32_t r = 0; r < SEARCHES; ++r) {
                    const uint32_t bound = k + (r0 + r < own ? 1u : 0u);
                    uint32_t c = 0;
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) c += x[r][e] < bound ? 1u : 0u;
                    pos[r] = 4 * pos[r] + (pos[r] < LEN ? c : 0u);
                }
            }
#pragma unroll
            for (uint32_t r = 0; r < SEARCHES; ++r) at += r0 + r < runs && r0 + r != own ? pos[r] : 0u;
        }
        if (share) places[share - 1][pair] = at;
        __syncthreads();
        if (share == 0 && (uint32_t)(first - group) + pair < n) {
            at += i % RUN;
#pragma unroll
            for (uint32_t s = 0; s < MGROUPS - 1; ++s) at += places[s][pair];
            key[group + at] = k;
            order[group + at] = o;
        }
        __syncthreads();                 // the next pairs' keys and places
    }
}

// Runs of `len`, WAYS at a time, searched in memory
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

// A wave's 64 x 16 bytes of a row's columns, without branches around the loads:
// VECTOR, 16 bytes a lane, where N is of whole 16-byte units or the wave's
// columns all exist (lanes past the row's end read its last ones and write
// nothing); else single columns, 64 apart, the last one read in the place of
// those past it.
template <typename T, bool VECTOR>
struct Cols {
    static constexpr int VEC = Elem<T>::VEC;
    static constexpr uint32_t ROWS = 8;          // in flight
    struct Row {
        u32x4 v;
    };
    int64_t c, N;
    bool in;
    __device__ __forceinline__ Cols(int64_t block, uint32_t lane, int64_t n) : N(n) {
        const int64_t at = (block * 64 + lane) * VEC;
        in = at < N;
        c = min(at, N - VEC);
    }
    __device__ __forceinline__ Row load(const T* row) const { return Row{ld16_any(row + c)}; }
    static __device__ __forceinline__ void add(const Row& r, float* acc) {
        float f[VEC];
        unpack<T>(r.v, f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += f[i];
    }
    template <typename E>
    __device__ __forceinline__ void get(const E* row, float* x) const {
#pragma unroll
        for (int q = 0; q < VEC; q += Elem<E>::VEC) unpack<E>(ld16_any(row + c + q), x + q);
    }
    template <typename E>
    __device__ __forceinline__ void put(E* row, const float* x) const {
        if (!in) return;
#pragma unroll
        for (int q = 0; q < VEC; q += Elem<E>::VEC) *(u32x4_any*)(row + c + q) = pack<E>(x + q);
    }
};
template <typename T>
struct Cols<T, false> {
    static constexpr int VEC = Elem<T>::VEC;
    static constexpr uint32_t ROWS = 4;          // a register for each of VEC values
    struct Row {
        T v[VEC];
    };
    int64_t c, N;
    __device__ __forceinline__ Cols(int64_t block, uint32_t lane, int64_t n) : c(block * 64 * VEC + lane), N(n) {}
    __device__ __forceinline__ int64_t at(int i) const { return min(c + 64 * i, N - 1); }
    __device__ __forceinline__ Row load(const T* row) const {
        Row r;
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = row[at(i)];
        return r;
    }
    static __device__ __forceinline__ void add(const Row& r, float* acc) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += (float)r.v[i];
    }
    template <typename E>
    __device__ __forceinline__ void get(const E* row, float* x) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = (float)row[at(i)];
    }
    template <typename E>
    __device__ __forceinline__ void put(E* row, const float* x) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + 64 * i < N) row[c + 64 * i] = (E)x[i];
    }
};
// f(true_type) where the wave's columns can go by vectors
template <int VEC, typename F>
__device__ __forceinline__ void with_cols(int64_t block, uint32_t N, F f) {
    if (N % VEC == 0 || (block + 1) * 64 * VEC <= N) f(std::true_type{});
    else f(std::false_type{});
}
// A row of dw: its sum, scaled, and what was there
template <typename COLS, typename W>
__device__ __forceinline__ void put_sum(const COLS& cols, W* row, float scale, float beta, const float* acc) {
    float x[COLS::VEC];
    if (beta != 0.0f) {
        cols.get(row, x);
#pragma unroll
        for (int i = 0; i < COLS::VEC; ++i) x[i] = beta * x[i] + scale * acc[i];
    } else {
#pragma unroll
        for (int i = 0; i < COLS::VEC; ++i) x[i] = scale * acc[i];
    }
    cols.put(row, x);
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// ---- few tokens
//
// A workgroup: every ranges-th row of dw (frequent tokens often have
// neighbouring ids), 64 x 16 bytes of dy's columns.  The ids of its rows are
// listed in order of m.  A row with up to HEAVY is a wave's, one with more all
// waves' on a part of the list each.  Rows without one are zeroed or scaled in
// all of their columns, by the workgroups of the same rows in turn.
// Against the sort and its launches (us, sorted / so): bf16 64 x 1000 x 512 11.1 / 6.6,
// 1024 x 32000 x 1024 18.1 / 17.7, 4096 x 32000 x 1024 24.1 / 22.8, 4096 x 500 x 512
// 16.7 / 12.7, fp32 1003 x 997 x 515 12.0 / 7.4, 4096 x 16000 x 1024 25.1 / 26.4; where
// few tokens fill the batch the sort is ahead, three in ten of 4096 the same 35 / 42,
// all of them 41 / 81.
constexpr uint32_t DIRECT = VKBLAS_EMBEDDING_SMALL, DTHREADS = 512, DWAVES = DTHREADS / 64;
constexpr uint32_t DROWS = 4096, HEAVY = 8;   // DROWS: the most rows of a workgroup
struct DirectParams {
    uint32_t M, V, N, ranges;
    const int64_t* ids;
    int64_t pad;
    const void* dy;
    int64_t lddy;
    void* dw;
    int64_t lddw;
    float scale, beta;
};
// acc += the rows of dy whose list entries a .. b - 1 are of row r
template <typename T, typename COLS>
__device__ __forceinline__ void add_listed(const DirectParams& p, const COLS& cols, const uint32_t* list, uint32_t a,
                                           uint32_t b, uint32_t r, float* acc) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t i = a; i < b; i += 64) {
        const uint32_t e = i + lane < b ? list[i + lane] : ~0u;
        uint64_t mask = __ballot(e / DIRECT == r);
        while (mask) {
            typename COLS::Row x[COLS::ROWS];
            const uint32_t n = (uint32_t)__popcll(mask);
#pragma unroll
            for (uint32_t k = 0; k < COLS::ROWS; ++k) {
                if (k >= n) continue;
                const int at = __builtin_ctzll(mask);
                mask &= mask - 1;
                const uint32_t m = (uint32_t)__builtin_amdgcn_readlane((int)e, at) % DIRECT;
                x[k] = cols.load((const T*)p.dy + (int64_t)m * p.lddy);
            }
#pragma unroll
            for (uint32_t k = 0; k < COLS::ROWS; ++k)
                if (k < n) COLS::add(x[k], acc);
        }
    }
}
template <typename T, typename W, uint32_t DSTEPS>
__global__ __launch_bounds__(DTHREADS) void direct_kernel(DirectParams p) {
    constexpr int VEC = Elem<T>::VEC, WV = Elem<W>::VEC;
    __shared__ uint32_t list[DSTEPS * DTHREADS];         // the workgroup's row times DIRECT, and m
    __shared__ uint32_t met[DROWS / 32], heavy[DROWS / 32], counts[DWAVES];
    __shared__ float sums[DWAVES - 1][64][VEC + 1];
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const uint32_t r0 = blockIdx.x, rows = (p.V - r0 + p.ranges - 1) / p.ranges;
    for (uint32_t i = threadIdx.x; i < (rows + 31) / 32; i += DTHREADS) met[i] = heavy[i] = 0;
    // a wave's ids are consecutive: DSTEPS times 64 of them
    const uint32_t first = wave * (DSTEPS * 64) + lane;
    uint32_t at[DSTEPS];
#pragma unroll
    for (uint32_t s = 0; s < DSTEPS; ++s) {
        const uint32_t m = first + s * 64;
        const int64_t id = m < p.M ? p.ids[m] : -1;
        const uint32_t v = id != p.pad && id >= 0 && id < p.V ? (uint32_t)id : p.V, r = v / p.ranges;
        at[s] = v < p.V && v - r * p.ranges == r0 ? r : ~0u;
    }
    uint32_t n = 0;
#pragma unroll
    for (uint32_t s = 0; s < DSTEPS; ++s) n += (uint32_t)__popcll(__ballot(at[s] != ~0u));
    if (lane == 0) counts[wave] = n;
    __syncthreads();
    uint32_t total = 0, base = 0;
    for (uint32_t w = 0; w < DWAVES; ++w) {
        if (w == wave) base = total;
        total += counts[w];
    }
#pragma unroll
    for (uint32_t s = 0; s < DSTEPS; ++s) {
        const uint64_t mask = __ballot(at[s] != ~0u);
        if (at[s] != ~0u) {
            list[base + __popcll(mask & ((1ull << lane) - 1))] = at[s] * DIRECT + first + s * 64;
            atomicOr(&met[at[s] / 32], 1u << at[s] % 32);
        }
        base += (uint32_t)__popcll(mask);
    }
    __syncthreads();
    total = uniform(total);
    W* dw = (W*)p.dw + (int64_t)r0 * p.lddw;
    const int64_t step = (int64_t)p.ranges * p.lddw;
    if (p.beta != 1.0f) {
        // as many waves to a row as it has 64 chunks
        const uint32_t per = min(DWAVES, (p.N + 64 * WV - 1) / (64 * WV)), at_once = DWAVES / per;
        const uint32_t mine = wave / per < at_once ? wave / per + blockIdx.y * at_once : rows;
        for (uint32_t r = mine; r < rows; r += gridDim.y * at_once) {
            if (uniform(met[r / 32]) >> r % 32 & 1) continue;
            W* row = dw + r * step;
            for (int64_t k = (int64_t)(wave % per * 64 + lane) * WV; k < p.N; k += per * 64 * WV) {
                u32x4 v = {0u, 0u, 0u, 0u};
                if (p.beta != 0.0f) {
                    float x[WV];
                    unpack<W>(ld_chunk(row, k, p.N), x);
#pragma unroll
                    for (int e = 0; e < WV; ++e) x[e] *= p.beta;
                    v = pack<W>(x);
                }
                st_chunk(row, k, p.N, v);
            }
        }
    }
    with_cols<VEC>(blockIdx.y, p.N, [&](auto vector) {
        const Cols<T, decltype(vector)::value> cols(blockIdx.y, lane, p.N);
        float acc[VEC];
        auto sum = [&](uint32_t r, uint32_t a, uint32_t b) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
            add_listed<T>(p, cols, list, a, b, r, acc);
        };
        bool any = false;
        for (uint32_t r = wave; r < rows; r += DWAVES) {
            if (!(uniform(met[r / 32]) >> r % 32 & 1)) continue;
            uint32_t of = 0;
            for (uint32_t i = 0; i < total; i += 64)
                of += (uint32_t)__popcll(__ballot(i + lane < total && list[i + lane] / DIRECT == r));
            if (of > HEAVY) {
                if (lane == 0) atomicOr(&heavy[r / 32], 1u << r % 32);
                any = true;
                continue;
            }
            sum(r, 0, total);
            put_sum(cols, dw + r * step, p.scale, p.beta, acc);
        }
        if (!__syncthreads_or(any)) return;
        const uint32_t each = (total + DWAVES - 1) / DWAVES, a = min(wave * each, total), b = min(a + each, total);
        for (uint32_t r = 0; r < rows; ++r) {
            if (!(uniform(heavy[r / 32]) >> r % 32 & 1)) continue;
            sum(r, a, b);
            if (wave) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) sums[wave - 1][lane][i] = acc[i];
            }
            __syncthreads();
            if (wave == 0) {
                for (uint32_t w = 0; w < DWAVES - 1; ++w)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[i] += sums[w][lane][i];
                put_sum(cols, dw + r * step, p.scale, p.beta, acc);
            }
            __syncthreads();
        }
    });
}

// ---- sorted tokens

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

// A wave: one chunk, 64 x 16 bytes of its rows' columns, ROWS of dy's rows in
// flight.  bf16 16384 x 4096 into a vocabulary of 128000: 63 us for 134 MB of dy and
// 70 MB of sums and parts, which leave after the zeros' 1 GB has gone through the
// caches.
template <typename T, typename W, typename COLS>
__device__ __forceinline__ void sum_chunk(const SumParams& p, const COLS& cols, uint32_t chunk) {
    constexpr int VEC = Elem<T>::VEC;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t p0 = chunk * p.chunk, p1 = p0 + min(p.chunk, p.M - p0);
    float acc[VEC];
    uint32_t now = ~0u;              // the token
    bool began = false;              // ... before this chunk
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    };
    float* part = p.part + (int64_t)chunk * 2 * p.N;
    clear();
    // VKB_EMBED_PAIRS pairs at a time in lanes 1 .. 62, the key before them and the one behind them beside
    for (uint32_t base = p0; base < p1; base += VKB_EMBED_PAIRS) {
        const uint32_t n = min(VKB_EMBED_PAIRS, p1 - base), at = min(base + lane, p.M) - (base + lane > 0 ? 1 : 0);
        const uint32_t keys = p.key[at], rows = p.order[min(at, p1 - 1)];
        auto key = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)keys, (int)(i + 1)); };
        if (base == p0) {
            now = key(0);
            began = p0 && key(-1) == now;
        }
        // the token ends before another one or the padding
        auto done = [&] {
            if (began) cols.put(part, acc);
            else put_sum(cols, (W*)p.dw + (int64_t)now * p.lddw, p.scale, p.beta, acc);
            clear();
            began = false;
        };
        for (uint32_t i = 0; i < n; i += COLS::ROWS) {
            if (now >= p.V) return;
            typename COLS::Row x[COLS::ROWS];
#pragma unroll
            for (uint32_t r = 0; r < COLS::ROWS; ++r) {
                const uint32_t m = (uint32_t)__builtin_amdgcn_readlane((int)rows, (int)min(i + r, n - 1) + 1);
                x[r] = cols.load((const T*)p.dy + (int64_t)m * p.lddy);
            }
#pragma unroll
            for (uint32_t r = 0; r < COLS::ROWS; ++r) {
                if (i + r >= n) continue;
                const uint32_t k = key(i + r);
                if (k != now) {
                    if (now < p.V) done();
                    now = k;
                }
                if (k < p.V) COLS::add(x[r], acc);
            }
        }
        if (base + n < p1 || now >= p.V) continue;
        // the last token: it ends here, or goes on
        if (p1 < p.M && key(n) == now) cols.put(began ? part : part + p.N, acc);
        else done();
    }
}
template <typename T, typename W>
__global__ __launch_bounds__(WORK) void sum_kernel(SumParams p) {
    const uint64_t unit = (uint64_t)blockIdx.x * (WORK / 64) + uniform(threadIdx.x >> 6);
    const uint32_t chunk = (uint32_t)(unit / p.blocks), block = (uint32_t)(unit % p.blocks);
    if (chunk >= p.chunks) return;
    with_cols<Elem<T>::VEC>(block, p.N, [&](auto vector) {
        const Cols<T, decltype(vector)::value> cols(block, threadIdx.x & 63, p.N);
        sum_chunk<T, W>(p, cols, chunk);
    });
}

// dw = beta * dw on the rows without a token: each wave searches the ids of
// FROWS rows among the sorted keys, a lane each, and takes its part of them.
constexpr uint32_t FROWS = 64;
template <typename W>
__global__ __launch_bounds__(WORK) void others_kernel(uint32_t M, uint32_t V, uint32_t N, const uint32_t* key, W* dw,
                                                      int64_t lddw, float beta) {
    constexpr int VEC = Elem<W>::VEC;
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    // as many waves to a row as it has 64 chunks
    const uint32_t per = min(WORK / 64, (N + 64 * VEC - 1) / (64 * VEC)), at_once = WORK / 64 / per;
    for (uint64_t v0 = (uint64_t)blockIdx.x * FROWS; v0 < V; v0 += (uint64_t)gridDim.x * FROWS) {
        const uint64_t v = v0 + lane;
        uint32_t lo = 0, hi = v < V ? M : 0;
        while (__any(lo < hi)) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const bool less = lo < hi && key[mid] < v;
            if (less) lo = mid + 1;
            else if (lo < hi) hi = mid;
        }
        const uint64_t mask = __ballot(v < V && !(lo < M && key[lo] == v));
        for (uint32_t r = wave / per; r < FROWS && wave / per < at_once; r += at_once) {
            if (!(mask >> r & 1)) continue;
            W* row = dw + (int64_t)(v0 + r) * lddw;
            for (int64_t k = (int64_t)(wave % per * 64 + lane) * VEC; k < N; k += per * 64 * VEC) {
                float f[VEC];
                unpack<W>(ld_chunk(row, k, N), f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] *= beta;
                st_chunk(row, k, N, pack<W>(f));
            }
        }
    }
}

// A token that begins in a chunk and goes on: that chunk's part and those of
// the chunks it fills, the waves on a quarter each, in order, JROWS in flight.
// (Eight waves: level, a token's 80 parts 3 us faster, 4000 workgroups with two
// parts or none each 4 us slower.)
constexpr uint32_t JTHREADS = 256, JWAVES = JTHREADS / 64, JROWS = 8, AHEAD = 4;
template <typename T, typename W>
__global__ __launch_bounds__(JTHREADS) void join_kernel(SumParams p) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ float sh[JWAVES - 1][64][VEC + 1];
    const uint32_t chunk = blockIdx.y, block = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const uint32_t p0 = chunk * p.chunk, p1 = p0 + p.chunk;      // the last chunk is not here
    const uint32_t k = p.key[p1 - 1];
    if (k >= p.V || p.key[p1] != k || (p0 && p.key[p0] == k && p.key[p0 - 1] == k)) return;
    // the last chunk whose first key is k, AHEAD chunks a lane at a time (by a binary search, a chain of
    // reads, 0.9 us more)
    uint32_t lo = chunk;
    for (uint32_t n = 64 * AHEAD; n == 64 * AHEAD; lo += n) {
        uint32_t first[AHEAD];
        n = 0;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t c = lo + 1 + i * 64 + lane;
            first[i] = p.key[min(c, p.chunks - 1) * p.chunk];
        }
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            n += (uint32_t)__popcll(__ballot(lo + 1 + i * 64 + lane < p.chunks && first[i] == k));
    }
    const uint32_t parts = lo - chunk + 1, each = (parts + JWAVES - 1) / JWAVES;
    const uint32_t a = min(wave * each, parts), b = min(a + each, parts);
    // part i: the tail of the first chunk, then the heads of the others
    auto row = [&](uint32_t i) { return p.part + ((int64_t)(chunk + i) * 2 + (i ? 0 : 1)) * p.N; };
    with_cols<VEC>(block, p.N, [&](auto vector) {
        const Cols<T, decltype(vector)::value> cols(block, lane, p.N);
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
        for (uint32_t i = a; i < b; i += JROWS) {
            float x[JROWS][VEC];
#pragma unroll
            for (uint32_t r = 0; r < JROWS; ++r)
                if (i + r < b) cols.get(row(i + r), x[r]);
#pragma unroll
            for (uint32_t r = 0; r < JROWS; ++r)
                if (i + r < b) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) acc[e] += x[r][e];
                }
        }
        if (wave) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sh[wave - 1][lane][i] = acc[i];
        }
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 0; w < (int)JWAVES - 1; ++w)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += sh[w][lane][i];
        put_sum(cols, (W*)p.dw + (int64_t)k * p.lddw, p.scale, p.beta, acc);
    });
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

// One chunk a thread, up to 2^22 workgroups
static uint32_t blocks_of(uint64_t chunks) {
    const uint64_t b = (chunks + WORK - 1) / WORK;
    return (uint32_t)(b < 1u << 22 ? b : 1u << 22);
}

extern "C" int vkb_launch_embedding(int type, int w_type, uint32_t M, uint32_t V, uint32_t N, const int64_t* ids,
                                    int64_t pad, const void* w, int64_t ldw, float scale, void* y, int64_t ldy,
                                    void* stream) {
    const bool ok = with_types(type, w_type, [&](auto t, auto o) {
        using T = decltype(t);
        using W = decltype(o);
        hipLaunchKernelGGL((lookup_kernel<T, W>), dim3(blocks_of((uint64_t)M * chunks_of<T>(N))), dim3(WORK), 0,
                           (hipStream_t)stream, M, V, N, ids, pad, (const W*)w, ldw, scale, (T*)y, ldy);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_direct(int type, int w_type, uint32_t M, uint32_t V, uint32_t N, const int64_t* ids,
                                           int64_t pad, const void* dy, int64_t lddy, float scale, void* dw,
                                           int64_t lddw, float beta, void* stream) {
    if (M > DIRECT) return (int)hipErrorInvalidValue;
    const uint32_t cols = 64 * (type == VKB_T_F32 ? 4 : 8), blocks = (N + cols - 1) / cols;
    // one wave of workgroups (us for 256 / 1024 / 4096: fp32 1003 x 997 x 515 9.9 / 9.0 /
    // 12.2, bf16 1024 x 32000 x 1024 35 / 17.8 / 23.6)
    uint64_t rows = ((uint64_t)V * blocks + 1023) / 1024;
    if (rows > DROWS) rows = DROWS;
    const uint64_t ranges = (V + rows - 1) / rows;
    if (ranges > 0xffffffffull / DTHREADS || blocks > 65535) return (int)hipErrorInvalidValue;
    const DirectParams p{M, V, N, (uint32_t)ranges, ids, pad, dy, lddy, dw, lddw, scale, beta};
    const bool ok = with_types(type, w_type, [&](auto t, auto o) {
        using T = decltype(t);
        using W = decltype(o);
        // half the steps for half the tokens: fp32 1003 x 997 x 515 9.1 -> 7.7 us
        if (M <= DIRECT / 2)
            hipLaunchKernelGGL((direct_kernel<T, W, DIRECT / 2 / DTHREADS>), dim3((uint32_t)ranges, blocks),
                               dim3(DTHREADS), 0, (hipStream_t)stream, p);
        else
            hipLaunchKernelGGL((direct_kernel<T, W, DIRECT / DTHREADS>), dim3((uint32_t)ranges, blocks),
                               dim3(DTHREADS), 0, (hipStream_t)stream, p);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_rank(uint32_t M, uint32_t V, const int64_t* ids, int64_t pad, uint32_t* key,
                                         uint32_t* order, int w_type, uint32_t N, void* dw, int64_t lddw,
                                         void* stream) {
    const uint32_t tiles = (uint32_t)(((uint64_t)M + RTOK - 1) / RTOK), ranks = tiles < 65536 ? tiles : 65536;
    const bool ok = with_type(w_type, [&](auto t) {
        using W = decltype(t);
        const uint32_t fill = dw ? blocks_of((uint64_t)V * chunks_of<W>(N)) : 0;
        hipLaunchKernelGGL((rank_kernel<W>), dim3(ranks + fill), dim3(WORK), 0, (hipStream_t)stream, M, V, ids, pad,
                           key, order, ranks, N, (W*)dw, lddw);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_merge_runs(uint32_t M, const uint32_t* key_in, const uint32_t* order_in,
                                               uint32_t* key, uint32_t* order, void* stream) {
    const uint32_t all = (uint32_t)(((uint64_t)M + WORK - 1) / WORK), blocks = all < 16384 ? all : 16384;
    if (M <= RUN * WAYS)
        hipLaunchKernelGGL((merge_runs_kernel<1>), dim3(blocks), dim3(MTHREADS), 0, (hipStream_t)stream, M, key_in,
                           order_in, key, order);
    else
        hipLaunchKernelGGL((merge_runs_kernel<4>), dim3(blocks), dim3(MTHREADS), 0, (hipStream_t)stream, M, key_in,
                           order_in, key, order);
    return (int)hipGetLastError();
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

extern "C" int vkb_launch_embedding_others(int w_type, uint32_t M, uint32_t V, uint32_t N, const uint32_t* key, void* dw,
                                           int64_t lddw, float beta, void* stream) {
    const bool ok = with_type(w_type, [&](auto t) {
        using W = decltype(t);
        const uint32_t b = (uint32_t)(((uint64_t)V + FROWS - 1) / FROWS);
        hipLaunchKernelGGL((others_kernel<W>), dim3(b < 1u << 20 ? b : 1u << 20), dim3(WORK), 0, (hipStream_t)stream, M,
                           V, N, key, (W*)dw, lddw, beta);
    });
    return ok ? (int)hipGetLastError() : (int)hipErrorInvalidValue;
}

extern "C" int vkb_launch_embedding_sums(int type, int w_type, const vkb_embedding_sums* a, void* stream) {
    const uint32_t cols = 64 * (type == VKB_T_F32 ? 4 : 8);
    SumParams p{a->M, a->V, a->N, a->chunk, a->chunks, (a->N + cols - 1) / cols, a->key, a->order, a->dy, a->lddy,
                a->dw, a->lddw, a->scale, a->beta, a->part};
    const uint64_t sums = ((uint64_t)p.chunks * p.blocks + WORK / 64 - 1) / (WORK / 64);
    if (sums > 0xffffffffull / WORK) return (int)hipErrorInvalidValue;
    int rc = (int)hipErrorInvalidValue;
    with_types(type, w_type, [&](auto t, auto o) {
        using T = decltype(t);
        using W = decltype(o);
        hipLaunchKernelGGL((sum_kernel<T, W>), dim3((uint32_t)sums), dim3(WORK), 0, (hipStream_t)stream, p);
        rc = (int)hipGetLastError();
        if (rc != 0 || p.chunks == 1) return;
        hipLaunchKernelGGL((join_kernel<T, W>), dim3(p.blocks, p.chunks - 1), dim3(JTHREADS), 0, (hipStream_t)stream,
                           p);
        rc = (int)hipGetLastError();
    });
    return rc;
}
