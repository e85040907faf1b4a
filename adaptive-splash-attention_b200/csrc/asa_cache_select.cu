// asa_cache_select.cu -- choosing the pages that a query reads, by a score from
// the pages' bounds.
//
// score(page) = max over the group's heads of
//     unit_q * 2^e * sum_c max(n_c upper_c, n_c lower_c),  n = rint(q / unit_q)
// -- an upper bound of n.k over the page's keys.  max(n u, n l) is n u for n > 0
// and n l for n < 0, so the sum is one product of 2 d int8 numbers a page with 2 d
// a row, on mma.m16n8k32 (16 pages x 8 heads).  It is of whole numbers below
// 2^24: the same in any order, and ties are exact.
//
// The keep-th largest key is found two bits at a time from the highest that any two
// keys differ in, by counting, with the keys in shared memory: no atomics, and nothing
// depends on how scores cluster (a radix histogram's bins are hit by all threads at
// once, scores of one sign and size sharing their upper bits).
//
// Steps that wait for one another bound it, not bytes (2 d + 4 a page and key head):
// 6.7 us for 64 pages of 8 key heads, of which a launch is 2; 13.3 for 1024, 51.7 for 64
// sequences of 1024 (139 MB, 2.7 TB/s).
#include "asa_cache.h"

namespace asa {
namespace cache {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kShared = 4096;         // pages whose keys fit in shared memory
constexpr int kChunk = 256;           // pages a CTA of score_kernel scores

// Larger floats as larger integers; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float f) {
    if (f != f) return 0u;
    const uint32_t b = f == 0.0f ? 0u : __float_as_uint(f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Query {
    Shape s;
    const __nv_bfloat16* Q;
    Strides qs;
    const int8_t* bounds;
    const int32_t* table;
    const int32_t* lengths;
    int keep;
    int* err;
};

// The pages that query t of sequence b can see, its own last.
__device__ __forceinline__ int pages_seen(const Query& a, int b, int t) {
    const long long pos = min((long long)__ldg(a.lengths + b) - a.s.T + t, (long long)a.s.width * a.s.P - 1);
    return pos < 0 ? 0 : (int)(pos / a.s.P) + 1;
}

// A query's whole numbers for one key head, heads rounded up to eights: upper parts
// (max(n, 0)), then lower ones, and the units.
template <int D>
__device__ __forceinline__ void make_query(const Query& a, int b, int t, int h, int8_t* s_q, float* s_unit) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int heads = (a.s.G + 7) & ~7;
    for (int g = warp; g < heads; g += warps) {
        const __nv_bfloat16* src = a.Q + b * a.qs.b + t * a.qs.t + (int64_t)(h * a.s.G + g) * a.qs.h;
        float x[D / 32], big = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = g < a.s.G ? __bfloat162float(src[lane + 32 * i]) : 0.0f;
            big = fmaxf(big, fabsf(x[i]));
            bad |= x[i] != x[i];
        }
        big = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(big)));
        const float unit = __any_sync(~0u, bad) ? NAN : __fmul_rn(big, k127th);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int n = unit > 0.0f ? (int)rintf(__fdiv_rn(x[i], unit)) : 0;
            s_q[g * 2 * D + lane + 32 * i] = (int8_t)max(n, 0);
            s_q[g * 2 * D + D + lane + 32 * i] = (int8_t)min(n, 0);
        }
        if (lane == 0) s_unit[g] = unit;
    }
}

// The ids of the pages of the table that a lane scores: p0 + r and p0 + r + 8.
__device__ __forceinline__ void look_up(const Query& a, int b, int p0, int to, int (&next)[2]) {
    const int r = (threadIdx.x & 31) >> 2;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int page = p0 + r + 8 * e;
        next[e] = page < to ? __ldg(a.table + (int64_t)b * a.s.width + page) : -1;
    }
}

// Keys of pages from .. to - 1 (ordered scores; put(page, key, whether earlier heads had a say)) by
// the warps of a CTA, 16 pages each; `first`: the ids of a lane's first two.
template <int D, typename Put>
__device__ __forceinline__ void score_pages(const Query& a, int b, int h, int from, int to, int warps, const int8_t* s_q,
                                            const float* s_unit, const int (&first)[2], Put put) {
    constexpr int SEG = 2 * D / 64;                   // 64-byte stretches of a page's bounds
    const Shape& s = a.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q4 = lane & 3;
    for (int tile = 0; tile * 8 < s.G; ++tile) {
        uint4 w[SEG];
#pragma unroll
        for (int k = 0; k < SEG; ++k)
            w[k] = *reinterpret_cast<const uint4*>(s_q + (8 * tile + r) * 2 * D + 64 * k + 16 * q4);
        const float u0 = s_unit[8 * tile + 2 * q4], u1 = s_unit[8 * tile + 2 * q4 + 1];
        const bool in0 = 8 * tile + 2 * q4 < s.G, in1 = 8 * tile + 2 * q4 + 1 < s.G;
        int next[2] = {first[0], first[1]};           // the pages' ids, looked up an iteration ahead
        if (tile) look_up(a, b, from + 16 * warp, to, next);
        for (int p0 = from + 16 * warp; p0 < to; p0 += 16 * warps) {
            const int8_t* rec[2];
            float scale[2];
            uint4 x[2][SEG];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int id = p0 + r + 8 * e < to ? next[e] : -1;
                rec[e] = nullptr;
                scale[e] = 0.0f;
                if (id >= 0 && id < s.pages) rec[e] = a.bounds + ((int64_t)id * s.H + h) * bounds_bytes(D);
                else if (p0 + r + 8 * e < to && q4 == 0 && a.err) atomicCAS(a.err, 0, ASA_ERR_INVALID);
#pragma unroll
                for (int k = 0; k < SEG; ++k)
                    x[e][k] = rec[e] ? __ldg(reinterpret_cast<const uint4*>(rec[e] + 64 * k + 16 * q4)) : make_uint4(0u, 0u, 0u, 0u);
                if (rec[e]) scale[e] = __int_as_float((min(max(__ldg(reinterpret_cast<const int*>(rec[e] + 2 * D)), -126), 127) + 127) << 23);
            }
            look_up(a, b, p0 + 16 * warps, to, next);
            int acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < SEG; ++k) {
                mma_s8(acc, x[0][k].x, x[1][k].x, x[0][k].y, x[1][k].y, w[k].x, w[k].y);
                mma_s8(acc, x[0][k].z, x[1][k].z, x[0][k].w, x[1][k].w, w[k].z, w[k].w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t key = 0u;
                if (in0) key = ordered(__fmul_rn(__fmul_rn((float)acc[2 * e], scale[e]), u0));
                if (in1) key = max(key, ordered(__fmul_rn(__fmul_rn((float)acc[2 * e + 1], scale[e]), u1)));
                key = max(key, __shfl_xor_sync(~0u, key, 1));
                key = max(key, __shfl_xor_sync(~0u, key, 2));
                const int page = p0 + r + 8 * e;
                if (q4 == 0 && page < to) put(page, rec[e] ? key : 0u, tile > 0);
            }
        }
    }
}

// Keys of an item's pages, kChunk a CTA.
template <int D>
__global__ void __launch_bounds__(256) score_kernel(const __grid_constant__ Query a, uint32_t* __restrict__ keys, int chunks) {
    follow();
    const int item = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const int h = item % a.s.H, bt = item / a.s.H, t = bt % a.s.T, b = bt / a.s.T;
    uint32_t* key = keys + (int64_t)item * a.s.width;
    extern __shared__ __align__(16) int8_t s_q[];
    float* s_unit = reinterpret_cast<float*>(s_q + ((a.s.G + 7) & ~7) * 2 * D);
    int first[2];                                     // (its load and the query's do not wait for the length)
    look_up(a, b, chunk * kChunk + 16 * (threadIdx.x >> 5), a.s.width, first);
    const int n = pages_seen(a, b, t);
    make_query<D>(a, b, t, h, s_q, s_unit);
    __syncthreads();
    if (n <= a.keep) return;
    score_pages<D>(a, b, h, chunk * kChunk, min((chunk + 1) * kChunk, n - 1), 8, s_q, s_unit, first,
                   [&](int page, uint32_t k, bool more) { key[page] = more ? max(key[page], k) : k; });
}

// The bits in which a CTA's keys differ (0: none do), and a key: from each warp's.
__device__ __forceinline__ uint32_t cta_differ(uint32_t any, uint32_t all, uint32_t* slot, uint32_t* common) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slot[warp] = any, slot[kWarps + warp] = all;
    __syncthreads();
    any = __reduce_or_sync(~0u, lane < kWarps ? slot[lane] : 0u);
    all = __reduce_and_sync(~0u, lane < kWarps ? slot[kWarps + lane] : ~0u);
    *common = all;
    return any & ~all;
}

// Sum of a number a warp over the CTA, and over the warps before this one.  One
// barrier; `slot` must not be written again before another.
__device__ __forceinline__ int cta_sum(int v, int* slot, int* before = nullptr) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slot[warp] = v;
    __syncthreads();
    const int of = lane < kWarps ? slot[lane] : 0;
    if (before) *before = __reduce_add_sync(~0u, lane < warp ? of : 0);
    return __reduce_add_sync(~0u, of);
}

// One CTA a (query, key head): its keys (scored here, or read back), the edge between taken and left, and the taken pages in ascending order.
template <int D, bool SCORE>
__global__ void __launch_bounds__(kThreads) pick_kernel(const __grid_constant__ Query a, const uint32_t* __restrict__ keys,
                                                        int32_t* __restrict__ pages) {
    extern __shared__ __align__(16) int8_t s_q[];    // the query, its units, the keys
    __shared__ int s_count[2][kWarps];
    __shared__ uint32_t s_bits[2 * kWarps];
    __shared__ int4 s_three[2][kWarps];
    float* s_unit = reinterpret_cast<float*>(s_q + ((a.s.G + 7) & ~7) * 2 * D);
    uint32_t* s_key = reinterpret_cast<uint32_t*>(s_unit + ((a.s.G + 7) & ~7));
    const Shape& s = a.s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, keep = a.keep;
    follow();
    const int h = blockIdx.x % s.H, bt = blockIdx.x / s.H, t = bt % s.T, b = bt / s.T;
    int32_t* out = pages + (int64_t)blockIdx.x * keep;
    int first[2];                                     // (its load and the query's do not wait for the length)
    if constexpr (SCORE) look_up(a, b, 16 * warp, s.width, first);
    const int n = pages_seen(a, b, t);
    if constexpr (SCORE) make_query<D>(a, b, t, h, s_q, s_unit);
    if (n <= keep) {
        for (int i = tid; i < keep; i += kThreads) out[i] = i < n ? i : -1;
        return;
    }
    const int m = n - 1;                              // those that are weighed; the query's own is taken
    const uint32_t* key = keys + (int64_t)blockIdx.x * s.width;
    if constexpr (SCORE) {
        __syncthreads();
        score_pages<D>(a, b, h, 0, m, kWarps, s_q, s_unit, first,
                       [&](int page, uint32_t k, bool more) { s_key[page] = more ? max(s_key[page], k) : k; });
    } else if (m <= kShared) {
        s_key = reinterpret_cast<uint32_t*>(s_q);
        for (int i = tid; i < m; i += kThreads) s_key[i] = __ldg(key + i);
    }
    if (SCORE || m <= kShared) key = s_key;
    __syncthreads();
    // The largest number that `need` keys reach: the bits that all keys share, then two
    // bits a step, by the counts of keys that reach each of the three numbers.
    const int need = keep - 1;
    uint32_t edge = 0;
    int above = m;                                    // keys that reach it
    int turn = 0;
    if (need == 0) {
        edge = ~0u, above = -1;                       // (none is taken)
    } else {
        uint32_t any = 0u, every = ~0u;
        for (int i = tid; i < m; i += kThreads) any |= key[i], every &= key[i];
        const uint32_t differ = cta_differ(__reduce_or_sync(~0u, any), __reduce_and_sync(~0u, every), s_bits, &edge);
        int bit = differ ? (31 - __clz(differ)) & ~1 : -1;
        if (bit >= 0) edge &= bit == 30 ? 0u : ~0u << (bit + 2);
        for (; bit >= 0 && above != need; bit -= 2, turn ^= 1) {
            const uint32_t t1 = edge | 1u << bit, t2 = edge | 2u << bit, t3 = edge | 3u << bit;
            int n1 = 0, n2 = 0, n3 = 0;
            for (int i = tid; i < m; i += kThreads) {
                const uint32_t k = key[i];
                n1 += k >= t1, n2 += k >= t2, n3 += k >= t3;
            }
            n1 = __reduce_add_sync(~0u, n1), n2 = __reduce_add_sync(~0u, n2), n3 = __reduce_add_sync(~0u, n3);
            if (lane == 0) s_three[turn][warp] = make_int4(n1, n2, n3, 0);
            __syncthreads();
            const int4 of = lane < kWarps ? s_three[turn][lane] : make_int4(0, 0, 0, 0);
            n1 = __reduce_add_sync(~0u, of.x), n2 = __reduce_add_sync(~0u, of.y), n3 = __reduce_add_sync(~0u, of.z);
            if (n3 >= need) edge = t3, above = n3;
            else if (n2 >= need) edge = t2, above = n2;
            else if (n1 >= need) edge = t1, above = n1;
        }
    }
    // Keys beyond the edge are taken, and of those on it the first; where exactly
    // `need` reach it, all are.
    int before = 0, tied = 0, ties = 0;
    const bool all = above == need;
    if (!all && need) {
        int count = 0;
        for (int i = tid; i < m; i += kThreads) count += key[i] > edge;
        ties = need - cta_sum(__reduce_add_sync(~0u, count), s_count[turn]);
        turn ^= 1;
    }
    for (int base = 0; base < m; base += kThreads) {
        const int i = base + tid;
        const uint32_t k = i < m ? key[i] : 0u;
        bool take = i < m && need && (all ? k >= edge : k > edge);
        if (ties) {                                   // (the same in all threads)
            const bool tie = i < m && k == edge;
            const uint32_t votes = __ballot_sync(~0u, tie);
            int rank;
            const int sum = cta_sum(__popc(votes), s_count[turn], &rank);
            turn ^= 1;
            rank += tied + __popc(votes & ((1u << lane) - 1u));
            tied += sum;
            take |= tie && rank < ties;
        }
        const uint32_t votes = __ballot_sync(~0u, take);
        int at;
        const int sum = cta_sum(__popc(votes), s_count[turn], &at);
        turn ^= 1;
        if (take) out[before + at + __popc(votes & ((1u << lane) - 1u))] = i;
        before += sum;
    }
    if (tid == 0) out[keep - 1] = m;
}

// One launch where the tables are short, or the items fill the SMs; else the pages are
// scored by CTAs of their own first.  Us in one launch and in two, 8 key heads: 1 sequence
// of 512 pages 11.0, 11.9, of 1024 15.3, 13.3, of 4096 39.9, 18.7; 37 (296 items) of 512
// 19.2, 24.7; 64 of 1024 51.7, 61.1.
bool scores_itself(const Shape& s) {
    return s.width <= 512 || (s.width <= kShared && (int64_t)s.B * s.T * s.H >= 296);
}

template <int D>
cudaError_t select_as(const Query& a, int32_t* pages, void* ws, cudaStream_t st) {
    const unsigned items = (unsigned)(a.s.B * a.s.T * a.s.H);
    const size_t query = (size_t)((a.s.G + 7) & ~7) * (2 * D + 4) /* 67 KB at most */, keys = (size_t)a.s.width * 4;
    if (scores_itself(a.s)) {
        if (query + keys > 48 * 1024) {
            static Allowed allowed;
            const cudaError_t e = allow_shared(pick_kernel<D, true>, 116 * 1024, allowed);
            if (e != cudaSuccess) return e;
        }
        return launch(pick_kernel<D, true>, items, kThreads, query + keys, st, a, (const uint32_t*)nullptr, pages);
    }
    const int chunks = (a.s.width + kChunk - 1) / kChunk;
    if ((int64_t)items * chunks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    if (query > 48 * 1024) {
        static Allowed allowed;
        const cudaError_t e = allow_shared(score_kernel<D>, 100 * 1024, allowed);
        if (e != cudaSuccess) return e;
    }
    const cudaError_t e = launch(score_kernel<D>, items * chunks, 256, query, st, a, (uint32_t*)ws, chunks);
    return e != cudaSuccess ? e : launch(pick_kernel<D, false>, items, kThreads, keys < kShared * 4 ? keys : kShared * 4, st, a,
                                         (const uint32_t*)ws, pages);
}

}  // namespace

size_t select_workspace(const Shape& s) {
    return scores_itself(s) ? 0 : ((size_t)s.B * s.T * s.H * s.width * 4 + 15) & ~size_t(15);
}

cudaError_t select(const Shape& s, const void* Q, Strides qs, const int8_t* bounds, const int32_t* table,
                   const int32_t* lengths, int keep, int32_t* pages, void* ws, int* err, cudaStream_t st) {
    const Query a{s, (const __nv_bfloat16*)Q, qs, bounds, table, lengths, keep, err};
    switch (s.d) {
        case 32: return select_as<32>(a, pages, ws, st);
        case 64: return select_as<64>(a, pages, ws, st);
        case 96: return select_as<96>(a, pages, ws, st);
        default: return select_as<128>(a, pages, ws, st);
    }
}

}  // namespace cache
}  // namespace asa
