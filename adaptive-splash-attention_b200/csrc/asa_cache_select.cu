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
// The keep-th largest key is found bit by bit from the top by counting, with the
// keys in shared memory: no atomics, and nothing depends on how scores cluster
// (a radix histogram's bins are hit by all threads at once, scores of one sign and
// size sharing their upper bits).
#include "asa_cache.h"

namespace asa {
namespace cache {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kShared = 4096;         // pages whose keys fit in shared memory
constexpr int kChunk = 512;           // pages a CTA of score_kernel scores

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
    int vec;                          // q rows may be read 16 bytes at a time
    int* err;
};

// The pages that query t of sequence b can see, its own last.
__device__ __forceinline__ int pages_seen(const Query& a, int b, int t) {
    const long long pos = min((long long)__ldg(a.lengths + b) - a.s.T + t, (long long)a.s.width * a.s.P - 1);
    return pos < 0 ? 0 : (int)(pos / a.s.P) + 1;
}

// Keys of pages from .. to - 1 (ordered scores; put(page, key)) by the warps of a CTA, 16 pages each.
template <int D, typename Put>
__device__ __forceinline__ void score_pages(const Query& a, int b, int t, int h, int from, int to, int warps, Put put) {
    constexpr int SEG = 2 * D / 64;                   // 64-byte stretches of a page's bounds
    const Shape& s = a.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q4 = lane & 3;
    if (from + 16 * warp >= to) return;
    for (int tile = 0; tile * 8 < s.G; ++tile) {
        // the lane's part of head 8 tile + r: channels 16 q4 .. + 15 of each stretch, whole numbers
        const int g = 8 * tile + r;
        uint32_t raw[SEG][8], w[SEG][4];
        float big = 0.0f;
        bool bad = false;
        const __nv_bfloat16* src = a.Q + b * a.qs.b + t * a.qs.t + (int64_t)(h * s.G + g) * a.qs.h;
#pragma unroll
        for (int k = 0; k < SEG; ++k) {               // (the lower codes' stretches have the upper ones' channels)
            const uint16_t* e = reinterpret_cast<const uint16_t*>(src + (64 * k + 16 * q4) % D);
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[k][i] = 0u;
            if (g < s.G && a.vec) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(e) + i);
                    raw[k][4 * i] = v.x, raw[k][4 * i + 1] = v.y, raw[k][4 * i + 2] = v.z, raw[k][4 * i + 3] = v.w;
                }
            } else if (g < s.G) {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[k][i] = __ldg(e + 2 * i) | (uint32_t)__ldg(e + 2 * i + 1) << 16;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = __uint_as_float(raw[k][i] << 16), y = __uint_as_float(raw[k][i] & 0xffff0000u);
                big = fmaxf(big, fmaxf(fabsf(x), fabsf(y)));
                bad |= x != x || y != y;
            }
        }
        big = fmaxf(big, __shfl_xor_sync(~0u, big, 1));
        big = fmaxf(big, __shfl_xor_sync(~0u, big, 2));
        const bool row_bad = (__ballot_sync(~0u, bad) >> (lane & 28)) & 15u;
        const float unit = row_bad ? NAN : __fmul_rn(big, k127th);
#pragma unroll
        for (int k = 0; k < SEG; ++k) {
            const bool upper = 64 * k + 16 * q4 < D;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t word = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t two = raw[k][2 * j + i / 2];
                    const float x = __uint_as_float(i & 1 ? two & 0xffff0000u : two << 16);
                    const int n = unit > 0.0f ? (int)rintf(__fdiv_rn(x, unit)) : 0;
                    word |= (uint32_t)((upper ? max(n, 0) : min(n, 0)) & 255) << (8 * i);
                }
                w[k][j] = word;
            }
        }
        const float u0 = __shfl_sync(~0u, unit, 8 * q4), u1 = __shfl_sync(~0u, unit, 8 * q4 + 4);
        const bool in0 = 8 * tile + 2 * q4 < s.G, in1 = 8 * tile + 2 * q4 + 1 < s.G;
        for (int p0 = from + 16 * warp; p0 < to; p0 += 16 * warps) {
            const int8_t* rec[2];
            float scale[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int page = p0 + r + 8 * e;
                const int id = page < to ? __ldg(a.table + (int64_t)b * s.width + page) : -1;
                rec[e] = nullptr;
                scale[e] = 0.0f;
                if (id >= 0 && id < s.pages) rec[e] = a.bounds + ((int64_t)id * s.H + h) * bounds_bytes(D);
                else if (page < to && q4 == 0 && a.err) atomicCAS(a.err, 0, ASA_ERR_INVALID);
                if (rec[e]) scale[e] = __int_as_float((min(max(__ldg(reinterpret_cast<const int*>(rec[e] + 2 * D)), -126), 127) + 127) << 23);
            }
            int acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < SEG; ++k) {
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                const uint4 x = rec[0] ? __ldg(reinterpret_cast<const uint4*>(rec[0] + 64 * k + 16 * q4)) : zero;
                const uint4 y = rec[1] ? __ldg(reinterpret_cast<const uint4*>(rec[1] + 64 * k + 16 * q4)) : zero;
                mma_s8(acc, x.x, y.x, x.y, y.y, w[k][0], w[k][1]);
                mma_s8(acc, x.z, y.z, x.w, y.w, w[k][2], w[k][3]);
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

// Keys of an item's pages, kChunk a CTA, for items whose keys do not fit in shared memory.
template <int D>
__global__ void __launch_bounds__(256) score_kernel(const __grid_constant__ Query a, uint32_t* __restrict__ keys, int chunks) {
    const int item = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const int h = item % a.s.H, bt = item / a.s.H, t = bt % a.s.T, b = bt / a.s.T;
    const int n = pages_seen(a, b, t);
    if (n <= a.keep) return;
    uint32_t* key = keys + (int64_t)item * a.s.width;
    score_pages<D>(a, b, t, h, chunk * kChunk, min((chunk + 1) * kChunk, n - 1), 8, [&](int page, uint32_t k, bool more) {
        key[page] = more ? max(key[page], k) : k;
    });
}

// One CTA a (query, key head): its keys (scored here, where they fit in shared
// memory), the edge between taken and left, and the taken pages in ascending order.
template <int D, bool SHARED>
__global__ void __launch_bounds__(kThreads) pick_kernel(const __grid_constant__ Query a, const uint32_t* __restrict__ keys,
                                                        int32_t* __restrict__ pages) {
    extern __shared__ uint32_t s_key[];
    __shared__ int s_count[2][kWarps];
    const Shape& s = a.s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, keep = a.keep;
    const int h = blockIdx.x % s.H, bt = blockIdx.x / s.H, t = bt % s.T, b = bt / s.T;
    int32_t* out = pages + (int64_t)blockIdx.x * keep;
    const int n = pages_seen(a, b, t);
    if (n <= keep) {
        for (int i = tid; i < keep; i += kThreads) out[i] = i < n ? i : -1;
        return;
    }
    const int m = n - 1;                              // those that are weighed; the query's own is taken
    if constexpr (SHARED) {
        score_pages<D>(a, b, t, h, 0, m, kWarps, [&](int page, uint32_t k, bool more) {
            s_key[page] = more ? max(s_key[page], k) : k;
        });
        __syncthreads();
    }
    const uint32_t* key = SHARED ? s_key : keys + (int64_t)blockIdx.x * s.width;
    // the largest number that `need` keys reach
    const int need = keep - 1;
    uint32_t edge = 0;
    int above = m;                                    // keys that reach it
    if (need == 0) edge = ~0u, above = -1;            // (none is taken)
    for (int bit = 31, turn = 0; bit >= 0 && above != need && need; --bit, turn ^= 1) {
        const uint32_t next = edge | 1u << bit;
        int count = 0;
        for (int i = tid; i < m; i += kThreads) count += key[i] >= next;
        count = __reduce_add_sync(~0u, count);
        if (lane == 0) s_count[turn][warp] = count;
        __syncthreads();
        count = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) count += s_count[turn][w];
        if (count >= need) edge = next, above = count;
    }
    __syncthreads();
    // Keys beyond the edge are taken, and of those on it the first; where exactly
    // `need` reach it, all are.
    int before = 0, tied = 0, ties = 0;
    const bool all = above == need;
    if (!all && need) {
        int count = 0;
        for (int i = tid; i < m; i += kThreads) count += key[i] > edge;
        count = __reduce_add_sync(~0u, count);
        if (lane == 0) s_count[0][warp] = count;
        __syncthreads();
        ties = need;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) ties -= s_count[0][w];
        __syncthreads();
    }
    for (int base = 0; base < m; base += kThreads) {
        const int i = base + tid;
        const uint32_t k = i < m ? key[i] : 0u;
        bool take = i < m && need && (all ? k >= edge : k > edge);
        if (ties) {                                   // (the same in all threads)
            const bool tie = i < m && k == edge;
            const uint32_t votes = __ballot_sync(~0u, tie);
            if (lane == 0) s_count[0][warp] = __popc(votes);
            __syncthreads();
            int rank = tied + __popc(votes & ((1u << lane) - 1u));
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                rank += w < warp ? s_count[0][w] : 0;
                tied += s_count[0][w];
            }
            take |= tie && rank < ties;
        }
        const uint32_t votes = __ballot_sync(~0u, take);
        if (lane == 0) s_count[1][warp] = __popc(votes);
        __syncthreads();
        int at = before + __popc(votes & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            at += w < warp ? s_count[1][w] : 0;
            before += s_count[1][w];
        }
        if (take) out[at] = i;
        __syncthreads();
    }
    if (tid == 0) out[keep - 1] = m;
}

template <int D>
cudaError_t select_as(const Query& a, int32_t* pages, void* ws, cudaStream_t st) {
    const unsigned items = (unsigned)(a.s.B * a.s.T * a.s.H);
    if (a.s.width <= kShared) {
        pick_kernel<D, true><<<items, kThreads, (size_t)a.s.width * 4, st>>>(a, nullptr, pages);
    } else {
        const int chunks = (a.s.width + kChunk - 1) / kChunk;
        if ((int64_t)items * chunks > 0x7fffffff) return cudaErrorInvalidConfiguration;
        score_kernel<D><<<items * chunks, 256, 0, st>>>(a, (uint32_t*)ws, chunks);
        note_launch();
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        pick_kernel<D, false><<<items, kThreads, 0, st>>>(a, (const uint32_t*)ws, pages);
    }
    note_launch();
    return cudaGetLastError();
}

}  // namespace

size_t select_workspace(const Shape& s) {
    const size_t keys = s.width <= kShared ? 0 : (size_t)s.B * s.T * s.H * s.width * 4;
    return (keys + 16 + 15) & ~size_t(15);
}

cudaError_t select(const Shape& s, const void* Q, Strides qs, const int8_t* bounds, const int32_t* table,
                   const int32_t* lengths, int keep, int32_t* pages, void* ws, int* err, cudaStream_t st) {
    const int vec = (reinterpret_cast<uintptr_t>(Q) & 15) == 0 && qs.b % 8 == 0 && qs.t % 8 == 0 && qs.h % 8 == 0;
    const Query a{s, (const __nv_bfloat16*)Q, qs, bounds, table, lengths, keep, vec, err};
    switch (s.d) {
        case 32: return select_as<32>(a, pages, ws, st);
        case 64: return select_as<64>(a, pages, ws, st);
        case 96: return select_as<96>(a, pages, ws, st);
        default: return select_as<128>(a, pages, ws, st);
    }
}

}  // namespace cache
}  // namespace asa
