// asa_cache_attend.cuh -- what the cache's attention kernels share: how a call's
// work is cut (Plan), the workspace, and the joining of what was cut.
#pragma once
#include "asa_cache.h"
#include "asa_sm100.cuh"

namespace asa {
namespace cache {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Weights are powers of two of a score over its row's reference.  A reference is set
// so that the row's largest weight is 2^kTop, and stays until one would pass
// 2^kMost: fp16 holds 65504, and keeps 11 bits of weights down to 2^-14.
constexpr float kTop = 4.0f, kMost = 14.5f;
constexpr float kLow = -1.0e30f;      // below any score
// The most that the factor of a row's products may be (they count 2^-24, at most 2^13; in asa_cache_chunk.cu
// 1, at most 2^34, and 2^-24 of this factor): scores stay within 2^93, less than -kLow.  Queries of some 1e22
// and more, by the scale, would have a larger one, which fp32 need not hold (it made NaN of them); with either
// the largest score takes all, a code's step in such a query's largest channel being 2^40 and more.
constexpr float kMostFactor = 1.2089258e24f;          // 2^80
__device__ __forceinline__ float factor_of(float scale, int e, float most) {
    return fminf(fmaxf(scalbnf(scale, e), -most), most);
}
constexpr int kSms = 148;

// How a call's rows are tiled and its work cut.
struct Plan {
    int U, R, tiles;                  // units of rows (sequences; with lists, query tokens), rows each, tiles each
    int keep;                         // pages listed a query and key head (0: all of the table)
    int cap;                          // tiles an item can have at most
    int split;                        // items are cut into equal runs (else one cluster an item)
    int cluster;                      // CTAs of an item's cluster
    int values;                       // entmax: such CTAs for the values, where only the scores are cut (else 0)
    int vec;                          // q rows may be read 16 bytes at a time
    int page_shift;                   // log2 of the blocks of a page
    int tile;                         // tokens of a tile
    int item_cost;                    // what starting an item costs, in tiles of one CTA
    int least;                        // tiles a run has at least
};

// The workspace: [run length | prefix per unit | partials | scores, tile maxima, thresholds]
struct Space {
    int64_t* run;                     // [1 + U]
    float* part;                      // [2 * CTAs][rows][D]
    float* part_ml;                   // [2 * CTAs][2][rows]
    float4* score;                    // [items][cap][2][NT][32]
    float* top;                       // [items][cap][8 NT]
    float* tau;                       // [items][8 NT] at or just below the thresholds: by these tiles are chosen
    float2* edge;                     // [items][8 NT] a row's largest x, and its threshold relative to that
};

struct Args {
    Shape s;
    Plan p;
    Space w;
    Strides qs;
    const __nv_bfloat16* Q;
    const uint8_t* pool;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* list;
    __nv_bfloat16* O;
    int* err;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }   // e in -126..127

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar)) : "memory");
}
// Bounded wait for a phase, in naps of up to 20 us: a warp that waits takes few issue
// slots from those that work.  An error word set by something else than a wait that
// gave up (a page outside the pool) does not cut it short.
__device__ __forceinline__ bool nap(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(sm100::smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity, int naps, int* err) {
    if (nap(bar, parity)) return true;
    for (int i = naps; i > 0; --i) {
        if (nap(bar, parity)) return true;
        if (err && *reinterpret_cast<volatile int*>(err) == ASA_ERR_DEVICE_TIMEOUT) return false;
    }
    if (err) atomicExch(err, ASA_ERR_DEVICE_TIMEOUT);
    return false;
}

// After a wait gave up: waits for the phase that a barrier is in, a third of a second at most (it may not
// have been armed).
__device__ __forceinline__ void drain(uint64_t* bar) {
    const uint32_t parity = sm100::mbar_test(bar, 0) ? 1u : 0u;
    for (int i = 0; i < (1 << 14); ++i)
        if (nap(bar, parity)) return;
}
// Whether a wait of the cache's kernels has given up.
__device__ __forceinline__ bool timed_out(const int* err) {
    return err && *reinterpret_cast<const volatile int*>(err) == ASA_ERR_DEVICE_TIMEOUT;
}

__device__ __forceinline__ int unit_tiles(const Args& a, int u) {
    if (a.list) return a.p.cap;
    const long long n = min((long long)max(__ldg(a.lengths + u), 0), (long long)a.s.width * a.s.P);
    return (int)((n + a.p.tile - 1) / a.p.tile);
}

// Exclusive prefix of one value a thread over the CTA; *total to all.
template <int NTHR>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s_warp, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const int64_t y = __shfl_up_sync(~0u, x, k);
        if (lane >= k) x += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NTHR / 32; ++w) {
        if (w < warp) before += s_warp[w];
        sum += s_warp[w];
    }
    *total = sum;
    return before + x - v;
}

// ---- joining an item that several CTAs walked -------------------------------------
// A CTA K rows: its W warps take the parts in turn, a lane four channels of each row,
// and keep a running reference a row, as the walk does.  Few rows have many parts
// (the few items of long contexts), many rows few (the 128 of a prompt's chunk).
template <int D, int ROWS, int K, int W>
__global__ void __launch_bounds__(32 * W) combine_kernel(const __grid_constant__ Args a) {
    constexpr int U = K >= 4 ? 1 : 4;                 // parts of a warp whose loads are under way at once
    __shared__ float2 s_ml[W][K];
    __shared__ float4 s_acc[W][K][D / 4];
    follow();
    const Shape& s = a.s;
    const int per = a.p.tiles * s.H, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = (int)(blockIdx.x % (ROWS / K)) * K, item_no = blockIdx.x / (ROWS / K);
    const int u = item_no / per, item = item_no % per, h = item / a.p.tiles, tile = item % a.p.tiles;
    if (tile * ROWS + row0 >= a.p.R) return;
    const int of = unit_tiles(a, u);
    float m[K], l[K];
    float4 acc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) m[k] = kLow, l[k] = 0.0f, acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (of) {
        const int64_t run = a.w.run[0], x0 = a.w.run[1 + u] + (int64_t)item * (of + a.p.item_cost) + a.p.item_cost;
        const int64_t c0 = x0 / run, c1 = (x0 + of - 1) / run;
        if (c0 == c1) return;                         // one CTA had it all, and wrote the output
        const int n = (int)(c1 - c0) + 1;
#pragma unroll 1
        for (int i0 = warp; i0 < n; i0 += U * W) {
            float2 ml[U][K];
            float4 y[U][K];
#pragma unroll
            for (int e = 0; e < U; ++e) {
                // the last CTA's part is its first segment, the others' their last
                const int i = i0 + e * W, j = U == 1 ? i : min(i, n - 1);
                const int64_t at = (2 * (c0 + j) + (j + 1 < n ? 1 : 0)) * ROWS + row0;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    ml[e][k] = *reinterpret_cast<const float2*>(a.w.part_ml + (at + k) * 2);
                    y[e][k] = *reinterpret_cast<const float4*>(a.w.part + (at + k) * D + 4 * min(lane, D / 4 - 1));
                    if (U > 1 && i >= n) ml[e][k] = make_float2(kLow, 0.0f), y[e][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float top = m[k];
#pragma unroll
                for (int e = 0; e < U; ++e) top = fmaxf(top, ml[e][k].x);
                const float f = exp2_fast(m[k] - top);
                m[k] = top;
#pragma unroll
                for (int e = 0; e < U; ++e) {
                    const float g = exp2_fast(ml[e][k].x - top), by = e ? 1.0f : f;
                    l[k] = fmaf(l[k], by, ml[e][k].y * g);
                    acc[k] = make_float4(fmaf(acc[k].x, by, y[e][k].x * g), fmaf(acc[k].y, by, y[e][k].y * g),
                                         fmaf(acc[k].z, by, y[e][k].z * g), fmaf(acc[k].w, by, y[e][k].w * g));
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (lane == 0) s_ml[warp][k] = make_float2(m[k], l[k]);
        if (lane < D / 4) s_acc[warp][k][lane] = acc[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < K * (D / 4); i += 32 * W) {
        const int k = i / (D / 4), c4 = i % (D / 4), x = tile * ROWS + row0 + k;
        if (x >= a.p.R) break;
        float top = s_ml[0][k].x, sum = 0.0f;
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, s_ml[w][k].x);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = exp2_fast(s_ml[w][k].x - top);
            const float4 y = s_acc[w][k][c4];
            sum = fmaf(s_ml[w][k].y, f, sum);
            o = make_float4(fmaf(y.x, f, o.x), fmaf(y.y, f, o.y), fmaf(y.z, f, o.z), fmaf(y.w, f, o.w));
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        __nv_bfloat162 y[2] = {__floats2bfloat162_rn(o.x * inv, o.y * inv), __floats2bfloat162_rn(o.z * inv, o.w * inv)};
        const int b = a.list ? u / s.T : u;
        const int tq = a.list ? u % s.T : x / s.G, g = a.list ? x : x % s.G;
        *reinterpret_cast<uint2*>(a.O + (((int64_t)b * s.T + tq) * s.HQ + h * s.G + g) * D + 4 * c4) = *reinterpret_cast<uint2*>(y);
    }
}

}  // namespace

// Attention of many rows a key head, on tcgen05 (asa_cache_chunk.cu).
bool chunk_takes(const Shape& s, int keep);
size_t chunk_workspace(const Shape& s);
cudaError_t chunk_attend(const Shape& s, const void* Q, Strides qs, const uint8_t* pool, const int32_t* table,
                         const int32_t* lengths, void* O, void* ws, int* err, cudaStream_t st);

}  // namespace cache
}  // namespace asa
