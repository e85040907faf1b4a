// asa_cache_attend.cu -- attention over the 4-bit paged cache.
#include "asa_cache.h"

namespace asa {
namespace cache {
namespace {

__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
    for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(~0u, v, k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}
__device__ __forceinline__ float block_max(float v, float* part) {
#pragma unroll
    for (int k = 16; k; k >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, k));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// The j-th token that a query's walk over the cache meets: its record's block
// and row, or null where it sees none.
__device__ __forceinline__ const uint8_t* token_at(const Shape& s, const uint8_t* pool, const int32_t* table_b,
                                                   const int32_t* list, int h, long long pos, int j, int* err) {
    int page = j / s.P;
    if (list) page = __ldg(list + page);
    if (page < 0 || page >= s.width || (long long)page * s.P + j % s.P > pos) return nullptr;
    const int id = __ldg(table_b + page);
    if (id < 0 || id >= s.pages) {
        if (err) atomicCAS(err, 0, ASA_ERR_INVALID);
        return nullptr;
    }
    return pool + ((int64_t)id * s.H + h) * s.rec + (int64_t)(j % s.P / kBlock) * block_bytes(s.d);
}

// One CTA a row (query token and head): scores to the workspace, their weights,
// and the weighted sum of the values, a channel a thread.
__global__ void __launch_bounds__(128) rows_kernel(Shape s, const __nv_bfloat16* __restrict__ Q, Strides qs,
                                                   const uint8_t* __restrict__ pool,
                                                   const int32_t* __restrict__ table,
                                                   const int32_t* __restrict__ lengths,
                                                   const int32_t* __restrict__ list, int keep,
                                                   __nv_bfloat16* __restrict__ O, float* __restrict__ ws, int n_max,
                                                   int* err) {
    __shared__ float s_q[128], s_part[4];
    const int tid = threadIdx.x, hq = blockIdx.x % s.HQ, bt = blockIdx.x / s.HQ, t = bt % s.T, b = bt / s.T;
    const int h = hq / s.G, NG = s.d / 32;
    const int32_t* table_b = table + (int64_t)b * s.width;
    const int32_t* mine = list ? list + ((int64_t)bt * s.H + h) * keep : nullptr;
    const long long pos = (long long)__ldg(lengths + b) - s.T + t;
    const int n = list ? n_max : (int)max(0ll, min(pos + 1, (long long)n_max));
    float* sc = ws + (int64_t)blockIdx.x * n_max;
    if (tid < s.d) {
        const float x = __bfloat162float(Q[b * qs.b + t * qs.t + (int64_t)hq * qs.h + tid]);
        s_q[tid] = isfinite(x) ? x : NAN;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int j = tid; j < n; j += 128) {
        const uint8_t* blk = token_at(s, pool, table_b, mine, h, pos, j, err);
        float v = -INFINITY;
        if (blk) {
            const int r = j % kBlock;
            const uint8_t* row = blk + r * row_bytes(s.d);
            const __half* par = reinterpret_cast<const __half*>(blk + kBlock * row_bytes(s.d)) + r * 2 * NG;
            float acc = 0.0f;
            for (int c = 0; c < s.d; ++c) {
                const int g = c >> 5, w = c & 31;
                const uint32_t byte = row[(w >> 3) * 4 * NG + 4 * g + ((w & 7) >> 1)];
                acc += s_q[c] * fmaf((float)(c & 1 ? byte >> 4 : byte & 15u), __half2float(par[g]),
                                     __half2float(par[NG + g]));
            }
            v = acc * s.scale;
            if (s.alpha != 1.0f) v = v != v ? v : (s.alpha - 1.0f) * fminf(fmaxf(v, -10.0f), 10.0f);
            top = fmaxf(top, v);
            if (v != v) top = INFINITY;      // a NaN score makes the whole row NaN
        }
        sc[j] = v;
    }
    top = block_max(top, s_part);
    float total = 0.0f;
    if (top > -INFINITY) {
        float tau = 0.0f;
        if (s.alpha != 1.0f) {
            float lo = top - 1.0f, hi = top;
            const float ex = 1.0f / (s.alpha - 1.0f);
            for (int it = 0; it < 40; ++it) {
                const float mid = 0.5f * (lo + hi);
                float sum = 0.0f;
                for (int j = tid; j < n; j += 128) sum += sc[j] > mid ? powf(sc[j] - mid, ex) : 0.0f;
                if (block_sum(sum, s_part) >= 1.0f) lo = mid; else hi = mid;
            }
            tau = lo;
        }
        float sum = 0.0f;
        for (int j = tid; j < n; j += 128) {
            float p;
            if (s.alpha == 1.0f) p = sc[j] == -INFINITY ? 0.0f : expf(sc[j] - top);
            else p = sc[j] != sc[j] ? sc[j] : sc[j] > tau ? powf(sc[j] - tau, 1.0f / (s.alpha - 1.0f)) : 0.0f;
            if (top == INFINITY) p = NAN;
            sc[j] = p;
            sum += p;
        }
        total = block_sum(sum, s_part);
    }
    if (tid >= s.d) return;
    float acc = 0.0f;
    if (top > -INFINITY)
        for (int j = 0; j < n; ++j) {
            const uint8_t* blk = token_at(s, pool, table_b, mine, h, pos, j, nullptr);
            if (!blk) continue;
            blk += s.rec / 2;
            const int r = j % kBlock, g = tid >> 5, w = tid & 31;
            const __half* par = reinterpret_cast<const __half*>(blk + kBlock * row_bytes(s.d)) + r * 2 * NG;
            const uint32_t byte = blk[r * row_bytes(s.d) + (w >> 2) * 2 * NG + 2 * g + ((w & 3) >> 1)];
            acc += sc[j] * fmaf((float)(tid & 1 ? byte >> 4 : byte & 15u), __half2float(par[g]),
                                __half2float(par[NG + g]));
        }
    O[(int64_t)blockIdx.x * s.d + tid] = __float2bfloat16(top > -INFINITY ? acc / total : 0.0f);
}

}  // namespace

size_t attend_workspace(const Shape& s, int keep) {
    const size_t n = (size_t)(keep ? keep : s.width) * s.P;
    return (size_t)s.B * s.T * s.HQ * n * 4 + 16;
}

cudaError_t attend(const Shape& s, const void* Q, Strides qs, const uint8_t* pool, const int32_t* table,
                   const int32_t* lengths, const int32_t* list, int keep, void* O, void* ws, int* err,
                   cudaStream_t st) {
    rows_kernel<<<(unsigned)(s.B * s.T * s.HQ), 128, 0, st>>>(
        s, (const __nv_bfloat16*)Q, qs, pool, table, lengths, list, keep, (__nv_bfloat16*)O, (float*)ws,
        (list ? keep : s.width) * s.P, err);
    note_launch();
    return cudaGetLastError();
}

}  // namespace cache
}  // namespace asa
