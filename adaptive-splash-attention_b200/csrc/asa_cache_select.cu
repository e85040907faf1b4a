// asa_cache_select.cu -- choosing the pages that a query reads, by a score from
// the pages' bounds.
//
// score(page) = max over the group's heads of
//     unit_q * 2^e * sum_c max(n_c upper_c, n_c lower_c),  n = rint(q / unit_q)
// -- an upper bound of n.k over the page's keys.  The sum is of whole numbers
// below 2^24, so it is the same in any order and ties are exact.
#include "asa_cache.h"

namespace asa {
namespace cache {
namespace {

// Larger floats as larger integers; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float f) {
    if (f != f) return 0u;
    if (f == 0.0f) f = 0.0f;
    const uint32_t b = __float_as_uint(f == 0.0f ? 0.0f : f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One CTA a (query, key head): scores, a radix selection of the keep-th largest,
// then the chosen pages in ascending order.
__global__ void __launch_bounds__(256) select_kernel(Shape s, const __nv_bfloat16* __restrict__ Q, Strides qs,
                                                     const int8_t* __restrict__ bounds,
                                                     const int32_t* __restrict__ table,
                                                     const int32_t* __restrict__ lengths, int keep,
                                                     int32_t* __restrict__ pages, uint32_t* __restrict__ ws,
                                                     int* err) {
    extern __shared__ float s_q[];          // [G][d] codes, then [G] units
    __shared__ int s_hist[256], s_part[8][2];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_done;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x % s.H;
    const int bt = blockIdx.x / s.H, t = bt % s.T, b = bt / s.T;
    int32_t* out = pages + (int64_t)blockIdx.x * keep;
    const long long pos = min((long long)__ldg(lengths + b) - s.T + t, (long long)s.width * s.P - 1);
    const int n = pos < 0 ? 0 : (int)(pos / s.P) + 1;        // the pages it can see, its own last
    if (n <= keep) {
        for (int i = tid; i < keep; i += 256) out[i] = i < n ? i : -1;
        return;
    }
    float* s_unit = s_q + s.G * s.d;
    for (int g = warp; g < s.G; g += 8) {
        const __nv_bfloat16* q = Q + b * qs.b + t * qs.t + (int64_t)(h * s.G + g) * qs.h;
        float m = 0.0f;
        bool bad = false;
        for (int c = lane; c < s.d; c += 32) {
            const float x = __bfloat162float(q[c]);
            bad |= x != x;
            m = fmaxf(m, fabsf(x));
        }
#pragma unroll
        for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, k));
        const float unit = __any_sync(~0u, bad) ? NAN : __fmul_rn(m, k127th);
        for (int c = lane; c < s.d; c += 32)
            s_q[g * s.d + c] = unit > 0.0f ? rintf(__fdiv_rn(__bfloat162float(q[c]), unit)) : 0.0f;
        if (lane == 0) s_unit[g] = unit;
    }
    if (tid == 0) s_prefix = 0u, s_need = keep - 1;
    __syncthreads();
    uint32_t* key = ws + (int64_t)blockIdx.x * s.width;
    for (int i = tid; i < n - 1; i += 256) {
        const int id = __ldg(table + (int64_t)b * s.width + i);
        uint32_t k = 0u;
        if (id >= 0 && id < s.pages) {
            const int8_t* rb = bounds + ((int64_t)id * s.H + h) * bounds_bytes(s.d);
            const int e = min(max(*reinterpret_cast<const int*>(rb + 2 * s.d), -126), 127);
            const float unit = __int_as_float((e + 127) << 23);
            for (int g = 0; g < s.G; ++g) {
                float acc = 0.0f;
                for (int c = 0; c < s.d; ++c) {
                    const float q = s_q[g * s.d + c];
                    acc += q * (float)(q > 0.0f ? rb[c] : rb[s.d + c]);
                }
                k = max(k, ordered(__fmul_rn(__fmul_rn(acc, unit), s_unit[g])));
            }
        } else if (err) {
            atomicCAS(err, 0, ASA_ERR_INVALID);
        }
        key[i] = k;
    }
    // the (keep - 1)-th largest key, eight bits at a time
    for (int shift = 24; shift >= 0; shift -= 8) {
        s_hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int i = tid; i < n - 1; i += 256)
            if (shift == 24 || key[i] >> (shift + 8) == prefix) atomicAdd(&s_hist[key[i] >> shift & 255], 1);
        __syncthreads();
        if (tid == 0) {
            int need = s_need, v = 255;
            while (v > 0 && need > s_hist[v]) need -= s_hist[v--];
            s_need = need;
            s_prefix = prefix << 8 | (uint32_t)v;
        }
        __syncthreads();
    }
    const uint32_t edge = s_prefix;
    const int ties = s_need;                 // keys equal to the edge that are taken, the lowest pages first
    int before = 0, tied = 0;
    for (int base = 0; base < n; base += 256) {
        const int i = base + tid;
        const uint32_t k = i < n - 1 ? key[i] : 0u;
        const bool is_tie = i < n - 1 && k == edge;
        const uint32_t tie_votes = __ballot_sync(~0u, is_tie);
        if (lane == 0) s_part[warp][0] = __popc(tie_votes);
        __syncthreads();
        int rank = tied + __popc(tie_votes & ((1u << lane) - 1u)), all = 0;
        for (int w = 0; w < 8; ++w) {
            if (w < warp) rank += s_part[w][0];
            all += s_part[w][0];
        }
        const bool take = i == n - 1 || (i < n - 1 && (k > edge || (is_tie && rank < ties)));
        const uint32_t votes = __ballot_sync(~0u, take);
        if (lane == 0) s_part[warp][1] = __popc(votes);
        __syncthreads();
        int at = before + __popc(votes & ((1u << lane) - 1u)), sum = 0;
        for (int w = 0; w < 8; ++w) {
            if (w < warp) at += s_part[w][1];
            sum += s_part[w][1];
        }
        if (take) out[at] = i;
        before += sum;
        tied += all;
        __syncthreads();
    }
}

}  // namespace

size_t select_workspace(const Shape& s) {
    return ((size_t)s.B * s.T * s.H * s.width * 4 + 16 + 15) & ~size_t(15);
}

cudaError_t select(const Shape& s, const void* Q, Strides qs, const int8_t* bounds, const int32_t* table,
                   const int32_t* lengths, int keep, int32_t* pages, void* ws, int* err, cudaStream_t st) {
    const size_t smem = ((size_t)s.G * s.d + s.G) * 4;
    if (smem > 200 * 1024) return cudaErrorInvalidConfiguration;
    if (smem > 40 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    select_kernel<<<(unsigned)(s.B * s.T * s.H), 256, smem, st>>>(
        s, (const __nv_bfloat16*)Q, qs, bounds, table, lengths, keep, pages, (uint32_t*)ws, err);
    note_launch();
    return cudaGetLastError();
}

}  // namespace cache
}  // namespace asa
