// asa_cache_store.cu -- quantising keys and values into the 4-bit paged cache,
// keeping the pages' bounds, and reading both back.
//
// Per group of 32 channels: offset z = fp16(min), scale s = fp16((max - z) * fl(1/15)),
// code n = rint((x - z)/s) clipped to 0..15; a value reads back as z + n s (one
// rounding to fp32: n s is exact there), then as bf16 where asked.
#include "asa_cache.h"

namespace asa {
namespace cache {
namespace {

template <typename X>
__device__ __forceinline__ void load4(const X* p, float (&x)[4]);
template <>
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __ldg(p + i);
}
template <>
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(p[i]);
}

// One token's row of one key head by one warp: lane l has channels 4l..4l+3, a
// group is eight lanes.  Writes the codes (two bytes a lane) and, from each
// group's first lane, its scale and offset.
template <int D, bool KEY>
__device__ __forceinline__ void quantise_row(const float (&raw)[4], uint8_t* codes, __half* par) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x & 31;
    float x[4], lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        nan |= raw[i] != raw[i];
        x[i] = fminf(fmaxf(raw[i], -kF16Max), kF16Max);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(~0u, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, m));
    }
    nan = (__ballot_sync(~0u, nan) >> (lane & 24)) & 0xff;
    const __half z = __float2half_rn(lo);
    const float zf = __half2float(z);
    const __half s = __float2half_rn(__fmul_rn(hi - zf, kFifteenth));
    const float sf = __half2float(s);
    uint32_t n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        n[i] = sf > 0.0f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x[i] - zf, sf)), 0.0f), 15.0f) : 0u;
    const int g = lane >> 3, w = lane & 7;
    if (g >= NG) return;
    const uint16_t two = (uint16_t)(n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12);
    const int at = KEY ? (w >> 1) * 4 * NG + 4 * g + 2 * (w & 1) : w * 2 * NG + 2 * g;
    *reinterpret_cast<uint16_t*>(codes + at) = two;
    if (w == 0) {
        const __half bad = __ushort_as_half(0x7fff);
        par[g] = nan ? bad : s;
        par[NG + g] = nan ? bad : z;
    }
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// One CTA a (sequence, touched page, key head): its tokens, then the page's bounds.
template <typename X, int D>
__global__ void __launch_bounds__(256) write_kernel(Shape s, const X* __restrict__ K, const X* __restrict__ V,
                                                    Strides ks, Strides vs, uint8_t* __restrict__ pool,
                                                    int8_t* __restrict__ bounds, const int32_t* __restrict__ table,
                                                    const int32_t* __restrict__ start,
                                                    const int32_t* __restrict__ count, int touched, int* err) {
    constexpr int NG = D / 32, W = 8;
    __shared__ float s_hi[W][D], s_lo[W][D];
    __shared__ float s_m[W];
    const int h = blockIdx.x % s.H, j = blockIdx.x / s.H % touched, b = blockIdx.x / s.H / touched;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long begin = __ldg(start + b);
    const long long n = count ? min(max(__ldg(count + b), 0), s.T) : s.T;
    if (n == 0) return;
    // the pages that positions begin .. begin + n - 1 lie in, the j-th of them
    const long long page_no = (begin >= 0 ? begin / s.P : -((-begin + s.P - 1) / s.P)) + j;
    const long long first = max(begin, page_no * s.P), last = min(begin + n, (page_no + 1) * s.P);
    if (first >= last) return;
    int id = -1;
    if (page_no >= 0 && page_no < s.width) id = __ldg(table + (int64_t)b * s.width + page_no);
    if (id < 0 || id >= s.pages) {
        if (threadIdx.x == 0 && err) atomicCAS(err, 0, ASA_ERR_INVALID);
        return;
    }
    uint8_t* rec = pool + ((int64_t)id * s.H + h) * s.rec;
    float hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = -INFINITY, lo[i] = INFINITY;
    for (long long pos = first + warp; pos < last; pos += W) {
        const int slot = (int)(pos - page_no * s.P);
        const int64_t t = pos - begin;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (4 * lane < D) {
            load4<X>(K + b * ks.b + t * ks.t + h * ks.h + 4 * lane, x);
            load4<X>(V + b * vs.b + t * vs.t + h * vs.h + 4 * lane, y);
        }
        uint8_t* kb = rec + (int64_t)(slot / kBlock) * block_bytes(D);
        uint8_t* vb = kb + s.rec / 2;
        const int r = slot % kBlock;
        quantise_row<D, true>(x, kb + r * row_bytes(D),
                              reinterpret_cast<__half*>(kb + kBlock * row_bytes(D)) + r * 2 * NG);
        quantise_row<D, false>(y, vb + r * row_bytes(D),
                               reinterpret_cast<__half*>(vb + kBlock * row_bytes(D)) + r * 2 * NG);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = x[i] != x[i] ? 0.0f : fminf(fmaxf(x[i], -kF16Max), kF16Max);
            hi[i] = fmaxf(hi[i], c);
            lo[i] = fminf(lo[i], c);
        }
    }
    if (4 * lane < D)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_hi[warp][4 * lane + i] = hi[i], s_lo[warp][4 * lane + i] = lo[i];
    __syncthreads();
    int8_t* rb = bounds + ((int64_t)id * s.H + h) * bounds_bytes(D);
    const int c = threadIdx.x;
    float top = 0.0f, low = 0.0f;
    if (c < D) {
        top = s_hi[0][c];
        low = s_lo[0][c];
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, s_hi[w][c]), low = fminf(low, s_lo[w][c]);
        if (first > page_no * s.P) {         // begun by an earlier call: its bounds stand
            const float unit = pow2(min(max(*reinterpret_cast<const int*>(rb + 2 * D), -126), 127));
            top = fmaxf(top, (float)rb[c] * unit);
            low = fminf(low, (float)rb[D + c] * unit);
        }
    }
    float m = fmaxf(fabsf(top), fabsf(low));
#pragma unroll
    for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, k));
    if (lane == 0) s_m[warp] = m;
    __syncthreads();                         // also: every old bound has been read
    m = s_m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, s_m[w]);
    int e = -126;
    if (m > 0.0f) {
        const float f = frexpf(m, &e);
        e = max(e - 7 + (f > 127.0f / 128.0f ? 1 : 0), -126);
    }
    const float inv = pow2(-e);
    if (c < D) {
        rb[c] = (int8_t)ceilf(top * inv);
        rb[D + c] = (int8_t)floorf(low * inv);
    }
    if (c == 0) *reinterpret_cast<int*>(rb + 2 * D) = e;
}

template <typename X>
__device__ __forceinline__ void store8(X* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    __nv_bfloat162 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
}

// A thread an eight-channel run of a token: its key and its value.
template <typename X, int D>
__global__ void __launch_bounds__(256) read_kernel(Shape s, const uint8_t* __restrict__ pool,
                                                   const int32_t* __restrict__ table,
                                                   const int32_t* __restrict__ start,
                                                   const int32_t* __restrict__ count, X* __restrict__ K,
                                                   X* __restrict__ V, int* err) {
    constexpr int NG = D / 32, R = D / 8;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t row = i / R;                       // (b, t, h)
    if (row >= (int64_t)s.B * s.T * s.H) return;
    const int run = (int)(i % R), h = (int)(row % s.H);
    const int64_t bt = row / s.H;
    const int t = (int)(bt % s.T), b = (int)(bt / s.T);
    float k[8], v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) k[c] = v[c] = 0.0f;
    const int n = count ? __ldg(count + b) : s.T;
    if (t < n) {
        const long long pos = (long long)__ldg(start + b) + t;
        int id = -1;
        if (pos >= 0 && pos / s.P < s.width) id = __ldg(table + (int64_t)b * s.width + pos / s.P);
        if (id >= 0 && id < s.pages) {
            const int slot = (int)(pos % s.P), r = slot % kBlock;
            const uint8_t* kb = pool + ((int64_t)id * s.H + h) * s.rec + (int64_t)(slot / kBlock) * block_bytes(D);
            const uint8_t* vb = kb + s.rec / 2;
            const int g = run >> 2, q = run & 3;     // channels 32 g + 8 q ..
            const __half* kp = reinterpret_cast<const __half*>(kb + kBlock * row_bytes(D)) + r * 2 * NG;
            const __half* vp = reinterpret_cast<const __half*>(vb + kBlock * row_bytes(D)) + r * 2 * NG;
            const uint8_t* vr = vb + r * row_bytes(D);
            const uint32_t kw = *reinterpret_cast<const uint32_t*>(kb + r * row_bytes(D) + q * 4 * NG + 4 * g);
            const uint32_t vw = *reinterpret_cast<const uint16_t*>(vr + 2 * q * 2 * NG + 2 * g) |
                                (uint32_t)*reinterpret_cast<const uint16_t*>(vr + (2 * q + 1) * 2 * NG + 2 * g) << 16;
            const float ksc = __half2float(kp[g]), kz = __half2float(kp[NG + g]);
            const float vsc = __half2float(vp[g]), vz = __half2float(vp[NG + g]);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                k[c] = fmaf((float)((kw >> (4 * c)) & 15u), ksc, kz);
                v[c] = fmaf((float)((vw >> (4 * c)) & 15u), vsc, vz);
            }
        } else if (err) {
            atomicCAS(err, 0, ASA_ERR_INVALID);
        }
    }
    store8<X>(K + row * D + 8 * run, k);
    store8<X>(V + row * D + 8 * run, v);
}

__global__ void __launch_bounds__(256) bounds_kernel(Shape s, const int8_t* __restrict__ bounds,
                                                     const int32_t* __restrict__ pages, int n,
                                                     float* __restrict__ upper, float* __restrict__ lower,
                                                     int* err) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)n * s.H * s.d) return;
    const int c = (int)(i % s.d), h = (int)(i / s.d % s.H);
    const int id = __ldg(pages + i / s.d / s.H);
    float top = 0.0f, low = 0.0f;
    if (id >= 0 && id < s.pages) {
        const int8_t* rb = bounds + ((int64_t)id * s.H + h) * bounds_bytes(s.d);
        const float unit = pow2(min(max(*reinterpret_cast<const int*>(rb + 2 * s.d), -126), 127));
        top = (float)rb[c] * unit;
        low = (float)rb[s.d + c] * unit;
    } else if (err) {
        atomicCAS(err, 0, ASA_ERR_INVALID);
    }
    upper[i] = top;
    lower[i] = low;
}

template <typename X, int D>
cudaError_t write_as(const Shape& s, const void* K, const void* V, Strides ks, Strides vs, uint8_t* pool,
                     int8_t* bounds, const int32_t* table, const int32_t* start, const int32_t* count,
                     int* err, cudaStream_t st) {
    const int touched = (s.T + s.P - 2) / s.P + 1;
    const long long grid = (long long)s.B * touched * s.H;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    write_kernel<X, D><<<(unsigned)grid, 256, 0, st>>>(s, (const X*)K, (const X*)V, ks, vs, pool, bounds,
                                                       table, start, count, touched, err);
    note_launch();
    return cudaGetLastError();
}

template <typename X, int D>
cudaError_t read_as(const Shape& s, const uint8_t* pool, const int32_t* table, const int32_t* start,
                    const int32_t* count, void* K, void* V, int* err, cudaStream_t st) {
    const long long threads = (long long)s.B * s.T * s.H * (D / 8);
    const long long grid = (threads + 255) / 256;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    read_kernel<X, D><<<(unsigned)grid, 256, 0, st>>>(s, pool, table, start, count, (X*)K, (X*)V, err);
    note_launch();
    return cudaGetLastError();
}

}  // namespace

#define ASA_CACHE_BY_D(F, X, ...)                            \
    (s.d == 32   ? F<X, 32>(__VA_ARGS__)                     \
     : s.d == 64 ? F<X, 64>(__VA_ARGS__)                     \
     : s.d == 96 ? F<X, 96>(__VA_ARGS__)                     \
                 : F<X, 128>(__VA_ARGS__))

cudaError_t write(const Shape& s, const void* K, const void* V, Strides ks, Strides vs, uint8_t* pool,
                  int8_t* bounds, const int32_t* table, const int32_t* start, const int32_t* count,
                  int* err, cudaStream_t st) {
    return s.dtype == ASA_DTYPE_F32
               ? ASA_CACHE_BY_D(write_as, float, s, K, V, ks, vs, pool, bounds, table, start, count, err, st)
               : ASA_CACHE_BY_D(write_as, __nv_bfloat16, s, K, V, ks, vs, pool, bounds, table, start, count,
                                err, st);
}

cudaError_t read(const Shape& s, const uint8_t* pool, const int32_t* table, const int32_t* start,
                 const int32_t* count, void* K, void* V, int* err, cudaStream_t st) {
    return s.dtype == ASA_DTYPE_F32
               ? ASA_CACHE_BY_D(read_as, float, s, pool, table, start, count, K, V, err, st)
               : ASA_CACHE_BY_D(read_as, __nv_bfloat16, s, pool, table, start, count, K, V, err, st);
}

cudaError_t read_bounds(const Shape& s, const int8_t* bounds, const int32_t* pages, int n, float* upper,
                        float* lower, int* err, cudaStream_t st) {
    const long long grid = ((long long)n * s.H * s.d + 255) / 256;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    bounds_kernel<<<(unsigned)grid, 256, 0, st>>>(s, bounds, pages, n, upper, lower, err);
    note_launch();
    return cudaGetLastError();
}

}  // namespace cache
}  // namespace asa
