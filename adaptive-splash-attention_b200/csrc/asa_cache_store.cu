// asa_cache_store.cu -- quantising keys and values into the 4-bit paged cache,
// keeping the pages' bounds, and reading both back.
//
// Per group of 32 channels: offset z = fp16(min), scale s = fp16((max - z) * fl(1/15)),
// not below 0, code n = rint((x - z)/s) clipped to 0..15; a value reads back as z + n s (one
// rounding to fp32: n s is exact there), then as bf16 where asked.
#include "asa_cache.h"

namespace asa {
namespace cache {
namespace {

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Eight neighbouring channels as they lie in memory, and as fp32.
template <typename X>
struct Eight;
template <>
struct Eight<float> {
    float x[8];
    __device__ __forceinline__ void load(const float* p, bool vec) {
        if (vec) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __ldg(p + i);
        }
    }
    __device__ __forceinline__ float2 pair(int i) const { return make_float2(x[2 * i], x[2 * i + 1]); }
    // smallest and largest, NaN if there is one
    __device__ __forceinline__ void range(float& lo, float& hi) const {
        lo = hi = x[0];
        bool nan = x[0] != x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]), nan |= x[i] != x[i];
        if (nan) lo = hi = NAN;
    }
};
template <>
struct Eight<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* p, bool vec) {
        if (vec) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __ldg(e + 2 * i) | (uint32_t)__ldg(e + 2 * i + 1) << 16;
        }
    }
    __device__ __forceinline__ float2 pair(int i) const {
        return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    __device__ __forceinline__ void range(float& lo, float& hi) const {
        const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(w);
        const float2 a = __bfloat1622float2(__hmin2_nan(__hmin2_nan(v[0], v[1]), __hmin2_nan(v[2], v[3])));
        const float2 b = __bfloat1622float2(__hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3])));
        lo = a.x != a.x ? a.x : a.y != a.y ? a.y : fminf(a.x, a.y);
        hi = b.x != b.x ? b.x : b.y != b.y ? b.y : fmaxf(b.x, b.y);
    }
};

// The fp16 a code is counted in, from a group's smallest and largest.
struct Grid { float z, s; uint32_t bits; };           // bits: s, then z
__device__ __forceinline__ Grid grid_of(float lo, float hi) {
    Grid g;
    const __half z = __float2half_rn(lo);
    g.z = __half2float(z);
    // (below zero where a group of equal numbers has its offset rounded up)
    const __half s = __float2half_rn(fmaxf(__fmul_rn(hi - g.z, kFifteenth), 0.0f));
    g.s = __half2float(s);
    g.bits = __half_as_ushort(s) | (uint32_t)__half_as_ushort(z) << 16;
    return g;
}

// Codes of eight channels, the first in the lowest four bits.  The quotient is
// approximated by a product with 1 / s (within 2^-21 of it for codes up to 15) and
// rounded by adding 1.5 * 2^23; where it comes within 2^-18 of a half, or a code
// could leave 0..15, `sure` is lowered and exact_codes decides.
template <typename X>
__device__ __forceinline__ uint32_t quick_codes(const Eight<X>& x, const Grid& g, bool& sure) {
    const float inv = g.s > 0.0f ? __frcp_rn(g.s) : 0.0f, magic = 12582912.0f;
    float worst = 0.0f, r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __fmul2_rn(__fadd2_rn(x.pair(i), make_float2(-g.z, -g.z)), make_float2(inv, inv));
        const float2 f = __fadd2_rn(__fadd2_rn(v, make_float2(magic, magic)), make_float2(-magic, -magic));
        const float2 d = __fadd2_rn(v, make_float2(-f.x, -f.y));
        worst = fmaxf(worst, fmaxf(fabsf(d.x), fabsf(d.y)));
        r[2 * i] = f.x;
        r[2 * i + 1] = f.y;
    }
    sure &= worst < 0.5f - 3.8147e-6f;
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        const float sum = fmaf(fmaf(fmaf(r[i + 3], 16.0f, r[i + 2]), 16.0f, r[i + 1]), 16.0f, r[i]);
        out |= (__float_as_uint(sum + magic) & 0xffffu) << (4 * i);
    }
    return out;
}
template <typename X>
__device__ __noinline__ uint32_t exact_codes(const Eight<X>& x, float z, float s) {
    uint32_t out = 0;
    for (int i = 0; i < 4; ++i) {
        const float2 v = x.pair(i);
        for (int e = 0; e < 2; ++e) {
            const float c = fminf(fmaxf(e ? v.y : v.x, -kF16Max), kF16Max);
            const float n = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(c - z, s)), 0.0f), 15.0f) : 0.0f;
            out |= (uint32_t)n << (4 * (2 * i + e));
        }
    }
    return out;
}

// A row's part in one lane: codes and grid of its eight channels; the group is
// four lanes.  All lanes take part.
template <typename X>
__device__ __forceinline__ uint32_t quantise(const Eight<X>& x, uint32_t& grid, bool& nan) {
    float lo, hi;
    x.range(lo, hi);
    nan = lo != lo;
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(~0u, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, m));
    }
    const uint32_t group_nan = (__ballot_sync(~0u, nan) >> (threadIdx.x & 28)) & 15u;
    bool sure = lo >= -kF16Max && hi <= kF16Max;
    lo = fminf(fmaxf(lo, -kF16Max), kF16Max);
    hi = fminf(fmaxf(hi, -kF16Max), kF16Max);
    const Grid g = grid_of(lo, hi);
    // with the offset rounded up far enough, or the scale rounded down, codes would leave 0..15
    sure &= lo - g.z >= -0.25f * g.s && hi - g.z <= 15.25f * g.s;
    uint32_t codes = quick_codes<X>(x, g, sure);
    if (__any_sync(~0u, !sure)) codes = exact_codes<X>(x, g.z, g.s);
    grid = group_nan ? 0x7fff7fffu : g.bits;
    return codes;
}

// One CTA a (sequence, touched page, key head): its tokens' keys and values, then
// the page's bounds.  A row is D/8 lanes of eight channels, so that a warp
// reads 512 bytes of bf16 at a time.
template <typename X, int D, int W>
__global__ void __launch_bounds__(W * 32) write_kernel(Shape s, const X* __restrict__ K, const X* __restrict__ V,
                                                       Strides ks, Strides vs, int vec, uint8_t* __restrict__ pool,
                                                       int8_t* __restrict__ bounds, const int32_t* __restrict__ table,
                                                       const int32_t* __restrict__ start,
                                                       const int32_t* __restrict__ count, int touched, int* err) {
    constexpr int NG = D / 32, LR = D / 8, RW = 32 / LR, RB = row_bytes(D), NTHR = W * 32;
    __shared__ float s_hi[W * RW][D], s_lo[W * RW][D];
    __shared__ float s_m[W];
    const int h = blockIdx.x % s.H, j = blockIdx.x / s.H % touched, b = blockIdx.x / s.H / touched;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / LR, at = lane % LR, g = at >> 2, q = at & 3;   // row of the warp, channels 32 g + 8 q ..
    const bool lane_in = sub < RW;                    // (96 channels leave eight lanes over)
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
    const int64_t t0 = first - begin;
    const int rows = (int)(last - first), slot0 = (int)(first - page_no * s.P);
    const X* kp = K + b * ks.b + t0 * ks.t + h * ks.h + 8 * at;
    const X* vp = V + b * vs.b + t0 * vs.t + h * vs.h + 8 * at;
    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = -INFINITY, lo[i] = INFINITY;
    constexpr int U = 2;                              // rows in flight a lane
    for (int i0 = warp * RW; i0 < rows; i0 += U * W * RW) {
        Eight<X> k[U], v[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * W * RW + sub;
            in[u] = lane_in && i < rows;
            k[u] = v[u] = Eight<X>{};
            if (in[u]) {
                k[u].load(kp + i * ks.t, vec);
                v[u].load(vp + i * vs.t, vec);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * W * RW >= rows) break;
            const int slot = slot0 + i0 + u * W * RW + sub, r = slot % kBlock;
            uint8_t* kb = rec + (int64_t)(slot / kBlock) * block_bytes(D);
            uint8_t* vb = kb + s.rec / 2;
            uint32_t kg, vg;
            bool k_nan, v_nan;
            const uint32_t kc = quantise<X>(k[u], kg, k_nan), vc = quantise<X>(v[u], vg, v_nan);
            if (!in[u]) continue;
            *reinterpret_cast<uint32_t*>(kb + r * RB + q * 4 * NG + 4 * g) = kc;
            uint8_t* vr = vb + r * RB + 2 * q * 2 * NG + 2 * g;
            *reinterpret_cast<uint16_t*>(vr) = (uint16_t)vc;
            *reinterpret_cast<uint16_t*>(vr + 2 * NG) = (uint16_t)(vc >> 16);
            // the group's lanes store the key's scale and offset, the value's scale and offset
            uint8_t* par = (q < 2 ? kb : vb) + kBlock * RB + r * par_bytes(D) + 2 * g + (q & 1 ? 2 * NG : 0);
            const uint32_t pv = q < 2 ? kg : vg;
            *reinterpret_cast<uint16_t*>(par) = (uint16_t)(q & 1 ? pv >> 16 : pv);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float2 y = k[u].pair(c);
                if (k_nan) y.x = y.x != y.x ? 0.0f : y.x, y.y = y.y != y.y ? 0.0f : y.y;
                hi[2 * c] = fmaxf(hi[2 * c], y.x);
                lo[2 * c] = fminf(lo[2 * c], y.x);
                hi[2 * c + 1] = fmaxf(hi[2 * c + 1], y.y);
                lo[2 * c + 1] = fminf(lo[2 * c + 1], y.y);
            }
        }
    }
    if (lane_in)
#pragma unroll
        for (int i = 0; i < 8; ++i) s_hi[warp * RW + sub][8 * at + i] = hi[i], s_lo[warp * RW + sub][8 * at + i] = lo[i];
    __syncthreads();
    int8_t* rb = bounds + ((int64_t)id * s.H + h) * bounds_bytes(D);
    constexpr int C = (D + NTHR - 1) / NTHR;          // channels a thread
    float top[C], low[C], m = 0.0f;
    const bool grown = slot0 > 0;                     // begun by an earlier call: its bounds stand
    const float unit = grown ? pow2(min(max(*reinterpret_cast<const int*>(rb + 2 * D), -126), 127)) : 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int c = threadIdx.x + i * NTHR;
        top[i] = low[i] = 0.0f;
        if (c >= D) continue;
        float a = s_hi[0][c], z = s_lo[0][c];
        for (int w = 1; w < W * RW; ++w) a = fmaxf(a, s_hi[w][c]), z = fminf(z, s_lo[w][c]);
        a = fminf(a, kF16Max);
        z = fmaxf(z, -kF16Max);
        a = fmaxf(a, -kF16Max);
        z = fminf(z, kF16Max);
        if (grown) a = fmaxf(a, (float)rb[c] * unit), z = fminf(z, (float)rb[D + c] * unit);
        top[i] = a;
        low[i] = z;
        m = fmaxf(m, fmaxf(fabsf(a), fabsf(z)));
    }
    m = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(m)));
    if (lane == 0) s_m[warp] = m;
    __syncthreads();                                  // also: every old bound has been read
    m = s_m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, s_m[w]);
    int e = -126;
    if (m > 0.0f) {
        const float f = frexpf(m, &e);
        e = max(e - 7 + (f > 127.0f / 128.0f ? 1 : 0), -126);
    }
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int c = threadIdx.x + i * NTHR;
        if (c < D) {
            rb[c] = (int8_t)ceilf(top[i] * inv);
            rb[D + c] = (int8_t)floorf(low[i] * inv);
        }
    }
    if (threadIdx.x == 0) *reinterpret_cast<int*>(rb + 2 * D) = e;
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
    constexpr int64_t kVec = 16 / (int64_t)sizeof(X);     // elements of a 16-byte load
    const auto fits = [](const void* p, Strides x) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && x.b % kVec == 0 && x.t % kVec == 0 && x.h % kVec == 0;
    };
    const int vec = fits(K, ks) && fits(V, vs);
    // A step writes a token or a few of each sequence: two warps a page then start sooner than eight.
    if (s.T <= 4)
        write_kernel<X, D, 2><<<(unsigned)grid, 64, 0, st>>>(s, (const X*)K, (const X*)V, ks, vs, vec, pool, bounds,
                                                             table, start, count, touched, err);
    else
        write_kernel<X, D, 8><<<(unsigned)grid, 256, 0, st>>>(s, (const X*)K, (const X*)V, ks, vs, vec, pool,
                                                              bounds, table, start, count, touched, err);
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
