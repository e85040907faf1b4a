// asa_cache_store.cu -- quantising keys and values into the 4-bit paged cache,
// keeping the pages' bounds, and reading both back.
//
// Per group of 32 channels: offset z = fp16(min), scale s = fp16((max - z) * fl(1/15)),
// not below 0, code n = rint((x - z)/s) clipped to 0..15; a value reads back as z + n s (one
// rounding to fp32: n s is exact there), then as bf16 where asked.
//
// Measured, 65536 tokens of 8 key heads, d 128, bf16 (268 MB on the one side, 84 MB on
// the other; 54 us at a copy's rate): written in 90 us, 3.9 TB/s (about
// twelve instructions an element, most of them minima, maxima and the exact quotient, issued in 62 % of
// the cycles by 42 % of the warps that an SM holds: neither issue slots nor bytes alone bound it);
// read in 55 us, 6.4 TB/s, the copy's rate.  The bounds of its 1024 pages 9 us.  One token of each of 8 sequences: 3.5 us to write, a launch and
// three loads that wait for one another.
#include "asa_cache.h"

#include <type_traits>

namespace asa {
namespace cache {
namespace {

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Eight neighbouring channels: words as they lie in memory, values as fp32, and the
// lane-wise larger (NaN aside) and smaller (which keeps a NaN) of two.
template <typename X>
struct Eight;
template <>
struct Eight<float> {
    float x[8];
    template <bool VEC>
    __device__ __forceinline__ void load(const float* p) {
        if constexpr (VEC) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __ldg(p + i);
        }
    }
    __device__ __forceinline__ void fill(float v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v;
    }
    __device__ __forceinline__ float at(int i) const { return x[i]; }
    __device__ __forceinline__ bool nan() const {
        bool n = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) n |= x[i] != x[i];
        return n;
    }
    __device__ __forceinline__ void raise(const Eight& o) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaxf(x[i], o.x[i]);
    }
    __device__ __forceinline__ void lower(const Eight& o) {      // keeps a NaN
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("min.NaN.f32 %0, %0, %1;" : "+f"(x[i]) : "f"(o.x[i]));
    }
    __device__ __forceinline__ void nan_to_zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? 0.0f : x[i];
    }
};
template <>
struct Eight<__nv_bfloat16> {
    uint32_t w[4];
    template <bool VEC>
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        if constexpr (VEC) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __ldg(e + 2 * i) | (uint32_t)__ldg(e + 2 * i + 1) << 16;
        }
    }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __byte_perm(__float_as_uint(x), 0u, 0x3232);
    }
    __device__ __forceinline__ float at(int i) const {
        return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    __device__ __forceinline__ bool nan() const {     // a magnitude above infinity's carries into the sign
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n |= (w[i] & 0x7fff7fffu) + 0x007f007fu;
        return (n & 0x80008000u) != 0u;
    }
    __device__ __forceinline__ void raise(const Eight& o) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 c = __hmax2(reinterpret_cast<const __nv_bfloat162&>(w[i]), reinterpret_cast<const __nv_bfloat162&>(o.w[i]));
            w[i] = reinterpret_cast<const uint32_t&>(c);
        }
    }
    __device__ __forceinline__ void lower(const Eight& o) {      // keeps a NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 c = __hmin2_nan(reinterpret_cast<const __nv_bfloat162&>(w[i]), reinterpret_cast<const __nv_bfloat162&>(o.w[i]));
            w[i] = reinterpret_cast<const uint32_t&>(c);
        }
    }
    __device__ __forceinline__ void nan_to_zero() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((w[i] & 0x7fffu) > 0x7f80u) w[i] &= 0xffff0000u;
            if ((w[i] & 0x7fff0000u) > 0x7f800000u) w[i] &= 0xffffu;
        }
    }
};

// A group of 32 channels, all in one lane: codes (the first channel in the lowest
// four bits of the first word) and scale (low half) and offset.
//
// (x - z) / s is formed as Markstein does it (IBM J. Res. Dev. 34, 1990): with the
// correctly rounded reciprocal, a product, its exact remainder and one correction
// give the correctly rounded quotient.  So halves, which are not rare between
// numbers of few bits, go to the even code as the format's division has them.
// Adding 1.5 * 2^23 rounds to whole numbers.
template <typename X>
__device__ __forceinline__ void quantise(const Eight<X> (&x)[4], uint32_t (&codes)[4], uint32_t& grid) {
    constexpr float kMagic = 12582912.0f;
    Eight<X> least = x[0], most = x[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        least.lower(x[i]);
        most.raise(x[i]);
    }
    const bool nan = least.nan();
    float lo = least.at(0), hi = most.at(0);
#pragma unroll
    for (int i = 1; i < 8; ++i) lo = fminf(lo, least.at(i)), hi = fmaxf(hi, most.at(i));
    bool plain = lo >= -kF16Max && hi <= kF16Max;
    lo = fminf(fmaxf(lo, -kF16Max), kF16Max);
    hi = fminf(fmaxf(hi, -kF16Max), kF16Max);
    const __half zh = __float2half_rn(lo);
    const float z = __half2float(zh);
    // (below zero where a group of equal numbers has its offset rounded up)
    const __half sh = __float2half_rn(fmaxf(__fmul_rn(hi - z, kFifteenth), 0.0f));
    const float s = __half2float(sh), inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
    grid = nan ? 0x7fff7fffu : __half_as_ushort(sh) | (uint32_t)__half_as_ushort(zh) << 16;
    // with the offset rounded up far enough, or the scale rounded down, codes would leave 0..15
    plain &= lo - z >= -0.25f * s && hi - z <= 15.25f * s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float r[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {              // two at a time
            const float2 y = __fadd2_rn(make_float2(x[i].at(j), x[i].at(j + 1)), make_float2(-z, -z));
            const float2 inv2 = make_float2(inv, inv), q = __fmul2_rn(y, inv2);
            const float2 rest = __ffma2_rn(q, make_float2(-s, -s), y);
            const float2 n = __fadd2_rn(__fadd2_rn(__ffma2_rn(rest, inv2, q), make_float2(kMagic, kMagic)), make_float2(-kMagic, -kMagic));
            r[j] = n.x, r[j + 1] = n.y;
        }
        if (!plain)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float c = fminf(fmaxf(x[i].at(j), -kF16Max), kF16Max);
                r[j] = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(c - z, s)), 0.0f), 15.0f) : 0.0f;
            }
        uint32_t out = 0;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const float sum = fmaf(fmaf(fmaf(r[j + 3], 16.0f, r[j + 2]), 16.0f, r[j + 1]), 16.0f, r[j]);
            out |= (__float_as_uint(sum + kMagic) & 0xffffu) << (4 * j);
        }
        codes[i] = out;
    }
}

// One CTA a (sequence, touched page, key head): its tokens' keys and values, a
// group of 32 channels a lane at a time, laid out in shared memory as in the
// record and copied from there 16 bytes a lane; then the page's bounds, from the
// keys (in L1 by then).
template <typename X, int D, int NTHR>
__global__ void __launch_bounds__(NTHR) write_kernel(Shape s, const X* __restrict__ K, const X* __restrict__ V,
                                                     Strides ks, Strides vs, int vec, uint8_t* __restrict__ pool,
                                                     int8_t* __restrict__ bounds, const int32_t* __restrict__ table,
                                                     const int32_t* __restrict__ start,
                                                     const int32_t* __restrict__ count, int touched, int page_shift,
                                                     int* err) {
    constexpr int NG = D / 32, LR = D / 8, RB = row_bytes(D), PB = par_bytes(D), W = NTHR / 32;
    constexpr int SETS = NTHR / LR;                   // token sets that bounds are first taken over
    extern __shared__ __align__(16) uint8_t s_rec[];  // rows of codes and of scales: [2][page][RB], [2][page][PB]
    __shared__ float s_hi[SETS][D], s_lo[SETS][D];
    __shared__ float s_m[W];
    follow();
    const unsigned bj = blockIdx.x / (unsigned)s.H;
    const int h = blockIdx.x - bj * s.H, b = bj / (unsigned)touched, j = bj - b * touched;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int begin = __ldg(start + b), n = count ? min(max(__ldg(count + b), 0), s.T) : s.T;
    // the j-th of the pages that positions begin .. begin + n - 1 lie in, and the tokens there:
    // `from` of the call's, `rows` of them, the first in slot `slot0`
    const int page_no = (begin >> page_shift) + j, into = (begin & (s.P - 1)) - j * s.P;   // (begin - the page's first)
    const int from = max(0, -into), slot0 = max(0, into), rows = min(n - from, s.P - slot0);
    if (rows <= 0) return;
    int id = -1;
    if (page_no >= 0 && page_no < s.width) id = __ldg(table + (int64_t)b * s.width + page_no);
    if (id < 0 || id >= s.pages) {
        if (tid == 0 && err) atomicCAS(err, 0, ASA_ERR_INVALID);
        return;
    }
    uint8_t* rec = pool + ((int64_t)id * s.H + h) * s.rec;
    const X* kp = K + b * ks.b + (int64_t)from * ks.t + h * ks.h;
    const X* vp = V + b * vs.b + (int64_t)from * vs.t + h * vs.h;
    uint8_t* const s_par = s_rec + 2 * s.P * RB;
    auto body = [&](auto vec_c) {
        constexpr bool VEC = decltype(vec_c)::value;
        auto quantise_part = [&](auto part_c, const X* base, int64_t stride) {
            constexpr int part = decltype(part_c)::value;   // keys, values
            for (int i = tid; i < rows * NG; i += NTHR) {
                const int r = i / NG, g = i % NG;
                const X* src = base + r * stride + 32 * g;
                Eight<X> x[4];
                uint32_t codes[4], grid;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k].template load<VEC>(src + 8 * k);
                quantise<X>(x, codes, grid);
                uint8_t* to = s_rec + (part * s.P + r) * RB;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (part == 1) {
                        *reinterpret_cast<uint16_t*>(to + 2 * k * 2 * NG + 2 * g) = (uint16_t)codes[k];
                        *reinterpret_cast<uint16_t*>(to + (2 * k + 1) * 2 * NG + 2 * g) = (uint16_t)(codes[k] >> 16);
                    } else {
                        *reinterpret_cast<uint32_t*>(to + k * 4 * NG + 4 * g) = codes[k];
                    }
                }
                uint16_t* par = reinterpret_cast<uint16_t*>(s_par + (part * s.P + r) * PB) + g;
                par[0] = (uint16_t)grid;
                par[NG] = (uint16_t)(grid >> 16);
            }
        };
        quantise_part(std::integral_constant<int, 0>{}, kp, ks.t);
        quantise_part(std::integral_constant<int, 1>{}, vp, vs.t);
        // bounds of this thread's eight channels over its set of tokens
        const int set = tid / LR, c8 = tid % LR;
        if (set < SETS) {
            Eight<X> hi, lo;
            hi.fill(-INFINITY);
            lo.fill(INFINITY);
#pragma unroll 4
            for (int r = set; r < rows; r += SETS) {
                Eight<X> x;
                x.template load<VEC>(kp + r * ks.t + 8 * c8);
                hi.raise(x);
                lo.lower(x);
            }
            if (lo.nan()) {                           // again, with NaN as 0
                hi.fill(-INFINITY);
                lo.fill(INFINITY);
                for (int r = set; r < rows; r += SETS) {
                    Eight<X> x;
                    x.template load<VEC>(kp + r * ks.t + 8 * c8);
                    x.nan_to_zero();
                    hi.raise(x);
                    lo.lower(x);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                *reinterpret_cast<float4*>(&s_hi[set][8 * c8 + i]) = make_float4(hi.at(i), hi.at(i + 1), hi.at(i + 2), hi.at(i + 3));
                *reinterpret_cast<float4*>(&s_lo[set][8 * c8 + i]) = make_float4(lo.at(i), lo.at(i + 1), lo.at(i + 2), lo.at(i + 3));
            }
        }
    };
    if (vec) body(std::true_type{}); else body(std::false_type{});
    __syncthreads();
    // rows to the record
    constexpr int CW = RB / 16;                       // 16-byte pieces of a row of codes
    for (int i = tid; i < 2 * rows * CW; i += NTHR) {
        const int piece = i % CW, row = i / CW, part = row >= rows, r = part ? row - rows : row, slot = slot0 + r;
        *reinterpret_cast<uint4*>(rec + part * (s.rec / 2) + slot / kBlock * block_bytes(D) + slot % kBlock * RB + 16 * piece) =
            *reinterpret_cast<const uint4*>(s_rec + (part * s.P + r) * RB + 16 * piece);
    }
    for (int i = tid; i < 2 * rows * NG; i += NTHR) {
        const int piece = i % NG, row = i / NG, part = row >= rows, r = part ? row - rows : row, slot = slot0 + r;
        *reinterpret_cast<uint32_t*>(rec + part * (s.rec / 2) + slot / kBlock * block_bytes(D) + kBlock * RB + slot % kBlock * PB + 4 * piece) =
            *reinterpret_cast<const uint32_t*>(s_par + (part * s.P + r) * PB + 4 * piece);
    }
    int8_t* rb = bounds + ((int64_t)id * s.H + h) * bounds_bytes(D);
    constexpr int C = (D + NTHR - 1) / NTHR;          // channels a thread
    float top[C], low[C], m = 0.0f;
    const bool grown = slot0 > 0;                     // begun by an earlier call: its bounds stand
    const float unit = grown ? pow2(min(max(*reinterpret_cast<const int*>(rb + 2 * D), -126), 127)) : 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int c = tid + i * NTHR;
        top[i] = low[i] = 0.0f;
        if (c >= D) continue;
        float a = s_hi[0][c], z = s_lo[0][c];
#pragma unroll
        for (int w = 1; w < SETS; ++w) a = fmaxf(a, s_hi[w][c]), z = fminf(z, s_lo[w][c]);
        a = fmaxf(fminf(a, kF16Max), -kF16Max);
        z = fmaxf(fminf(z, kF16Max), -kF16Max);
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
        const int c = tid + i * NTHR;
        if (c < D) {
            rb[c] = (int8_t)ceilf(top[i] * inv);
            rb[D + c] = (int8_t)floorf(low[i] * inv);
        }
    }
    if (tid == 0) *reinterpret_cast<int*>(rb + 2 * D) = e;
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

// Four lanes a row (a token's keys and values of one head): a lane's stretch of a row
// of codes holds eight channels of every group, 8 q .. of quarter q, in one load of keys
// and one of values, and it needs the scales and offsets of all groups, one more load each.
// kReadRows rows a lane: the places of all, then what they hold, then the outputs, so that
// the loads of several are under way at once.
constexpr int kReadRows = 2;
template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {   // N words at an N-word (N = 3: a word) boundary
    if constexpr (N == 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    }
}
template <typename X, int D>
__global__ void __launch_bounds__(256) read_kernel(Shape s, const uint8_t* __restrict__ pool,
                                                   const int32_t* __restrict__ table,
                                                   const int32_t* __restrict__ start,
                                                   const int32_t* __restrict__ count, X* __restrict__ K,
                                                   X* __restrict__ V, unsigned chunks, int page_shift, int* err) {
    constexpr int NG = D / 32, RB = row_bytes(D), PB = par_bytes(D), ROWS = 64;   // rows of the CTA at a time
    follow();
    const unsigned b = blockIdx.x / chunks, chunk = blockIdx.x - b * chunks;
    const unsigned q = threadIdx.x & 3, first = chunk * (kReadRows * ROWS) + threadIdx.x / 4;
    const unsigned of = (unsigned)s.T * s.H;          // rows (token, head) of the sequence
    const int begin = __ldg(start + b), n = count ? __ldg(count + b) : s.T;
    const uint8_t* at[kReadRows];                     // their blocks
    unsigned in[kReadRows];                           // and rows there
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
        const unsigned row = first + u * ROWS, t = row / (unsigned)s.H, h = row - t * s.H;
        at[u] = nullptr;
        in[u] = 0;
        if (row >= of || (int)t >= n) continue;
        const long long pos = (long long)begin + t;
        int id = -1;
        if (pos >= 0 && pos >> page_shift < s.width) id = __ldg(table + (int64_t)b * s.width + (pos >> page_shift));
        if (id >= 0 && id < s.pages) {
            const unsigned slot = (unsigned)pos & (s.P - 1);
            at[u] = pool + ((int64_t)id * s.H + h) * s.rec + slot / kBlock * block_bytes(D);
            in[u] = slot % kBlock;
        } else if (err) {
            atomicCAS(err, 0, ASA_ERR_INVALID);
        }
    }
    uint32_t code[kReadRows][2][NG], par[kReadRows][2][NG];
#pragma unroll
    for (int u = 0; u < kReadRows; ++u)
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int g = 0; g < NG; ++g) code[u][part][g] = par[u][part][g] = 0u;
            if (!at[u]) continue;
            const uint8_t* block = at[u] + part * (s.rec / 2);
            load_words<NG>(block + in[u] * RB + q * 4 * NG, code[u][part]);
            load_words<NG>(block + kBlock * RB + in[u] * PB, par[u][part]);
        }
    auto half = [](const uint32_t (&w)[NG], int i) {
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
    };
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
        const unsigned row = first + u * ROWS;
        if (row >= of) break;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            X* to = (part ? V : K) + ((int64_t)b * of + row) * D + 8 * q;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                // keys: a word a group; values: a half word a group and four channels
                uint32_t w;
                if (part == 0) w = code[u][0][g];
                else if (NG % 2 == 0) w = __byte_perm(code[u][1][g / 2], code[u][1][(NG + g) / 2], g & 1 ? 0x7632 : 0x5410);
                else w = ((code[u][1][g / 2] >> (g & 1 ? 16 : 0)) & 0xffffu) |
                         ((code[u][1][(NG + g) / 2] >> ((NG + g) & 1 ? 16 : 0)) << 16);
                const float scale = half(par[u][part], g), offset = half(par[u][part], NG + g);
                float x[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) x[c] = fmaf((float)((w >> (4 * c)) & 15u), scale, offset);
                store8<X>(to + 32 * g, x);
            }
        }
    }
}

__global__ void __launch_bounds__(256) bounds_kernel(Shape s, const int8_t* __restrict__ bounds,
                                                     const int32_t* __restrict__ pages, int n,
                                                     float* __restrict__ upper, float* __restrict__ lower,
                                                     int* err) {
    follow();
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
    int page_shift = 4;
    while (1 << page_shift < s.P) ++page_shift;
    const long long grid = (long long)s.B * touched * s.H;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    constexpr int64_t kVec = 16 / (int64_t)sizeof(X);     // elements of a 16-byte load
    const auto fits = [](const void* p, Strides x) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && x.b % kVec == 0 && x.t % kVec == 0 && x.h % kVec == 0;
    };
    const int vec = fits(K, ks) && fits(V, vs);
    const size_t smem = (size_t)2 * s.P * (row_bytes(D) + par_bytes(D));   // 20 KB at most
    // Two warps a page where the page is small and pages are many, else four (which
    // shorten the way of one).  Us with 64 threads and with 128, 8 key heads, bfloat16: head
    // size 128, 65536 tokens in pages of 16 105.7 and 155.7, of 32 91.5 and 103.3, of 64 91.0
    // and 89.0; 2048 tokens in pages of 32 6.4 and 5.5, 512 in pages of 64 8.7 and 5.4.
    const bool two = s.P * D <= 4096 && grid >= 2048;
    const auto kernel = two ? write_kernel<X, D, 64> : write_kernel<X, D, 128>;
    return launch(kernel, (unsigned)grid, two ? 64 : 128, smem, st, s, (const X*)K, (const X*)V, ks, vs, vec, pool,
                  bounds, table, start, count, touched, page_shift, err);
}

template <typename X, int D>
cudaError_t read_as(const Shape& s, const uint8_t* pool, const int32_t* table, const int32_t* start,
                    const int32_t* count, void* K, void* V, int* err, cudaStream_t st) {
    constexpr int kRows = kReadRows * 64;             // a CTA
    const long long chunks = ((long long)s.T * s.H + kRows - 1) / kRows, grid = chunks * s.B;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    int page_shift = 4;
    while (1 << page_shift < s.P) ++page_shift;
    return launch(read_kernel<X, D>, (unsigned)grid, 256, 0, st, s, pool, table, start, count, (X*)K, (X*)V,
                  (unsigned)chunks, page_shift, err);
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
    return launch(bounds_kernel, (unsigned)grid, 256, 0, st, s, bounds, pages, n, upper, lower, err);
}

}  // namespace cache
}  // namespace asa
