// asa_cache_chunk.cu -- attention of many query rows a key head over the 4-bit
// cache: chunks of prompts, on tcgen05.
//
// An item is 128 query rows of one key head; its keys are walked in tiles of 128
// tokens, and the items' tiles are cut into equal runs, one a CTA, as in
// asa_cache_attend.cu (whose combine_kernel joins what a cut divides).  A CTA is one
// to an SM: a warp fetches the tiles' records (bulk copies), eight warps turn their
// codes into fp16 keys and values laid out for the tensor cores (128-byte swizzle),
// one issues S = Q K^T and O += P V, and eight take the softmax, a row each to
// two threads (half the keys each), P going back to tensor memory over its scores.
// S of the next tile is issued before P V of the last, and keys, values and scores
// are double-buffered, so that conversion, softmax and products of three tiles
// overlap.
//
// fp16 is chosen for all operands.  A key is (c + n s) + (z - c), c = -7.5 s: the first
// part, of the size of its group's spread, rounds to fp16's 11 bits (bf16 would keep 8),
// a 270th of a code's step at most; the second enters as a product of its own, z and c with
// the group sums of q in two fp16 halves each, so that an offset far above the
// scale takes no bits from the codes.  A value is z + n s, rounded once to 11 bits: that
// error is weighted as the value is, and lies below the output's.  P keeps 11 bits
// as well, of weights down to 2^-14 of its row's reference.  A row's reference moves only
// when a weight outgrows it (kMost); O in tensor memory is then rescaled by the
// rows' own warps.
//
// Measured, 32 heads over 8 key heads, 8192 tokens, d 128: 512 query tokens (66.6 GFLOP)
// 122 us, 546 TFLOP/s; of 4 sequences 485 us, 549 (0.33 of cuBLAS); d 64, 2048 tokens
// (120 GFLOP) 366 us, 329.  A tile takes 1.8 us, of which the products are 0.8: the
// exponentials and the conversion of codes, which do not depend on d and on the rows
// respectively, take the SM's other issue slots.  Starting and ending an item is some 10 us.
//
// Channels are not moved into their order: keys and queries share the order in
// which masking words yields them, and the output's is undone as it is stored.
#include "asa_cache_attend.cuh"

#include <type_traits>

namespace asa {
namespace cache {
namespace {

using namespace sm100;

constexpr int kRows = 128, kTokens = 128, kBlocks = kTokens / kBlock;
constexpr int kBox = 16384;                           // 128 rows of 128 bytes
constexpr int kEdge = 128 * 32;                       // 128 rows of the offsets' product: two columns of 16 bytes
constexpr int kWarps = 18, kThreads = kWarps * 32;
constexpr int kChunkCost = 4;                         // Plan::item_cost
constexpr int kMaxUnits = 1184;                       // units whose prefix sums a CTA keeps

// Warps: 0 fetches, 1 issues the products; 2, 3, 12..17 convert; 4..11 take the
// softmax (a warp reaches the 32 lanes of tensor memory that its number mod 4 names).
struct Bars {
    uint64_t staged_full[2], staged_free[2], k_ready[2], k_free[2], v_ready[2], v_free[2];
    uint64_t s_full[2], p_full[2], pv_done[2], q_ready, o_done, o_free, drain;
};
struct TileInfo { int base, present; };               // first position; the 16-token blocks that are there

template <int D>
struct ChunkSmem {
    static constexpr int kTileBytes = D * kTokens * 2;
    alignas(1024) uint8_t q[kTileBytes];
    alignas(1024) uint8_t k[2][kTileBytes];
    alignas(1024) uint8_t v[2][kTileBytes];
    // rows of 16 fp16: of queries the group sums hi, lo, -hi, -lo; of keys z, z, c, c
    alignas(128) uint8_t qz[kEdge];
    alignas(128) uint8_t kz[2][kEdge];
    alignas(128) uint8_t staged[2][2 * kBlocks * block_bytes(D)];
    float row[2][2][kRows];                           // maxima of a tile's halves; sums; queries' maxima
    uint16_t nan[2][D / 32][kBlocks];                 // of a tile some rows see in part: value groups holding a NaN
    TileInfo info[8];
    Bars b;
    uint32_t tmem;
    int64_t scan[kWarps];
    int64_t pref[kMaxUnits + 1];
};

struct Seg { int u, item, from, n, of; };

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int a_mn, int b_mn) {
    return idesc_bf16(M, N, a_mn, b_mn) & ~((7u << 7) | (7u << 10));   // operands fp16
}

// The next segment of the run [x, x1) (false at its end).
__device__ __forceinline__ bool next_segment(const Args& a, const int64_t* pref, int64_t& x, int64_t x1, Seg& g) {
    const int per = a.p.tiles * a.s.H;
    if (!a.p.split) {
        if (x >= x1) return false;
        const int u = blockIdx.x / per, of = unit_tiles(a, u);
        g = Seg{u, (int)(blockIdx.x % per), 0, of, of};
        x = x1;
        return true;
    }
    while (x < x1) {
        int lo = 0, hi = a.p.U;                       // the last unit that starts at or before x
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pref[mid] <= x) lo = mid; else hi = mid;
        }
        const int of = (int)((pref[lo + 1] - pref[lo]) / per) - a.p.item_cost;
        const int item = (int)((x - pref[lo]) / (of + a.p.item_cost));
        const int64_t begin = pref[lo] + (int64_t)item * (of + a.p.item_cost) + a.p.item_cost;
        const int from = (int)max((int64_t)0, x - begin), to = (int)min((int64_t)of, x1 - begin);
        x = min(x1, begin + of);
        if (to > from) {
            g = Seg{lo, item, from, to - from, of};
            return true;
        }
    }
    return false;
}

// Eight codes of a word as fp16 values z + n s: nibbles (0, 4), (1, 5), (2, 6), (3, 7).
// OR-ing a nibble into 1024's mantissa gives 1024 + n, or 1024 + 16 n.
template <bool CLIP>
__device__ __forceinline__ void values_of(uint32_t w, uint32_t s, uint32_t z, uint32_t (&out)[4]) {
    const __half2 sh = *reinterpret_cast<const __half2*>(&s), zh = *reinterpret_cast<const __half2*>(&z);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = ((i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
        const __half2 m = *reinterpret_cast<const __half2*>(&x);
        const __half2 n = i & 1 ? __hfma2(m, __float2half2_rn(0.0625f), __float2half2_rn(-64.0f))
                                : __hsub2(m, __float2half2_rn(1024.0f));
        __half2 v = __hfma2(n, sh, zh);
        if constexpr (CLIP) v = __hmin2_nan(v, __float2half2_rn(kF16Max));   // the largest may round past fp16
        out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
// -7.5 s, and no less than fp16's least: what a key's codes are about the middle of.
__device__ __forceinline__ uint32_t middle_of(uint32_t s) {
    const __half2 c = __hmax2_nan(__hmul2(*reinterpret_cast<const __half2*>(&s), __float2half2_rn(-7.5f)), __float2half2_rn(-kF16Max));
    return *reinterpret_cast<const uint32_t*>(&c);
}
// Whether some value 15 s + z passes fp16's largest (or is NaN already).
__device__ __forceinline__ bool passes_largest(uint32_t s, uint32_t z) {
    const __half2 top = __hfma2(__float2half2_rn(15.0f), *reinterpret_cast<const __half2*>(&s), *reinterpret_cast<const __half2*>(&z));
    const uint32_t h = *reinterpret_cast<const uint32_t*>(&top);
    return (h & 0x7c00u) == 0x7c00u || (h & 0x7c000000u) == 0x7c000000u;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const __grid_constant__ Args a) {
    constexpr int NG = D / 32, NP = NG / 2, BB = block_bytes(D), RB = row_bytes(D), PB = par_bytes(D);
    constexpr uint32_t kO = 256;                      // tensor memory: scores (P over them) 2 x 128 columns, then O
    extern __shared__ uint8_t smem_raw[];
    auto& sm = *reinterpret_cast<ChunkSmem<D>*>(smem_raw + (-smem_u32(smem_raw) & 1023u));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Shape& s = a.s;
    const int per = a.p.tiles * s.H;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.b.staged_full[i], 1);
            mbar_init(&sm.b.staged_free[i], 8);
            mbar_init(&sm.b.k_ready[i], 8);
            mbar_init(&sm.b.k_free[i], 1);
            mbar_init(&sm.b.v_ready[i], 8);
            mbar_init(&sm.b.v_free[i], 1);
            mbar_init(&sm.b.s_full[i], 1);
            mbar_init(&sm.b.p_full[i], 8);
            mbar_init(&sm.b.pv_done[i], 1);
        }
        mbar_init(&sm.b.q_ready, 8);
        mbar_init(&sm.b.o_done, 1);
        mbar_init(&sm.b.o_free, 8);
        mbar_init(&sm.b.drain, 1);
        fence_barrier_init();
    }
    follow();
    // this CTA's run of all the items' tiles
    int64_t x = 0, x1 = 1;
    if (a.p.split) {
        int64_t total = 0;
        for (int base = 0; base < a.p.U; base += kThreads) {
            int64_t v = 0, sum;
            if (base + tid < a.p.U) {
                const int n = unit_tiles(a, base + tid);
                if (n) v = (int64_t)(n + a.p.item_cost) * per;
            }
            const int64_t e = total + block_scan<kThreads>(v, sm.scan, &sum);
            if (base + tid < a.p.U) {
                sm.pref[base + tid] = e;
                if (blockIdx.x == 0) a.w.run[1 + base + tid] = e;
            }
            total += sum;
        }
        if (tid == 0) sm.pref[a.p.U] = total;
        const int64_t run = max((int64_t)a.p.least, (total + gridDim.x - 1) / gridDim.x);
        if (blockIdx.x == 0 && tid == 0) a.w.run[0] = run;
        x = run * blockIdx.x;
        x1 = min(x + run, total);
        if (x >= x1) return;
    }
    if (warp == 1) {
        tmem_alloc(&sm.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;

    auto wait = [&](uint64_t& bar, uint32_t parity) { wait_full(&bar, parity & 1u, s.naps, a.err); };
    auto position = [&](int u, int row) -> int {      // of an item's row (its tile's first row added)
        if (row >= a.p.R) return -1;
        return (int)max(-1ll, min((long long)__ldg(a.lengths + u) - s.T + row / s.G, (long long)s.width * s.P - 1));
    };
    // what all warps of a CTA know of a segment
    struct View { int h, row0, pos_lo, pos_hi, n; };
    auto view_of = [&](const Seg& g) {
        View v;
        v.h = g.item / a.p.tiles;
        v.row0 = g.item % a.p.tiles * kRows;
        v.pos_lo = position(g.u, v.row0);
        v.pos_hi = position(g.u, min(v.row0 + kRows, a.p.R) - 1);      // rows stand in order
        // tiles that some row sees
        v.n = min(g.n, max(0, (v.pos_hi < 0 ? 0 : v.pos_hi / kTokens + 1) - g.from));
        return v;
    };
    auto arrive = [&](uint64_t& bar) {                // a warp's
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar);
    };

    uint32_t j = 0;                                   // tiles, counted through the launch
    uint32_t segs = 0;
    Seg g;
    if (warp == 0) {
        // ---- the tiles' records ---------------------------------------------------
        const int pieces = kTokens / s.P, blocks = s.P / kBlock;       // pages a tile, blocks a page (P <= 128)
        bool lost = false;                            // a wait gave up: no more is fetched
        while (!lost && next_segment(a, sm.pref, x, x1, g)) {
            const View v = view_of(g);
            const int32_t* table = a.table + (int64_t)g.u * s.width;
            auto look_up = [&](int i) {               // this lane's page of the i-th tile: its id, -1 where none is to be read
                const int page = (g.from + i) * pieces + lane;
                if (lane >= pieces || page >= s.width || page * s.P > v.pos_hi) return -1;
                const int id = __ldg(table + page);
                if (id >= 0 && id < s.pages) return id;
                if (a.err) atomicCAS(a.err, 0, ASA_ERR_INVALID);
                return -1;
            };
            int next = v.n ? look_up(0) : -1;
            for (int i = 0; i < v.n; ++i, ++j) {
                const int id = next, st = j & 1;
                if (i + 1 < v.n) next = look_up(i + 1);
                // read by all that convert it, and (should one of them have given up) landed
                lost = !__all_sync(~0u, wait_full(&sm.b.staged_free[st], ((j >> 1) ^ 1u) & 1u, s.naps, a.err) &&
                                            wait_full(&sm.b.staged_full[st], ((j >> 1) ^ 1u) & 1u, s.naps, a.err));
                if (lost) break;
                const uint32_t votes = __ballot_sync(~0u, id >= 0);
                if (lane == 0) {
                    uint32_t present = 0;
                    for (int p = 0; p < pieces; ++p)
                        if (votes >> p & 1u) present |= ((1u << blocks) - 1u) << (p * blocks);
                    sm.info[j & 7] = TileInfo{(g.from + i) * kTokens, (int)present};
                    mbar_expect_tx(&sm.b.staged_full[st], __popc(votes) * 2 * blocks * BB);
                }
                __syncwarp();
                if (id >= 0) {
                    const uint8_t* src = a.pool + ((int64_t)id * s.H + v.h) * s.rec;
                    uint8_t* dst = sm.staged[st] + lane * blocks * BB;
                    bulk_load(dst, src, blocks * BB, &sm.b.staged_full[st]);
                    bulk_load(dst + kBlocks * BB, src + s.rec / 2, blocks * BB, &sm.b.staged_full[st]);
                }
            }
        }
        if (lost || timed_out(a.err))                 // no copy may outlive the CTA
            for (uint32_t i = 0; i < 2 && i < j; ++i) mbar_drain(&sm.b.staged_full[(j - 1 - i) & 1], ((j - 1 - i) >> 1) & 1u);
    } else if (warp == 1) {
        // ---- the products -----------------------------------------------------------
        constexpr uint32_t idS = idesc_f16(kRows, kTokens, 0, 0), idV = idesc_f16(kRows, D, 0, 1);
        const uint64_t dQ = sdesc(smem_u32(sm.q), 16, 1024), dQz = sdesc_plain(smem_u32(sm.qz), kEdge / 2, 128);
        auto k_step = [](int kk) { return (uint64_t)((((kk >> 2) * kBox) + (kk & 3) * 32) >> 4); };
        auto values = [&](uint32_t i, bool first) {   // O += P V of tile i
            const int b = i & 1;
            wait(sm.b.v_ready[b], i >> 1);
            wait(sm.b.p_full[b], i >> 1);
            tc_fence_after();
            if (lane == 0) {
                const uint64_t dV = sdesc(smem_u32(sm.v[b]), kBox, 1024);
#pragma unroll
                for (int kk = 0; kk < kTokens / 16; ++kk)
                    mma_bf16_ts(tmem + kO, tmem + b * 128 + kk * 16, dV + (uint64_t)((kk * 16 * 128) >> 4), idV, !first || kk > 0);
                mma_commit(&sm.b.pv_done[b]);
                mma_commit(&sm.b.v_free[b]);
            }
            __syncwarp();
        };
        while (next_segment(a, sm.pref, x, x1, g)) {
            const View v = view_of(g);
            wait(sm.b.q_ready, segs);
            wait(sm.b.o_free, segs ^ 1u);
            for (int i = 0; i < v.n; ++i, ++j) {
                const int b = j & 1;
                wait(sm.b.k_ready[b], j >> 1);
                tc_fence_after();
                if (lane == 0) {
                    const uint64_t dK = sdesc(smem_u32(sm.k[b]), 16, 1024);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        mma_bf16_ss(tmem + b * 128, dQ + k_step(kk), dK + k_step(kk), idS, kk > 0);
                    mma_bf16_ss(tmem + b * 128, dQz, sdesc_plain(smem_u32(sm.kz[b]), kEdge / 2, 128), idS, 1);
                    mma_commit(&sm.b.s_full[b]);
                    mma_commit(&sm.b.k_free[b]);
                }
                __syncwarp();
                if (i) values(j - 1, i == 1);
            }
            if (v.n) values(j - 1, v.n == 1);
            if (lane == 0) mma_commit(&sm.b.o_done);
            __syncwarp();
            ++segs;
        }
        if (lane == 0 && timed_out(a.err)) {          // a wait gave up: let the products finish
            mma_commit(&sm.b.drain);
            mbar_drain(&sm.b.drain, 0);
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 12) {
        // ---- softmax: row `row`, keys 64 half .. + 63 of each tile ------------------------
        const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);    // the warp's lanes (32 of them) in bits 16..
        auto all_rows = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        while (next_segment(a, sm.pref, x, x1, g)) {
            const View v = view_of(g);
            const int at = v.row0 + row, pos = position(g.u, at), tq = at / s.G, hq = v.h * s.G + at % s.G;
            // the queries, a power of two a row (fp16 holds bf16 exactly then, and the group sums,
            // below 2^15), in the keys' order
            float rf;
            {
                uint32_t w[NG][2][4];
                float big = 0.0f, sum = 0.0f;
                const __nv_bfloat16* src = a.Q + g.u * a.qs.b + tq * a.qs.t + hq * a.qs.h + 16 * half;
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {     // channels 32 i + 8 (2 half + k) ..
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[i][k][e] = 0u;
                        if (at < a.p.R && a.p.vec) {
                            const uint4 y = __ldg(reinterpret_cast<const uint4*>(src + 32 * i + 8 * k));
                            w[i][k][0] = y.x, w[i][k][1] = y.y, w[i][k][2] = y.z, w[i][k][3] = y.w;
                        } else if (at < a.p.R) {
                            const uint16_t* y = reinterpret_cast<const uint16_t*>(src + 32 * i + 8 * k);
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[i][k][e] = __ldg(y + 2 * e) | (uint32_t)__ldg(y + 2 * e + 1) << 16;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float y = __uint_as_float(w[i][k][e] << 16), z = __uint_as_float(w[i][k][e] & 0xffff0000u);
                            big = fmaxf(big, fmaxf(fabsf(y), fabsf(z)));
                            sum = fmaf(y, 0.0f, fmaf(z, 0.0f, sum));   // NaN from a NaN or an infinity
                        }
                    }
                sm.row[0][half][row] = sum != sum ? INFINITY : big;
                all_rows();
                big = fmaxf(big, sm.row[0][half ^ 1][row]);
                const bool bad = sum != sum || !(big < INFINITY);
                const int up = big == 0.0f || bad ? 0 : 9 - max((int)(__float_as_uint(big) >> 23) - 127, -117);
                const float f = bad ? NAN : pow2i(up);
                rf = factor_of(s.scale * kLog2e, -up, kMostFactor * 5.9604645e-8f);   // 2^56
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {  // channels e and e + 4 of the eight
                            const uint32_t lo = w[i][k][e >> 1], hi = w[i][k][2 + (e >> 1)];
                            const __half2 p = __floats2half2_rn(__uint_as_float(e & 1 ? lo & 0xffff0000u : lo << 16) * f,
                                                                __uint_as_float(e & 1 ? hi & 0xffff0000u : hi << 16) * f);
                            y[e] = *reinterpret_cast<const uint32_t*>(&p);
                        }
                        const int c = NG * (2 * half + k) + i;          // 16-byte piece of the row
                        *reinterpret_cast<uint4*>(sm.q + (c >> 3) * kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                            make_uint4(y[0], y[1], y[2], y[3]);
                    }
                all_rows();
                // the sums of half the groups, of the operands as they are
                uint32_t hi[NP], lo[NP];              // a group a half word
#pragma unroll
                for (int p = 0; p < NP; ++p) hi[p] = lo[p] = 0u;
#pragma unroll
                for (int j2 = 0; j2 < NP; ++j2) {
                    const int i = half * NP + j2;
                    float2 v2 = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int c = NG * k + i;
                        const uint4 y = *reinterpret_cast<const uint4*>(sm.q + (c >> 3) * kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4));
                        const uint32_t words[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v2 = __fadd2_rn(v2, __half22float2(*reinterpret_cast<const __half2*>(&words[e])));
                    }
                    const float own = v2.x + v2.y;
                    const __half h = __float2half_rn(own), l = __float2half_rn(own - __half2float(h));
                    hi[j2 >> 1] |= (uint32_t)__half_as_ushort(h) << (16 * (j2 & 1));
                    lo[j2 >> 1] |= (uint32_t)__half_as_ushort(l) << (16 * (j2 & 1));
                }
                uint8_t* edge = sm.qz + row * 16;
                if constexpr (NG == 4) {
                    *reinterpret_cast<uint32_t*>(edge + 4 * half) = hi[0];
                    *reinterpret_cast<uint32_t*>(edge + 8 + 4 * half) = lo[0];
                    *reinterpret_cast<uint32_t*>(edge + kEdge / 2 + 4 * half) = hi[0] ^ 0x80008000u;
                    *reinterpret_cast<uint32_t*>(edge + kEdge / 2 + 8 + 4 * half) = lo[0] ^ 0x80008000u;
                } else {
                    uint16_t* at2 = reinterpret_cast<uint16_t*>(edge) + half;
                    at2[0] = (uint16_t)hi[0], at2[2] = (uint16_t)lo[0];
                    at2[4] = (uint16_t)(hi[0] ^ 0x8000u), at2[6] = (uint16_t)(lo[0] ^ 0x8000u);
                    if (half) *reinterpret_cast<uint4*>(edge + kEdge / 2) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_async_smem();
                all_rows();                           // (also: sm.row may be written again)
                arrive(sm.b.q_ready);
            }
            float m = 0.0f, room = -INFINITY;         // as in asa_cache_attend.cu
            float2 l2 = make_float2(0.0f, 0.0f);      // the weights' sum, in two parts
            uint32_t nan_groups = 0;
            for (int i = 0; i < v.n; ++i, ++j) {
                const int b = j & 1;
                wait(sm.b.s_full[b], j >> 1);
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld32(lanes + b * 128 + half * 64, r[0]);
                tmem_ld32(lanes + b * 128 + half * 64 + 32, r[1]);
                const TileInfo info = sm.info[j & 7];
                const bool whole = info.present == 0xff && info.base + kTokens - 1 <= v.pos_lo;
                tmem_ld_wait();
                float top = -INFINITY;
                const float2 rf2 = make_float2(rf, rf), m2 = make_float2(-m, -m);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float2 y = __ffma2_rn(make_float2(__uint_as_float(r[c][k]), __uint_as_float(r[c][k + 1])), rf2, m2);
                        r[c][k] = __float_as_uint(y.x), r[c][k + 1] = __float_as_uint(y.y);
                    }
                if (!whole) {
                    const int see = pos - info.base - 64 * half;   // the last of this thread's keys that the row sees
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (32 * c + k > see || !(info.present >> (4 * half + 2 * c + (k >> 4)) & 1)) r[c][k] = 0xff800000u;
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int k = 0; k < 32; ++k) top = fmaxf(top, __uint_as_float(r[c][k]));
                sm.row[b][half][row] = top;
                all_rows();
                top = fmaxf(top, sm.row[b][half ^ 1][row]);
                if (__any_sync(~0u, top > room)) {    // (the same in both halves' warps)
                    float by = 0.0f;
                    const bool none = room == -INFINITY;      // no key of the row seen yet
                    if (top > room) by = top, room = kMost;   // the largest weight 1: fp16 has room below too
                    m += by;
                    // (a first reference may lie far below 0: nothing is summed yet that it could scale)
                    const float f = none ? 1.0f : exp2_fast(-by);
                    l2.x *= f, l2.y *= f;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[c][k] = __float_as_uint(__uint_as_float(r[c][k]) - by);
                    if (i) {                          // this half of O's channels, once the last product is in
                        wait(sm.b.pv_done[b ^ 1], (j - 1) >> 1);
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(lanes + kO + half * (D / 2) + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_st16(lanes + kO + half * (D / 2) + c, o);
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {     // 16 keys: eight columns over their scores
                        uint32_t p[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float y = exp2_fast(__uint_as_float(r[c][16 * e + 2 * k]));
                            const float z = exp2_fast(__uint_as_float(r[c][16 * e + 2 * k + 1]));
                            l2 = __fadd2_rn(l2, make_float2(y, z));
                            const __half2 two = __floats2half2_rn(y, z);
                            p[k] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        tmem_st8(lanes + b * 128 + half * 64 + 32 * c + 16 * e, p);
                    }
                if (!whole) {                         // NaN values that this row sees
                    wait(sm.b.v_ready[b], j >> 1);
                    const int see = min(max(pos - info.base + 1, 0), kTokens);
#pragma unroll
                    for (int k = 0; k < NG; ++k)
#pragma unroll
                        for (int e = 0; e < kBlocks; ++e) {
                            const int in = min(max(see - kBlock * e, 0), kBlock);
                            if (sm.nan[b][k][e] & ((1u << in) - 1u)) nan_groups |= 1u << k;
                        }
                }
                tmem_st_wait();
                tc_fence_before();
                arrive(sm.b.p_full[b]);
            }
            wait(sm.b.o_done, segs);
            tc_fence_after();
            float l = l2.x + l2.y;
            sm.row[0][half][row] = l;
            all_rows();
            l += sm.row[0][half ^ 1][row];
            const bool all = g.n == g.of, real = at < a.p.R;
            const int64_t slot = 2 * (int64_t)blockIdx.x + (g.from + g.n < g.of ? 1 : 0);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            __nv_bfloat16* out = a.O + (((int64_t)g.u * s.T + tq) * s.HQ + hq) * D;
            float* part = a.w.part + (slot * kRows + row) * D;
            if (!all && real && half == 0)
                *reinterpret_cast<float2*>(a.w.part_ml + (slot * kRows + row) * 2) = make_float2(room > -INFINITY ? m : kLow, l);
            // eight neighbouring channels of one group
            auto put = [&](int channel, const float (&y)[8]) {
                if (!real) return;
                if (all) {
                    __nv_bfloat162 z[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) z[k] = __floats2bfloat162_rn(y[2 * k] * inv, y[2 * k + 1] * inv);
                    *reinterpret_cast<uint4*>(out + channel) = *reinterpret_cast<uint4*>(z);
                } else {
                    *reinterpret_cast<float4*>(part + channel) = make_float4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<float4*>(part + channel + 4) = make_float4(y[4], y[5], y[6], y[7]);
                }
            };
#pragma unroll 1
            for (int c = 0; c < D / 64; ++c) {        // 32 of this half's columns at a time
                uint32_t o[32];
                tmem_ld32(lanes + kO + half * (D / 2) + 32 * c, o);
                tmem_ld_wait();
                // column q of a run of 4 NG: channel 4 run + i of group 2 p + e, q = 8 p + 2 i + e
                const int run0 = (half * (D / 2) + 32 * c) / (4 * NG);
#pragma unroll
                for (int k = 0; k < NG; ++k)
#pragma unroll
                    for (int two = 0; two < 32 / (4 * NG); two += 2) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float z = __uint_as_float(o[(two + (e >> 2)) * 4 * NG + 8 * (k >> 1) + 2 * (e & 3) + (k & 1)]);
                            y[e] = v.n == 0 ? 0.0f : nan_groups >> k & 1u ? NAN : z;
                        }
                        put(32 * k + 4 * (run0 + two), y);
                    }
            }
            tc_fence_before();
            all_rows();                               // (sm.row may be written again)
            arrive(sm.b.o_free);
            ++segs;
        }
    } else {
        // ---- codes to fp16: 16 tokens of each tile a warp ----------------------------------
        const int dq = warp < 4 ? warp - 2 : warp - 10;
        // where a lane's pieces of a key row and of a value row go (token lane % 8 of the warp's 16)
        const int tok = lane & 7, run = lane >> 3;
        uint32_t to_k[NG], to_v[2][NP];
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            const int c = NG * run + e;
            to_k[e] = (c >> 3) * kBox + (16 * dq + tok) * 128 + (((c & 7) ^ tok) << 4);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                const int c = NP * (run + 4 * q) + e;
                to_v[q][e] = (c >> 3) * kBox + (16 * dq + tok) * 128 + (((c & 7) ^ tok) << 4);
            }
        while (next_segment(a, sm.pref, x, x1, g)) {
            const View v = view_of(g);
            for (int i = 0; i < v.n; ++i, ++j) {
                const int st = j & 1;
                wait(sm.b.staged_full[st], j >> 1);
                const TileInfo info = sm.info[j & 7];
                const bool there = info.present >> dq & 1;
                const uint8_t* kb = sm.staged[st] + dq * BB;
                const uint8_t* vb = kb + kBlocks * BB;
                wait(sm.b.k_free[st], (j >> 1) ^ 1u);
                // keys: a lane eight channels of every group, of tokens lane % 8 and 8 on
                {
                    uint32_t w[2][NG], sc[2][NP], zo[2][NP], mid[2][NP];
                    bool clip = false;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint8_t *row = kb + (tok + 8 * k) * RB + run * 4 * NG, *par = kb + kBlock * RB + (tok + 8 * k) * PB;
#pragma unroll
                        for (int e = 0; e < NG; ++e) w[k][e] = reinterpret_cast<const uint32_t*>(row)[e];
#pragma unroll
                        for (int e = 0; e < NP; ++e) {
                            sc[k][e] = reinterpret_cast<const uint32_t*>(par)[e];
                            zo[k][e] = reinterpret_cast<const uint32_t*>(par)[NP + e];
                            if (!there) sc[k][e] = zo[k][e] = 0u;
                            mid[k][e] = middle_of(sc[k][e]);
                            clip |= passes_largest(sc[k][e], mid[k][e]);
                        }
                    }
                    auto store = [&](auto clip_c) {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int e = 0; e < NG; ++e) {
                                const uint32_t pick = e & 1 ? 0x3232u : 0x1010u;
                                uint32_t y[4];
                                values_of<decltype(clip_c)::value>(w[k][e], __byte_perm(sc[k][e >> 1], 0u, pick), __byte_perm(mid[k][e >> 1], 0u, pick), y);
                                *reinterpret_cast<uint4*>(sm.k[st] + to_k[e] + 8 * k * 128) = make_uint4(y[0], y[1], y[2], y[3]);
                            }
                    };
                    if (__any_sync(~0u, clip)) store(std::true_type{}); else store(std::false_type{});
                    if (run < 2)                      // the columns z, z and c, c (64: all in the first 16 bytes)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint4 y;
                            if constexpr (NG == 4) y = run ? make_uint4(mid[k][0], mid[k][1], mid[k][0], mid[k][1])
                                                           : make_uint4(zo[k][0], zo[k][1], zo[k][0], zo[k][1]);
                            else y = run ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(zo[k][0], zo[k][0], mid[k][0], mid[k][0]);
                            *reinterpret_cast<uint4*>(sm.kz[st] + run * (kEdge / 2) + (16 * dq + tok + 8 * k) * 16) = y;
                        }
                }
                fence_async_smem();
                arrive(sm.b.k_ready[st]);
                wait(sm.b.v_free[st], (j >> 1) ^ 1u);
                // values: a lane four channels of every group, of two tokens and two runs
                const bool whole = info.present == 0xff && info.base + kTokens - 1 <= v.pos_lo;
                {
                    uint32_t w[2][2][NP], sc[2][NP], zo[2][NP];
                    bool clip = false;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint8_t *row = vb + (tok + 8 * k) * RB, *par = vb + kBlock * RB + (tok + 8 * k) * PB;
#pragma unroll
                        for (int e = 0; e < NP; ++e) {
                            w[k][0][e] = reinterpret_cast<const uint32_t*>(row + run * 2 * NG)[e];
                            w[k][1][e] = reinterpret_cast<const uint32_t*>(row + (run + 4) * 2 * NG)[e];
                            sc[k][e] = reinterpret_cast<const uint32_t*>(par)[e];
                            zo[k][e] = reinterpret_cast<const uint32_t*>(par)[NP + e];
                        }
                    }
                    if (!whole) {
                        // what no row sees may be anything, and becomes zero; so does a NaN that some
                        // rows see, and they are told
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const bool seen = there && info.base + 16 * dq + tok + 8 * k <= v.pos_hi;
#pragma unroll
                            for (int e = 0; e < NG; ++e) {
                                const uint32_t half = 0xffffu << (16 * (e & 1)), inf = 0x7c00u << (16 * (e & 1));
                                const bool bad = (sc[k][e >> 1] & inf) == inf || (zo[k][e >> 1] & inf) == inf;
                                const uint32_t votes = __ballot_sync(~0u, seen && bad) & 255u;
                                if (lane == 0) reinterpret_cast<uint8_t*>(&sm.nan[st][e][dq])[k] = (uint8_t)votes;
                                if (!seen || bad) sc[k][e >> 1] &= ~half, zo[k][e >> 1] &= ~half;
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < NP; ++e) clip |= passes_largest(sc[k][e], zo[k][e]);
                    auto store = [&](auto clip_c) {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int q = 0; q < 2; ++q)
#pragma unroll
                                for (int e = 0; e < NP; ++e) {
                                    uint32_t y[4];
                                    values_of<decltype(clip_c)::value>(w[k][q][e], sc[k][e], zo[k][e], y);
                                    *reinterpret_cast<uint4*>(sm.v[st] + to_v[q][e] + 8 * k * 128) = make_uint4(y[0], y[1], y[2], y[3]);
                                }
                    };
                    if (__any_sync(~0u, clip)) store(std::true_type{}); else store(std::false_type{});
                }
                fence_async_smem();
                arrive(sm.b.v_ready[st]);
                if (lane == 0) mbar_arrive(&sm.b.staged_free[st]);
            }
        }
    }
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

Plan chunk_plan(const Shape& s) {
    Plan p{};
    p.U = s.B;
    p.R = s.T * s.G;
    p.tiles = (p.R + kRows - 1) / kRows;
    p.cap = (int)(((int64_t)s.width * s.P + kTokens - 1) / kTokens);
    p.tile = kTokens;
    p.item_cost = kChunkCost;
    const int64_t items = (int64_t)p.U * p.tiles * s.H;
    // Items are left whole, or cut into equal runs, whose parts' way through memory
    // costs as much as about nine tiles and one to each twenty items.  Head size 128, 8 key
    // heads of 4 query heads, us whole and cut: 128 tokens behind 384 18.4, 24.6, behind
    // 3968 65.8, 35.8; 512 tokens behind 3584 67.6, 91.3, behind 32256 454, 428; 640
    // tokens (160 items to 148 SMs) behind 7552 236.8, 168.4.
    const int64_t whole = (items + kSms - 1) / kSms * p.cap, runs = items * p.cap / kSms + 9 + items / 20;
    p.split = items < 8 * kSms && whole > runs;
    p.least = kChunkCost + 2;
    p.cluster = 1;
    while (kBlock << p.page_shift < s.P) ++p.page_shift;
    return p;
}

size_t chunk_lay_out(const Shape& s, const Plan& p, void* base, Space* w) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* q = (char*)base + at;
        at += (bytes + 255) & ~size_t(255);
        return q;
    };
    Space x{};
    if (p.split) {
        x.run = (int64_t*)take(((size_t)p.U + 1) * 8);
        x.part = (float*)take((size_t)2 * kSms * kRows * s.d * 4);
        x.part_ml = (float*)take((size_t)2 * kSms * 2 * kRows * 4);
    }
    if (w) *w = x;
    return at;
}

template <int D>
cudaError_t chunk_as(const Args& a, cudaStream_t st) {
    constexpr int smem = (int)sizeof(ChunkSmem<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory");
    const int64_t items = (int64_t)a.p.U * a.p.tiles * a.s.H;
    if (items * kRows > 0x7fffffff) return cudaErrorInvalidConfiguration;
    static Allowed allowed;
    cudaError_t e = allow_shared(chunk_kernel<D>, smem, allowed);
    if (e == cudaSuccess) e = launch(chunk_kernel<D>, a.p.split ? kSms : (unsigned)items, kThreads, smem, st, a);
    if (e != cudaSuccess || !a.p.split) return e;
    return launch(combine_kernel<D, kRows, 8, 4>, (unsigned)(items * (kRows / 8)), 128, 0, st, a);
}

}  // namespace

// Rows enough for a 128-row tile a key head to pay.  Us here and on mma.sync (asa_cache_attend.cu),
// 8 key heads: 8 sequences of 4096 tokens, d 128, 16 rows 48.9, 30.6, 32 rows 50.2, 54.2, 64 rows
// 52.3, 91.4, 128 rows 59.1, 160.5; d 64, 32 rows 37.2, 30.3, 64 rows 37.6, 49.6; one
// sequence of 4096, whose few items clusters share, 64 rows 28.2, 19.6, 128 rows 30.4, 29.3.
bool chunk_takes(const Shape& s, int keep) {
    return keep == 0 && s.alpha == 1.0f && (s.d == 64 || s.d == 128) && (int64_t)s.T * s.G >= 64;
}

size_t chunk_workspace(const Shape& s) { return chunk_lay_out(s, chunk_plan(s), nullptr, nullptr); }

cudaError_t chunk_attend(const Shape& s, const void* Q, Strides qs, const uint8_t* pool, const int32_t* table,
                         const int32_t* lengths, void* O, void* ws, int* err, cudaStream_t st) {
    Args a{};
    a.s = s;
    a.p = chunk_plan(s);
    chunk_lay_out(s, a.p, ws, &a.w);
    a.p.vec = (reinterpret_cast<uintptr_t>(Q) & 15) == 0 && qs.b % 8 == 0 && qs.t % 8 == 0 && qs.h % 8 == 0;
    a.qs = qs;
    a.Q = (const __nv_bfloat16*)Q;
    a.pool = pool;
    a.table = table;
    a.lengths = lengths;
    a.O = (__nv_bfloat16*)O;
    a.err = err;
    return s.d == 64 ? chunk_as<64>(a, st) : chunk_as<128>(a, st);
}

}  // namespace cache
}  // namespace asa
