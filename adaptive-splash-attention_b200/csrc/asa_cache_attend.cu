// asa_cache_attend.cu -- attention over the 4-bit paged cache.
//
// For each query row: softmax weights in one pass over keys and values, or the
// exact alpha-entmax in three (scores; the threshold of each row; the weighted
// values of the blocks that the threshold leaves weight in).
//
// Work.  An item is a tile of 8 or 16 query rows of one key head (rows of one
// sequence, or of one query token where each has its own pages); its keys are
// walked in tiles of 32 tokens.  Short items are taken whole, by a CTA or a cluster
// that joins its sums over shared memory.  Else the items' tiles, laid end to end with
// a few tiles' worth of time between items for what starting one costs, are cut into
// equal runs, one a CTA, so that a batch of very unequal sequences keeps every SM
// busy; an item that a cut divides is joined by combine_kernel from its runs'
// partial sums (largest score, sum of weights, weighted values), in a fixed order.
// A CTA's warps take an item's tiles in turn, each with its own ring of bulk
// copies that runs ahead into the CTA's next item.
//
// What it reads bounds it: 1.25 d bytes a token and key head, against 4 d operations
// a query head.  Two sequences of 131072 tokens, 4 key heads of 8 query heads, d 128
// (168 MB) take 53 us with the join, 3.2 TB/s: 36 us of that go by the tokens (65536 more
// of each 18.0), 4.7 TB/s or 0.72 of a copy's rate, the rest is starting, the warps' and the runs' joins.  A tile
// is some 1.6 us of a warp, most of it waiting on its own chain (codes, products,
// maxima, weights, products); 16 warps an SM at 128 registers each cover that, and
// keeping the next tile's products in registers as well was slower (it spilled).
// Below a few thousand tokens the chain itself is what is left: 8 us for 100 tokens.
// Entmax, 8 sequences of 32768, 8 key heads: scores 44 us (168 MB of keys in, 34 MB of
// scores out), thresholds 14, values 19 of which most is finding the few tiles
// that have weight: 76 in all; at alpha 2 82, 3 86, 1.25 (much support) 239.
//
// Arithmetic.  A code 0..15 in an fp16 half is the subnormal n * 2^-24, and in
// the next nibble n * 2^-20: masking a word gives tensor-core operands without
// converting anything.  Scores are S^T = K Q^T on mma.m16n8k16 (tokens x rows):
// per group of 32 channels the product of codes and q (q scaled by a power of two
// a row, so that fp16 holds bf16 exactly), times the token's fp32 scale; offsets
// enter as one more product, with the group sums of q in two fp16 halves.
// Weights stay in registers: a movmatrix turns P^T into the operand of
// O^T = V^T P^T.  P is rounded to fp16 once (11 bits; the plain rounding of an
// output to bf16 has 8); its products with the values' scales are taken as the
// rounded product and the rest, two products of the codes, so that codes and
// offsets are weighted by the same P and a value near zero, a difference of the
// two, is not disturbed by more than its own size.  There the codes are brought to
// n * 2^-9 first: the tensor cores align a product of a subnormal by the least normal
// exponent, and cut what lies ten bits further up than need be (a value near zero
// under a weight near one was off by 2^-16 of its offset).  Scores have room for that.  A
// running exponent e of the largest scale fits P to the scales, so that small ones stay
// clear of fp16's subnormals and large ones do not overflow: a row's largest P starts at
// 2^4 (2^(4 - e) for e below 0, and less from e = 8 on) and may grow until P times the scales
// reach 2^15.5 before its reference is moved.  So P keeps its 11 bits down to 2^-18 of the
// largest weight, and 2^-12 at the largest scales.  Sums, maxima and accumulators are fp32.
#include "asa_cache_attend.cuh"

namespace asa {
namespace cache {
namespace {

constexpr int kTile = 2;              // blocks of a tile
constexpr int kStages = 2;            // tiles a warp has in flight
constexpr uint32_t kUp15 = 0x78007800u, kUp11 = 0x68006800u;   // fp16 pairs: 2^15, 2^11
constexpr int kLeast = -8;            // weights are raised for small scales by 2^8 at most
constexpr float kRoom = 3.0f;         // log2 of what a row's largest weight may grow by, at least, before its reference moves
// Plan::item_cost.  Measured: 48 ragged sequences of up to 8192 tokens 58.5 us with 8, 51.3 with
// 12, 49.3 with 16, 49.8 with 20, 52.5 with 28; 12 of up to 16384 43.6, 37.1, 35.8, 35.9, 36.6;
// listed pages (items of one size) 41.8 with 8, 44.8 with 12, 46.2 with 4 where they are cut.
constexpr int kItemCost = 16, kListedCost = 8;
constexpr int kSegments = 32;         // segments a CTA lines up at a time

enum Mode { kSoftmax = 0, kScores = 1, kValues = 2 };

// ---- small pieces --------------------------------------------------------------
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zero.
__device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                     uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Larger and smaller that keep a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float c;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
}
// a * b - c: with c the rounded a * b, what the rounding cut off.
__device__ __forceinline__ uint32_t hrest2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              __hneg2(*reinterpret_cast<const __half2*>(&c)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b) {
    const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// What lies at a place of this CTA's shared memory, in the cluster's CTA `rank`.
template <typename V>
__device__ __forceinline__ V remote(const V* p, int rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_u32(p)), "r"(rank));
    V v;
    if constexpr (sizeof(V) == 16)
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    else
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

// The token (0..7) that stands at index m of an 8-token half block in the
// fragments: neighbours 2, 3 and 6, 7 trade places, which spreads the values' rows
// over the shared-memory banks.
__device__ __forceinline__ int token_of(int m) { return m ^ ((m >> 1) & 1); }

// NW words from shared memory, as wide as their number allows.
template <int NW>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&w)[NW]) {
    if constexpr (NW == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (NW == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}
// NH halves (2 NH bytes) as ceil(NH / 2) words.
template <int NH>
__device__ __forceinline__ void lds_halves(const uint8_t* p, uint32_t (&w)[(NH + 1) / 2]) {
    if constexpr (NH == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else if constexpr (NH == 3) {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
        w[0] = q[0] | (uint32_t)q[1] << 16;
        w[1] = q[2];
    } else if constexpr (NH == 2) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
}

// ---- the walk over keys and values ----------------------------------------------
struct Segment { int u, item, from, n, of; };         // tiles from .. from + n - 1 of an item's `of`
struct Info { int pos0, pos1, tile, seg; };           // a ring stage: its blocks' first positions, where it belongs

// A segment's query rows, made ready by one warp for all.
template <int NG, int NT>
struct Rows {
    uint32_t q[NT][4 * NG + 1][32];                   // B fragments, and the group sums' halves
    float factor[8 * NT];                             // a score's, from the product's unit
    int pos[8 * NT];                                  // the rows' positions, -1 before the first key and past the last row
    int out[8 * NT];                                  // their rows of O
};

template <int D, int NT, int W>
struct Smem {
    static constexpr int kStride = D + 4;             // a float4 of each of 8 rows of lanes: no bank twice
    alignas(128) uint8_t ring[W][kStages][2 * kTile * block_bytes(D)];
    float4 o[W / 2][8 * NT][kStride / 4];
    float m[W][8 * NT], l[W][8 * NT];
    float2 ml[8 * NT];                                // this CTA's references and sums, for its cluster
    Rows<D / 32, NT> rows[2];
    Info info[W][kStages];
    uint64_t full[W][kStages];
    Segment seg[kSegments];
    int segs;
    int64_t next;
    int64_t pref[W * 32 + 1];
    int64_t scan[W];
};

template <int D, int NT, int W, int MODE>
__global__ void __launch_bounds__(W * 32, NT == 1 ? 2 : 3) walk_kernel(const __grid_constant__ Args a) {
    constexpr int NG = D / 32, ROWS = 8 * NT, NTHR = W * 32, BB = block_bytes(D), NS = (NG + 1) / 2;
    constexpr int RB = row_bytes(D), PB = par_bytes(D);
    constexpr int kNone = 0x3fffffff;                 // the first position of a block that is not there
    extern __shared__ __align__(128) uint8_t smem_raw[];
    auto& sm = *reinterpret_cast<Smem<D, NT, W>*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
    const Shape& s = a.s;
    const int per = a.p.tiles * s.H;                  // items of a unit

    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) sm100::mbar_init(&sm.full[warp][i], 1);
        sm100::fence_barrier_init();
    }
    follow();
    __syncthreads();

    // this CTA's run [x, x1) of all the items' tiles
    int64_t x = 0, x1 = 1;
    int chunk = 0;                                    // the units whose prefix sums are in sm.pref
    auto load_chunk = [&](int base, int64_t before) -> int64_t {
        __syncthreads();
        int64_t sum, v = 0;
        if (base + tid < a.p.U) {
            const int n = unit_tiles(a, base + tid);
            if (n) v = (int64_t)(n + a.p.item_cost) * per;
        }
        const int64_t e = block_scan<NTHR>(v, sm.scan, &sum);
        sm.pref[tid] = before + e;
        if (tid == 0) sm.pref[NTHR] = before + sum;
        __syncthreads();
        chunk = base;
        return before + sum;
    };
    if (a.p.split) {
        int64_t total = 0;
        for (int base = 0; base < a.p.U; base += NTHR) {
            total = load_chunk(base, total);
            if (blockIdx.x == 0 && base + tid < a.p.U) a.w.run[1 + base + tid] = sm.pref[tid];
        }
        const int64_t run = max((int64_t)a.p.least, (total + gridDim.x - 1) / gridDim.x);
        if (blockIdx.x == 0 && tid == 0) a.w.run[0] = run;
        x = run * blockIdx.x;
        x1 = min(x + run, total);
        if (x >= x1) return;
        if (a.p.U > NTHR) {                           // back to the chunk that the run starts in
            int64_t before = load_chunk(0, 0);
            while (x >= before) before = load_chunk(chunk + NTHR, before);
        }
    }
    // where this lane's operands lie in a stage: tokens t0, t0 + 8 of a block of keys, ta, tb
    // and those 8 on of a block of values
    const int t0 = token_of(r), ta = token_of(2 * t), tb = ta ^ 1;
    const uint8_t* const ring = sm.ring[warp][0];
    constexpr int kStage = 2 * kTile * BB;
    const int at_kc = t0 * RB + t * 4 * NG, at_kp = kBlock * RB + t0 * PB;
    // (lanes past the last group read a scale; their part of q's sums is zero)
    const int at_kz = at_kp + (NG == 4 || t < NG ? 2 * (NG + t) : 0);
    const int at_vc = kTile * BB + r * 2 * NG, at_vp = kTile * BB + kBlock * RB;
    const int at_vz = at_vp + 2 * NG + 2 * (NG == 4 ? r & 3 : r < NG ? r : 0);
    // the product with the offsets has a group a row, and a row of ones that sums the weights
    const uint32_t z_and = r < NG ? ~0u : 0u, z_or = r == NG ? 0x3c003c00u : 0u;

    int stage_in = 0, stage_out = 0;                  // the ring's next stage to fill and to read
    uint32_t parity = 0;                              // of the stage to read
    bool lost = false;

    while (x < x1) {
        // ---- the next segments of the run -----------------------------------------
        __syncthreads();                              // every warp is done with the last ones
        if (a.p.split) {
            while (x >= sm.pref[NTHR]) load_chunk(chunk + NTHR, sm.pref[NTHR]);
            if (tid == 0) {
                int lo = 0, hi = NTHR, k = 0;         // the last unit that starts at or before x
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (sm.pref[mid] <= x) lo = mid; else hi = mid;
                }
                int64_t y = x;
                const int64_t stop = min(x1, sm.pref[NTHR]);
                while (y < stop && k < kSegments) {
                    while (sm.pref[lo + 1] <= y) ++lo;
                    const int of = (int)((sm.pref[lo + 1] - sm.pref[lo]) / per) - a.p.item_cost;
                    const int64_t off = y - sm.pref[lo];
                    const int item = (int)(off / (of + a.p.item_cost));
                    const int64_t begin = sm.pref[lo] + (int64_t)item * (of + a.p.item_cost) + a.p.item_cost;
                    const int from = (int)max((int64_t)0, y - begin), to = (int)min((int64_t)of, stop - begin);
                    if (to > from) sm.seg[k++] = Segment{chunk + lo, item, from, to - from, of};
                    y = min(stop, begin + of);
                }
                sm.segs = k;
                sm.next = y;
            }
        } else if (tid == 0) {
            const unsigned no = blockIdx.x / (unsigned)a.p.cluster, rank = blockIdx.x % (unsigned)a.p.cluster;
            const int u = no / (unsigned)per, of = unit_tiles(a, u);
            const int from = (int)((int64_t)of * rank / a.p.cluster), to = (int)((int64_t)of * (rank + 1) / a.p.cluster);
            sm.seg[0] = Segment{u, (int)(no % (unsigned)per), from, to - from, of};
            sm.segs = 1;
            sm.next = 1;
        }
        __syncthreads();
        const int segs = sm.segs;
        x = sm.next;

        // ---- the tiles that this warp reads, fetched ahead across segments -----------
        auto token_of_row = [&](int u, int row) { return a.list ? u % s.T : row / s.G; };
        auto position = [&](int u, int row) -> int {  // of an item's row (its tile's first row added)
            const long long len = __ldg(a.lengths + (a.list ? u / s.T : u));
            return (int)max(-1ll, min(len - s.T + token_of_row(u, row), (long long)s.width * s.P - 1));
        };
        int ahead = -1, mine = 0, c = 0;              // the segment being fetched, the warp's tiles of it, 32 c of them passed
        uint32_t there = 0;                           // of the 32 that the lanes have looked up
        const uint8_t *at0 = nullptr, *at1 = nullptr; // this lane's: its blocks' records and first positions
        int pos0 = 0, pos1 = 0;
        auto locate = [&](const Segment& g, int k) -> bool {
            at0 = at1 = nullptr;
            pos0 = pos1 = kNone;
            if (k >= mine) return false;
            const int j = g.from + warp + k * W, h = g.item / a.p.tiles, tile = g.item % a.p.tiles;
            const int64_t item_no = (int64_t)g.u * per + g.item;
            const int pos_hi = position(g.u, min(tile * ROWS + ROWS, a.p.R) - 1);
            bool wanted = true;
            if constexpr (MODE == kValues) {          // only tiles that a threshold leaves weight in
                const float* top = a.w.top + (item_no * a.p.cap + j) * ROWS;
                wanted = false;
#pragma unroll
                for (int i = 0; i < ROWS; i += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(top + i);
                    const float4 z = *reinterpret_cast<const float4*>(a.w.tau + item_no * ROWS + i);
                    wanted |= !(y.x <= z.x) | !(y.y <= z.y) | !(y.z <= z.z) | !(y.w <= z.w);
                }
            }
            if (wanted) {
                const int32_t* table_b = a.table + (int64_t)(a.list ? g.u / s.T : g.u) * s.width;
                const int32_t* list = a.list ? a.list + ((int64_t)g.u * s.H + h) * a.p.keep : nullptr;
                auto block = [&](int blk, const uint8_t*& at, int& pos) {
                    int page = blk >> a.p.page_shift;
                    const int in_page = blk & ((1 << a.p.page_shift) - 1);
                    if (list) page = page < a.p.keep ? __ldg(list + page) : -1;
                    if (page < 0 || page >= s.width) return;
                    const int first = page * s.P + in_page * kBlock;
                    if (first > pos_hi) return;
                    const int id = __ldg(table_b + page);
                    if (id >= 0 && id < s.pages) {
                        at = a.pool + ((int64_t)id * s.H + h) * s.rec + in_page * BB;
                        pos = first;
                    } else if (a.err) {
                        atomicCAS(a.err, 0, ASA_ERR_INVALID);
                    }
                };
                block(kTile * j, at0, pos0);
                if (a.p.page_shift == 0) block(kTile * j + 1, at1, pos1);
                else if (at0 && pos0 + kBlock <= pos_hi) pos1 = pos0 + kBlock;   // the tile lies in one page
            }
            const bool found = at0 || at1;
            if constexpr (MODE == kScores)
                if (!found)
                    for (int i = 0; i < ROWS; ++i) a.w.top[(item_no * a.p.cap + j) * ROWS + i] = -INFINITY;
            return found;
        };
        int in_flight = 0;
        auto fetch = [&]() {                          // the next tile that is there, into the ring
            while (!there) {
                if (32 * c >= mine) {
                    if (ahead + 1 >= segs) return;
                    ++ahead;
                    c = 0;
                    mine = sm.seg[ahead].n > warp ? (sm.seg[ahead].n - warp + W - 1) / W : 0;
                    continue;
                }
                there = __ballot_sync(~0u, locate(sm.seg[ahead], 32 * c + lane));
                ++c;
            }
            const int k = __ffs(there) - 1;
            there &= there - 1;
            if (lane == k)                            // the lane that looked it up issues its copies
                sm.info[warp][stage_in] = Info{pos0, pos1, sm.seg[ahead].from + warp + (32 * (c - 1) + k) * W, ahead};
            // (a lane none of whose waits gave up has seen all that the stage held before; another must not
            // arm it again, since its last copy may still be awaited)
            if (lane == k && !lost) {
                uint8_t* dst = sm.ring[warp][stage_in];
                uint64_t* bar = &sm.full[warp][stage_in];
                constexpr int kParts = MODE == kSoftmax ? 2 : 1;
                if (a.p.page_shift) {                 // two blocks on end
                    sm100::mbar_expect_tx(bar, kParts * kTile * BB);
                    if (MODE != kValues) bulk_load(dst, at0, kTile * BB, bar);
                    if (MODE != kScores) bulk_load(dst + kTile * BB, at0 + s.rec / 2, kTile * BB, bar);
                } else {
                    sm100::mbar_expect_tx(bar, kParts * BB * ((at0 ? 1 : 0) + (at1 ? 1 : 0)));
#pragma unroll
                    for (int i = 0; i < kTile; ++i) {
                        const uint8_t* src = i ? at1 : at0;
                        if (!src) continue;
                        if (MODE != kValues) bulk_load(dst + i * BB, src, BB, bar);
                        if (MODE != kScores) bulk_load(dst + (kTile + i) * BB, src + s.rec / 2, BB, bar);
                    }
                }
            }
            __syncwarp();
            stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
            ++in_flight;
        };
        for (int i = 0; i < kStages; ++i) fetch();

        // ---- queries as B fragments, a power of two a row: n-tile nt of segment sg --------
        auto make_rows = [&](int sg, int nt) {
            const Segment g = sm.seg[sg];
            auto& out = sm.rows[sg & 1];
            const int h = g.item / a.p.tiles, row = g.item % a.p.tiles * ROWS + 8 * nt + r;
            const int b = a.list ? g.u / s.T : g.u;
            const bool real = row < a.p.R;
            const int tq = token_of_row(g.u, row), hq = h * s.G + (a.list ? row : row % s.G);
            if (t == 0) {
                out.pos[8 * nt + r] = real ? position(g.u, row) : -1;
                out.out[8 * nt + r] = (b * s.T + tq) * s.HQ + hq;
            }
            if constexpr (MODE != kValues) {
                float q[NG][8], big = 0.0f;
                const __nv_bfloat16* src = a.Q + b * a.qs.b + tq * a.qs.t + hq * a.qs.h + 8 * t;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    uint32_t w[4] = {0u, 0u, 0u, 0u};
                    if (real && a.p.vec) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + 32 * i));
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    } else if (real) {
                        const uint16_t* e = reinterpret_cast<const uint16_t*>(src + 32 * i);
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = __ldg(e + 2 * k) | (uint32_t)__ldg(e + 2 * k + 1) << 16;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        q[i][2 * k] = __uint_as_float(w[k] << 16);
                        q[i][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                        big = fmaxf(big, fmaxf(fabsf(q[i][2 * k]), fabsf(q[i][2 * k + 1])));
                    }
                }
                float sum = 0.0f;                     // a NaN or an infinity makes the sum of 0 * q NaN
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum = fmaf(q[i][k], 0.0f, sum);
                big = fmaxf(big, __shfl_xor_sync(~0u, big, 1));
                big = fmaxf(big, __shfl_xor_sync(~0u, big, 2));
                const bool bad = (__ballot_sync(~0u, sum != sum) >> (lane & 28)) & 15u;
                // big * 2^up lies in [2^13, 2^14), but for what is below 2^-113
                const int up = big == 0.0f || bad ? 0 : 13 - max((int)(__float_as_uint(big) >> 23) - 127, -113);
                const float f = bad ? NAN : pow2i(up), f16 = bad ? NAN : pow2i(up - 4);
                float own = 0.0f;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    // channels 8t .. 8t + 7 of the group, in the order that masking a word of codes gives
                    out.q[nt][4 * i][lane] = pack(q[i][0] * f, q[i][4] * f);
                    out.q[nt][4 * i + 1][lane] = pack(q[i][1] * f16, q[i][5] * f16);
                    out.q[nt][4 * i + 2][lane] = pack(q[i][2] * f, q[i][6] * f);
                    out.q[nt][4 * i + 3][lane] = pack(q[i][3] * f16, q[i][7] * f16);
                    float v = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) v += q[i][k] * f16;
                    v += __shfl_xor_sync(~0u, v, 1);
                    v += __shfl_xor_sync(~0u, v, 2);
                    own = t == i ? v : own;
                }
                const float hi = __half2float(__float2half_rn(own));
                out.q[nt][4 * NG][lane] = pack(hi, own - hi);
                if (t == 0) out.factor[8 * nt + r] = factor_of(s.scale * (MODE == kSoftmax ? kLog2e : s.alpha - 1.0f), 24 - up, kMostFactor);
            }
        };
        if (warp < NT && segs) make_rows(0, warp);
        __syncthreads();

        for (int sg = 0; sg < segs; ++sg) {
            const Segment g = sm.seg[sg];
            const int tile = g.item % a.p.tiles;
            const int64_t item_no = (int64_t)g.u * per + g.item;
            const int rows = min(ROWS, a.p.R - tile * ROWS);
            const auto& mine_rows = sm.rows[sg & 1];
            const int pos_hi = mine_rows.pos[rows - 1], pos_lo = mine_rows.pos[0];   // rows stand in order
            uint32_t qf[NT][NG][4], qz[NT];
            float rf[NT][2];                          // the factor of rows 2t, 2t + 1's scores
            float m[NT][2], room[NT][2];              // references, and how far above them a score may lie (-inf: unset)
            float oz[NT][4], o[NT][2 * NG][4];        // oz: by group the offsets' sums, and the weights'
            // log2 by which weights are lowered for large scales (raised for small ones), and the
            // fp16 scale 2^(lift + 1) that this allows
            int lift = MODE == kSoftmax ? kLeast : 0;
            uint32_t s_most = (uint32_t)(lift + 16) << 10;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (MODE != kValues) {
#pragma unroll
                    for (int i = 0; i < 4 * NG; ++i) qf[nt][i / 4][i % 4] = mine_rows.q[nt][i][lane];
                    qz[nt] = mine_rows.q[nt][4 * NG][lane];
                }
                if constexpr (MODE != kValues) {
                    const float2 f2 = *reinterpret_cast<const float2*>(&mine_rows.factor[8 * nt + 2 * t]);
                    rf[nt][0] = f2.x, rf[nt][1] = f2.y;
                }
                m[nt][0] = m[nt][1] = MODE == kSoftmax ? 0.0f : -14.0f;   // (entmax weights are at most 1)
                room[nt][0] = room[nt][1] = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) oz[nt][e] = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
            }

            // ---- the segment's tiles ---------------------------------------------------
            while (in_flight) {
                const Info info = sm.info[warp][stage_out];
                if (info.seg != sg) break;
                if (!wait_full(&sm.full[warp][stage_out], parity, s.naps, a.err)) lost = true;
                __syncwarp();
                const uint8_t* const st = ring + stage_out * kStage;
                // every row sees all of both blocks
                const bool whole = max(info.pos0, info.pos1) + kBlock - 1 <= pos_lo;
                float v[kTile][NT][4];
                auto each = [&](auto fn) {            // of the scores: (block, n-tile, element, its token)
#pragma unroll
                    for (int i = 0; i < kTile; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) fn(i, nt, e);
                };
                auto mask = [&]() {                   // scores of keys that a row does not see
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int2 pos = *reinterpret_cast<const int2*>(&mine_rows.pos[8 * nt + 2 * t]);
#pragma unroll
                        for (int i = 0; i < kTile; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if ((i ? info.pos1 : info.pos0) + t0 + (e < 2 ? 0 : 8) > (e & 1 ? pos.y : pos.x))
                                    v[i][nt][e] = -INFINITY;
                    }
                };

                if constexpr (MODE != kValues) {
                    // scores of tokens t0, t0 + 8 and rows 2t, 2t + 1, group by group
#pragma unroll
                    for (int i = 0; i < kTile; ++i) {
                        uint32_t w0[NG], w1[NG], p0[NS], p1[NS];
                        lds<NG>(st + at_kc + i * BB, w0);
                        lds<NG>(st + at_kc + i * BB + 8 * RB, w1);
                        lds_halves<NG>(st + at_kp + i * BB, p0);
                        lds_halves<NG>(st + at_kp + i * BB + 8 * PB, p1);
                        uint32_t z0 = *reinterpret_cast<const uint16_t*>(st + at_kz + i * BB);
                        uint32_t z1 = *reinterpret_cast<const uint16_t*>(st + at_kz + i * BB + 8 * PB);
                        z0 = __byte_perm(z0, z0, 0x1010);
                        z1 = __byte_perm(z1, z1, 0x1010);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float cz[4];
                            mma0(cz, z0, z1, 0u, 0u, qz[nt], 0u);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[i][nt][e] = cz[e] * 9.5367431640625e-7f;   // 2^-20: codes and halves count 2^-24, 2^-4
                        }
#pragma unroll
                        for (int k = 0; k < NG; ++k) {
                            const uint32_t x0 = w0[k], y0 = w1[k], x8 = x0 >> 8, y8 = y0 >> 8;
                            const float2 s0 = unpack(p0[k >> 1]), s1 = unpack(p1[k >> 1]);
                            const float f0 = k & 1 ? s0.y : s0.x, f1 = k & 1 ? s1.y : s1.x;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float acc[4];
                                mma0(acc, x0 & 0x000f000fu, y0 & 0x000f000fu, x0 & 0x00f000f0u, y0 & 0x00f000f0u,
                                     qf[nt][k][0], qf[nt][k][1]);
                                mma(acc, x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u,
                                    qf[nt][k][2], qf[nt][k][3]);
                                v[i][nt][0] = fmaf(acc[0], f0, v[i][nt][0]);
                                v[i][nt][1] = fmaf(acc[1], f0, v[i][nt][1]);
                                v[i][nt][2] = fmaf(acc[2], f1, v[i][nt][2]);
                                v[i][nt][3] = fmaf(acc[3], f1, v[i][nt][3]);
                            }
                        }
                    }
                }
                if constexpr (MODE == kScores) {
                    const float most = 10.0f * (s.alpha - 1.0f);   // x = (alpha - 1) score, clamped as in training
                    const int64_t place = item_no * a.p.cap + info.tile;
                    each([&](int i, int nt, int e) {
                        v[i][nt][e] = min_nan(max_nan(v[i][nt][e] * rf[nt][e & 1], -most), most);
                    });
                    if (!whole) mask();
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float top[2] = {-INFINITY, -INFINITY};     // a NaN score: its row is NaN
#pragma unroll
                        for (int i = 0; i < kTile; ++i) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) top[e & 1] = max_nan(top[e & 1], v[i][nt][e]);
                            if (8 * nt + 2 * t < rows)
                                a.w.score[((place * kTile + i) * NT + nt) * 32 + 8 * t + r] =
                                    make_float4(v[i][nt][0], v[i][nt][1], v[i][nt][2], v[i][nt][3]);
                        }
#pragma unroll
                        for (int k = 4; k < 32; k <<= 1) {
                            top[0] = max_nan(top[0], __shfl_xor_sync(~0u, top[0], k));
                            top[1] = max_nan(top[1], __shfl_xor_sync(~0u, top[1], k));
                        }
                        // rows past the last take no part
                        if (8 * nt + 2 * t >= rows) top[0] = -INFINITY;
                        if (8 * nt + 2 * t + 1 >= rows) top[1] = -INFINITY;
                        if (r == 0) *reinterpret_cast<float2*>(a.w.top + place * ROWS + 8 * nt + 2 * t) = make_float2(top[0], top[1]);
                    }
                } else {
                    // v: a score less its row's reference (softmax), or less its threshold
                    if constexpr (MODE == kValues) {
                        const int64_t place = item_no * a.p.cap + info.tile;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            // rows 2t, 2t + 1: the largest x, and the threshold relative to it
                            const float4 edge = __ldg(reinterpret_cast<const float4*>(a.w.edge + item_no * ROWS + 8 * nt + 2 * t));
#pragma unroll
                            for (int i = 0; i < kTile; ++i) {
                                float4 y = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                                if (8 * nt + 2 * t < rows) y = a.w.score[((place * kTile + i) * NT + nt) * 32 + 8 * t + r];
                                // (close to the largest the first difference is exact, and so keeps what
                                // the threshold's distance from it, 1e-9 and less among many ties, is made of)
                                v[i][nt][0] = (y.x - edge.x) - edge.y, v[i][nt][1] = (y.y - edge.z) - edge.w;
                                v[i][nt][2] = (y.z - edge.x) - edge.y, v[i][nt][3] = (y.w - edge.z) - edge.w;
                            }
                        }
                    } else {
                        each([&](int i, int nt, int e) { v[i][nt][e] = fmaf(v[i][nt][e], rf[nt][e & 1], -m[nt][e & 1]); });
                        if (!whole) mask();
                    }
                    // the values' scales of tokens ta, tb (k = 2t, 2t + 1) and those 8 on, as pairs a group
                    uint32_t sp[kTile][NG][2], zp[kTile][2];
#pragma unroll
                    for (int i = 0; i < kTile; ++i) {
                        uint32_t ra[NS], rb[NS], rc[NS], rd[NS];
                        const uint8_t *pa = st + at_vp + ta * PB + i * BB, *pb_ = st + at_vp + tb * PB + i * BB;
                        lds_halves<NG>(pa, ra);
                        lds_halves<NG>(pb_, rb);
                        lds_halves<NG>(pa + 8 * PB, rc);
                        lds_halves<NG>(pb_ + 8 * PB, rd);
#pragma unroll
                        for (int k = 0; k < NG; ++k) {
                            const uint32_t pick = k & 1 ? 0x7632u : 0x5410u;
                            sp[i][k][0] = __byte_perm(ra[k >> 1], rb[k >> 1], pick);
                            sp[i][k][1] = __byte_perm(rc[k >> 1], rd[k >> 1], pick);
                        }
                        const uint8_t *za = st + at_vz + ta * PB + i * BB, *zb = st + at_vz + tb * PB + i * BB;
                        zp[i][0] = __byte_perm(*reinterpret_cast<const uint16_t*>(za), *reinterpret_cast<const uint16_t*>(zb), 0x5410);
                        zp[i][1] = __byte_perm(*reinterpret_cast<const uint16_t*>(za + 8 * PB), *reinterpret_cast<const uint16_t*>(zb + 8 * PB), 0x5410);
                        zp[i][0] = (zp[i][0] & z_and) | z_or;
                        zp[i][1] = (zp[i][1] & z_and) | z_or;
                    }
                    if (!whole) {
                        // Tokens that no row sees may hold anything: their scales and
                        // offsets become zero.  So do those of tokens that only some rows
                        // see and that hold a NaN; it goes to the rows that see it by way
                        // of the offsets' sums.
#pragma unroll
                        for (int i = 0; i < kTile; ++i) {
                            const int first = i ? info.pos1 : info.pos0;
                            uint32_t bad = 0;         // of group r: the tokens with a NaN, by position
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int tok = (e ? tb : ta) + 8 * j;
                                    const uint32_t half = 0xffffu << (16 * e), inf = 0x7c00u << (16 * e);
                                    const bool seen = first + tok <= pos_hi;
                                    bool nan = (zp[i][j] & inf) == inf;
#pragma unroll
                                    for (int k = 0; k < NG; ++k) {
                                        const bool off = (sp[i][k][j] & inf) == inf;
                                        if (k == r) nan |= off;
                                        if (!seen || off) sp[i][k][j] &= ~half;
                                    }
                                    if (r < NG && (!seen || nan)) zp[i][j] &= ~half;
                                    if (r < NG && seen && nan) bad |= 1u << tok;
                                }
                            bad |= __shfl_xor_sync(~0u, bad, 1);
                            bad |= __shfl_xor_sync(~0u, bad, 2);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int see = min(max(mine_rows.pos[8 * nt + 2 * t + e] - first + 1, 0), kBlock);
                                    if (bad & ((1u << see) - 1u)) oz[nt][e] = NAN;
                                }
                        }
                    }
                    // weights below 2^(kMost - max(lift, 0)), scales below 2^(lift + 1),
                    // so that their products stay within fp16: rescale where a score or a scale
                    // has outgrown what they were fitted to
                    uint32_t sbig = hmax2(sp[0][0][0], sp[0][0][1]);
#pragma unroll
                    for (int k = 1; k < kTile * NG; ++k) sbig = hmax2(sbig, hmax2(sp[k / NG][k % NG][0], sp[k / NG][k % NG][1]));
                    sbig = max(sbig & 0x7fffu, sbig >> 16 & 0x7fffu);   // (no scale is far below zero)
                    bool grow = sbig > s_most;
                    if constexpr (MODE == kSoftmax) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                grow |= fmaxf(fmaxf(v[0][nt][e], v[0][nt][e + 2]), fmaxf(v[1][nt][e], v[1][nt][e + 2])) > room[nt][e];
                    }
                    if (__any_sync(~0u, grow)) {
                        // NaN scales aside: what they touch is NaN whatever the weights
                        const uint32_t all = __reduce_max_sync(~0u, min(sbig, 0x7bffu));
                        const int up = max(lift, (int)(all >> 10) - 15);   // 2^up <= largest scale < 2^(up + 1)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float f[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float by = (float)(up - lift);     // what the reference rises by
                                const bool none = MODE == kSoftmax && room[nt][e] == -INFINITY;   // no key of it seen yet
                                if constexpr (MODE == kSoftmax) {
                                    float top = fmaxf(fmaxf(v[0][nt][e], v[0][nt][e + 2]), fmaxf(v[1][nt][e], v[1][nt][e + 2]));
                                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
                                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
                                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
                                    // a large scale leaves less room above, not fewer bits below, down to kRoom
                                    const float to = top - (up > 0 ? fminf(kTop, kMost - kRoom - (float)up) : kTop - (float)up);
                                    if (room[nt][e] > -INFINITY) by = fmaxf(by, to);
                                    else by = top > -INFINITY ? to : 0.0f;
                                    if (room[nt][e] > -INFINITY || top > -INFINITY) room[nt][e] = kMost - (float)max(up, 0);
#pragma unroll
                                    for (int i = 0; i < kTile; ++i) v[i][nt][e] -= by, v[i][nt][e + 2] -= by;
                                }
                                // (a first reference may lie far below 0: nothing is summed yet that it could scale)
                                f[e] = none ? 1.0f : exp2_fast(-by);
                                m[nt][e] += by;
                                oz[nt][e] *= f[e];
                            }
#pragma unroll
                            for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nt][i][e] *= f[e & 1];
                        }
                        lift = up;
                        s_most = (uint32_t)(up + 16) << 10;
                    }
                    // P, and P^T as an operand
                    uint32_t pb[kTile][NT][2];
#pragma unroll
                    for (int i = 0; i < kTile; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float p[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float y = v[i][nt][e];
                                if constexpr (MODE == kSoftmax) {
                                    p[e] = exp2_fast(y);
                                } else {
                                    const float unit = exp2_fast(-m[nt][e & 1]);
                                    if (s.alpha == 1.5f) p[e] = y > 0.0f ? y * y * unit : 0.0f;
                                    else p[e] = y > 0.0f ? exp2f(log2f(y) / (s.alpha - 1.0f)) * unit : 0.0f;
                                    if (y != y) p[e] = y;
                                }
                            }
                            pb[i][nt][0] = transpose8(pack(p[0], p[1]));
                            pb[i][nt][1] = transpose8(pack(p[2], p[3]));
                            mma(oz[nt], zp[i][0], 0u, zp[i][1], 0u, pb[i][nt][0], pb[i][nt][1]);
                        }
                    // the values' codes: a half word of each token and group, four channels
#pragma unroll
                    for (int i = 0; i < kTile; ++i) {
                        uint32_t ca[NS], cb[NS], cc[NS], cd[NS];
                        const uint8_t *qa = st + at_vc + ta * RB + i * BB, *qb = st + at_vc + tb * RB + i * BB;
                        lds_halves<NG>(qa, ca);
                        lds_halves<NG>(qb, cb);
                        lds_halves<NG>(qa + 8 * RB, cc);
                        lds_halves<NG>(qb + 8 * RB, cd);
#pragma unroll
                        for (int k = 0; k < NG; ++k) {
                            const uint32_t pick = k & 1 ? 0x7632u : 0x5410u;
                            const uint32_t x0 = __byte_perm(ca[k >> 1], cb[k >> 1], pick), x8 = x0 >> 8;
                            const uint32_t y0 = __byte_perm(cc[k >> 1], cd[k >> 1], pick), y8 = y0 >> 8;
                            uint32_t c[2][4];         // the codes times 2^-9
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t x = e ? x8 : x0, y = e ? y8 : y0;
                                c[e][0] = hmul2(x & 0x000f000fu, kUp15), c[e][1] = hmul2(x & 0x00f000f0u, kUp11);
                                c[e][2] = hmul2(y & 0x000f000fu, kUp15), c[e][3] = hmul2(y & 0x00f000f0u, kUp11);
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const uint32_t b0 = hmul2(pb[i][nt][0], sp[i][k][0]), b1 = hmul2(pb[i][nt][1], sp[i][k][1]);
                                const uint32_t e0 = hrest2(pb[i][nt][0], sp[i][k][0], b0), e1 = hrest2(pb[i][nt][1], sp[i][k][1], b1);
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    mma(o[nt][2 * k + e], c[e][0], c[e][1], c[e][2], c[e][3], b0, b1);
                                    mma(o[nt][2 * k + e], c[e][0], c[e][1], c[e][2], c[e][3], e0, e1);
                                }
                            }
                        }
                    }
                }
                __syncwarp();                         // the stage has been read by all lanes
                if (++stage_out == kStages) stage_out = 0, parity ^= 1u;
                --in_flight;
                fetch();
            }
            if constexpr (MODE == kSoftmax)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (!(room[nt][e] > -INFINITY)) m[nt][e] = kLow;
            // the next segment's rows, by the warps that may be first done
            if (warp >= W - NT && sg + 1 < segs) make_rows(sg + 1, warp - (W - NT));

            // ---- the warps' sums together; the item's output, or this run's part of it ---
            if constexpr (MODE == kScores) {
                __syncthreads();
            } else {
                // a row's weight sum is in the lanes r = NG; scale the sums to one reference a row
                if (r == NG)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            sm.m[warp][8 * nt + 2 * t + e] = m[nt][e];
                            sm.l[warp][8 * nt + 2 * t + e] = oz[nt][e];
                        }
                __syncthreads();
                constexpr int H = W / 2;
#pragma unroll
                for (int half = 1; half >= 0; --half) {   // the upper warps hand theirs to the lower ones
                    if ((warp >= H) == (half == 1)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int row = 8 * nt + 2 * t + e;
                                float top = sm.m[0][row];
#pragma unroll
                                for (int w = 1; w < W; ++w) top = fmaxf(top, sm.m[w][row]);
                                const float f = exp2_fast(m[nt][e] - top), k0 = 512.0f * f;   // codes count 2^-9
#pragma unroll
                                for (int k = 0; k < NG; ++k) {
                                    const float z = __shfl_sync(~0u, oz[nt][e], 4 * k + t) * f;
                                    float4 y = make_float4(fmaf(o[nt][2 * k][e], k0, z), fmaf(o[nt][2 * k][e + 2], k0, z),
                                                           fmaf(o[nt][2 * k + 1][e], k0, z), fmaf(o[nt][2 * k + 1][e + 2], k0, z));
                                    float4* dst = &sm.o[warp % H][row][8 * k + r];
                                    if (half == 0) {
                                        const float4 u = *dst;
                                        y = make_float4(y.x + u.x, y.y + u.y, y.z + u.z, y.w + u.w);
                                    }
                                    *dst = y;
                                }
                            }
                    }
                    __syncthreads();
                }
                const bool all = g.n == g.of && a.p.cluster == 1;
                const int64_t slot = 2 * (int64_t)blockIdx.x + (g.from + g.n < g.of ? 1 : 0);
                auto put = [&](int row, int c4, float4 acc, float sum) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    __nv_bfloat162 y[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv),
                                           __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
                    *reinterpret_cast<uint2*>(a.O + (int64_t)mine_rows.out[row] * D + 4 * c4) = *reinterpret_cast<uint2*>(y);
                };
                for (int i = tid; i < rows * (D / 4); i += NTHR) {
                    const int row = i / (D / 4), c4 = i % (D / 4);
                    float top = sm.m[0][row];
#pragma unroll
                    for (int w = 1; w < W; ++w) top = fmaxf(top, sm.m[w][row]);
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < W; ++w) sum = fmaf(sm.l[w][row], exp2_fast(sm.m[w][row] - top), sum);
                    float4 acc = sm.o[0][row][c4];
#pragma unroll
                    for (int w = 1; w < H; ++w) {
                        const float4 y = sm.o[w][row][c4];
                        acc = make_float4(acc.x + y.x, acc.y + y.y, acc.z + y.z, acc.w + y.w);
                    }
                    if (all) {
                        put(row, c4, acc, sum);
                    } else if (a.p.cluster > 1) {
                        sm.o[0][row][c4] = acc;       // (no other thread reads or writes this place)
                        if (c4 == 0) sm.ml[row] = make_float2(top, sum);
                    } else {
                        *reinterpret_cast<float4*>(a.w.part + (slot * ROWS + row) * D + 4 * c4) = acc;
                        if (c4 == 0) *reinterpret_cast<float2*>(a.w.part_ml + (slot * ROWS + row) * 2) = make_float2(top, sum);
                    }
                }
                if (a.p.cluster > 1) {                // the cluster's CTAs each join a part of the item's outputs
                    cluster_sync();
                    const int total = rows * (D / 4), share = (total + a.p.cluster - 1) / a.p.cluster;
                    const int first = (int)(blockIdx.x % (unsigned)a.p.cluster) * share;
                    for (int i = first + tid; i < min(first + share, total); i += NTHR) {
                        const int row = i / (D / 4), c4 = i % (D / 4);
                        float top = kLow, sum = 0.0f;
                        for (int k = 0; k < a.p.cluster; ++k) top = fmaxf(top, remote<float2>(&sm.ml[row], k).x);
                        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                        for (int k = 0; k < a.p.cluster; ++k) {
                            const float2 ml = remote<float2>(&sm.ml[row], k);
                            const float4 y = remote<float4>(&sm.o[0][row][c4], k);
                            const float f = exp2_fast(ml.x - top);
                            sum = fmaf(ml.y, f, sum);
                            acc = make_float4(fmaf(y.x, f, acc.x), fmaf(y.y, f, acc.y), fmaf(y.z, f, acc.z), fmaf(y.w, f, acc.w));
                        }
                        put(row, c4, acc, sum);
                    }
                    cluster_sync();                   // no CTA leaves while its sums are read
                }
                __syncthreads();                      // sm.m, sm.o and the rows are free again
            }
        }
        if (!a.p.split) break;
    }
    // A wait gave up: nothing of this CTA may be in flight when it ends
    if (lost)
        for (int i = 0; i < kStages; ++i) drain(&sm.full[warp][i]);
}

// ---- the alpha-entmax threshold ----------------------------------------------------
// One CTA an item's eight rows, a warp a row in the end.  A row's support lies
// within 1 of its largest x = (alpha - 1) score, and above the threshold of any part of
// its x: a few of Newton's steps over the tiles' maxima give such a bound (to the left
// of the root the steps stay there, the sum being convex for alpha <= 2).  Of the tiles whose
// maxima reach it (listed first) each such x is put on its row's list, every lane in a stretch of its
// own, so that no sum depends on timing; the stretches are closed up, and the root of
// sum (x - tau)_+^(1/(alpha-1)) = 1 is found among them by Newton's steps from the left,
// kept inside a bracket.  Rows with more than a list holds (a flat row, a small
// alpha) have every step read the tiles again.  One dependent step after another is
// what it costs: 9 us over 2000 tokens, 14 over 32768 (64 items, 2 MB of maxima).
constexpr int kTauThreads = 512, kTauWarps = kTauThreads / 32;
constexpr int kTileList = 2048;       // tiles listed
constexpr int kListCap = 1024;        // of a row, closed up
// Without the bound, 8 sequences of 32768 tokens took 84 to 131 us by their numbers (a list
// overflowed now and then), with it 80; three guesses of 2000 tokens 24.0 without, 25.4 with.
constexpr int kBoundSteps = 4;
constexpr int kPart = 13;             // of a row and lane (odd: no bank twice)
// A threshold lies n^-(alpha-1) below n equal largest x: at alpha 3 and 1500 of them 4e-7, less than
// fp32 tells apart at x = 20.  So it is held relative to the largest x, and found to this part of itself.
constexpr float kDone = 4e-7f;
constexpr int kTauSmem = (kTileList + 8 * kListCap + 8 * kTauWarps * 8 * kPart) * 4;

template <int NT>
__global__ void __launch_bounds__(kTauThreads) threshold_kernel(const __grid_constant__ Args a) {
    constexpr int ROWS = 8 * NT, W = kTauWarps;
    extern __shared__ int s_tiles[];
    float* const s_list = reinterpret_cast<float*>(s_tiles + kTileList);     // [8][kListCap]
    float* const s_part = s_list + 8 * kListCap;                             // [8][W * 8][kPart]
    __shared__ float s_max[W][8], s_top[8], s_low[8], s_sum[W][8][2], s_tau[8];
    __shared__ int s_count[W], s_rows[8][W * 8], s_mine[8];
    follow();
    const Shape& s = a.s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane >> 3;
    const int per = a.p.tiles * s.H, nt = blockIdx.x % NT;
    const int64_t item_no = blockIdx.x / NT;
    const int u = (int)(item_no / per), tile = (int)(item_no % per) % a.p.tiles;
    const int rows = min(8, a.p.R - tile * ROWS - 8 * nt);
    float* tau_out = a.w.tau + item_no * ROWS + 8 * nt;
    float2* edge_out = a.w.edge + item_no * ROWS + 8 * nt;
    if (rows <= 0) {
        if (tid < 8) tau_out[tid] = INFINITY, edge_out[tid] = make_float2(0.0f, INFINITY);
        return;
    }
    const int nb = unit_tiles(a, u);
    const float* tops = a.w.top + item_no * a.p.cap * ROWS + 8 * nt;
    const float4* tiles = a.w.score + (item_no * a.p.cap * kTile * NT + nt) * 32;
    auto tops_of = [&](int j, float (&y)[8]) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(tops + (int64_t)j * ROWS));
        const float4 z = __ldg(reinterpret_cast<const float4*>(tops + (int64_t)j * ROWS) + 1);
        y[0] = x.x, y[1] = x.y, y[2] = x.z, y[3] = x.w, y[4] = z.x, y[5] = z.y, y[6] = z.z, y[7] = z.w;
    };
    // the rows' maxima (-inf in rows past the last)
    float top[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) top[i] = -INFINITY;
#pragma unroll 4
    for (int j = tid; j < nb; j += kTauThreads) {
        float y[8];
        tops_of(j, y);
        // on the rows' lists for now, from kListCap tiles on the larger of what shares a place
        float* const place = s_list + j % kListCap;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top[i] = max_nan(top[i], y[i]);
            place[i * kListCap] = j < kListCap ? y[i] : max_nan(place[i * kListCap], y[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int k = 16; k; k >>= 1) top[i] = max_nan(top[i], __shfl_xor_sync(~0u, top[i], k));
        if (lane == 0) s_max[warp][i] = top[i];
    }
    __syncthreads();
    if (tid < 8) {
        float y = s_max[0][tid];
        for (int w = 1; w < W; ++w) y = max_nan(y, s_max[w][tid]);
        s_top[tid] = y;
    }
    const float ex = 1.0f / (s.alpha - 1.0f);
    auto gain = [&](float y, float tau, float& f, float& df) {   // y, tau relative to the row's maximum
        const float d = y - tau;
        if (!(d > 0.0f)) return;
        if (s.alpha == 1.5f) {
            f = fmaf(d, d, f);
            df = fmaf(2.0f, d, df);
        } else {
            const float p = exp2f(log2f(d) * ex);
            f += p;
            df += ex * p / d;
        }
    };
    __syncthreads();
    if (warp < 8) {                                   // row `warp`: a bound of its threshold
        const float* list = s_list + warp * kListCap;
        const float y0 = s_top[warp];
        float tau = -1.0f;
        for (int it = 0; it < (s.alpha <= 2.0f ? kBoundSteps : 0); ++it) {
            float f = 0.0f, df = 0.0f;
#pragma unroll 4
            for (int i = lane; i < min(nb, kListCap); i += 32) gain(list[i] - y0, tau, f, df);
#pragma unroll
            for (int k = 16; k; k >>= 1) {
                f += __shfl_xor_sync(~0u, f, k);
                df += __shfl_xor_sync(~0u, df, k);
            }
            if (!(f > 1.0f)) break;                   // (also: no key, or a NaN)
            tau += (f - 1.0f) / df;
        }
        if (lane == 0) s_low[warp] = fmaxf(tau - 1e-4f, -1.0f);   // sums of fp32 are not that far off
    }
    __syncthreads();
    float low[8];                                     // x that may have weight lie above
#pragma unroll
    for (int i = 0; i < 8; ++i) low[i] = s_top[i] + s_low[i];
    const float low0 = s_low[2 * t], low1 = s_low[2 * t + 1];
    const float top0 = 2 * t < rows ? s_top[2 * t] : INFINITY, top1 = 2 * t + 1 < rows ? s_top[2 * t + 1] : INFINITY;
    // the tiles that may hold support, in order
    int listed = 0;
    for (int base = 0; base < nb; base += kTauThreads) {
        bool want = false;
        if (base + tid < nb) {
            float y[8];
            tops_of(base + tid, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) want |= y[i] > low[i];
        }
        const uint32_t votes = __ballot_sync(~0u, want);
        if (lane == 0) s_count[warp] = __popc(votes);
        __syncthreads();
        int at = listed + __popc(votes & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < W; ++w) {
            at += w < warp ? s_count[w] : 0;
            listed += s_count[w];
        }
        if (want && at < kTileList) s_tiles[at] = base + tid;
        __syncthreads();
    }
    // the warp's share of them, several tiles' loads at a time; fn(four scores of rows 2t, 2t + 1)
    auto each = [&](auto fn) {
        constexpr int U = 4;
        const bool all = listed > kTileList;          // (then every tile is read)
        const int n = all ? nb : listed;
        for (int i0 = warp; i0 < n; i0 += U * W) {
            float4 y[2 * U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int i = i0 + k * W;
                y[2 * k] = y[2 * k + 1] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (i < n && 2 * t < rows) {
                    const int64_t j = all ? i : s_tiles[i];
                    bool read = true;
                    if (all) {                        // (a tile that is not there has no scores)
                        float z[8];
                        tops_of((int)j, z);
                        read = false;
#pragma unroll
                        for (int e = 0; e < 8; ++e) read |= z[e] > low[e];
                    }
                    if (read) {
                        y[2 * k] = __ldg(tiles + j * kTile * NT * 32 + lane);
                        y[2 * k + 1] = __ldg(tiles + (j * kTile + 1) * NT * 32 + lane);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 2 * U; ++k) fn(y[k]);
        }
    };
    int n0 = 0, n1 = 0;                               // on the lane's stretches of rows 2t, 2t + 1
    const int stretch = warp * 8 + (lane & 7);
    float* const l0 = s_part + (2 * t * W * 8 + stretch) * kPart;
    float* const l1 = l0 + W * 8 * kPart;
    auto put = [&](float y, float least, float* list, int& n) {
        if (y > least) {
            if (n < kPart) list[n] = y;
            ++n;
        }
    };
    each([&](float4 y) {
        put(y.x - top0, low0, l0, n0);
        put(y.z - top0, low0, l0, n0);
        put(y.y - top1, low1, l1, n1);
        put(y.w - top1, low1, l1, n1);
    });
    s_rows[2 * t][stretch] = n0;
    s_rows[2 * t + 1][stretch] = n1;
    __syncthreads();
    if (warp < 8) {                                   // where row `warp`'s stretches go
        int n[W / 4], sum = 0;
#pragma unroll
        for (int k = 0; k < W / 4; ++k) n[k] = s_rows[warp][lane * (W / 4) + k], sum += n[k];
        int at = sum;
#pragma unroll
        for (int k = 1; k < 32; k <<= 1) {
            const int y = __shfl_up_sync(~0u, at, k);
            if (lane >= k) at += y;
        }
        if (lane == 31) s_mine[warp] = at;
        at -= sum;
#pragma unroll
        for (int k = 0; k < W / 4; ++k) s_rows[warp][lane * (W / 4) + k] = at, at += n[k];
    }
    bool fits = n0 <= kPart && n1 <= kPart;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) fits &= s_mine[i] <= kListCap;
    fits = __syncthreads_and(fits);
    const int mine = s_mine[warp & 7];                // on the list of row `warp`
    if (fits) {
        for (int k = 0; k < n0; ++k) s_list[2 * t * kListCap + s_rows[2 * t][stretch] + k] = l0[k];
        for (int k = 0; k < n1; ++k) s_list[(2 * t + 1) * kListCap + s_rows[2 * t + 1][stretch] + k] = l1[k];
    }
    __syncthreads();
    // One step: the bracket [lo, hi] around the root, the next point within it.  Above alpha 2 keys enter
    // the sum with infinite slope, and Newton's steps may go to and fro across one without end, or be
    // short far from the root: every second step halves the bracket (its logarithm, where it spans
    // more than two octaves), and the sum or the bracket tells the end: 16 to 20 steps, 34 at most
    // of 9000 rows of 2 to 3000 keys (Newton's alone 5 to 10, but some never ended, weights 7 % off).
    // One sequence of 4096 tokens, alpha 2.5: 26.0 us by Newton's alone, 33.8; 8 of 32768 83.5, 84.7.
    const bool steep = s.alpha > 2.0f;
    // no more than all keys share the sum: the root lies at least that far below the largest
    const float hi0 = steep ? -0.99f * exp2f((1.0f - s.alpha) * log2f((float)nb * (kTile * kBlock))) : 0.0f;
    auto step = [&](int it, float f, float df, float& lo, float& hi, float& tau) {
        if (f >= 1.0f) lo = tau; else hi = tau;
        const float next = tau + (f - 1.0f) / df;
        const bool inside = next >= lo && next <= hi;
        if (steep) {
            if (fabsf(f - 1.0f) <= 1e-6f || hi - lo <= kDone * fabsf(lo)) return true;
            const float mid = lo < 4.0f * hi ? -sqrtf(lo * hi) : 0.5f * (lo + hi);
            tau = inside && !(it & 1) ? next : mid;
            return false;
        }
        const float to_ = inside ? next : 0.5f * (lo + hi);
        const bool end = fminf(fabsf(to_ - tau), hi - lo) <= kDone * fabsf(to_);
        tau = to_;
        return end;
    };
    constexpr int kSteps = 100;
    if (fits) {
        if (warp < 8) {
            const float* list = s_list + warp * kListCap;
            float tau = s_low[warp], lo = tau, hi = hi0;
            for (int it = 0; it < kSteps; ++it) {
                float f = 0.0f, df = 0.0f;
                for (int i = lane; i < mine; i += 32) gain(list[i], tau, f, df);
#pragma unroll
                for (int k = 16; k; k >>= 1) {
                    f += __shfl_xor_sync(~0u, f, k);
                    df += __shfl_xor_sync(~0u, df, k);
                }
                if (step(it, f, df, lo, hi, tau)) break;
            }
            if (lane == 0) s_tau[warp] = tau;
        }
    } else {
        float tau[2] = {low0, low1}, lo[2] = {low0, low1}, hi[2] = {hi0, hi0};
        for (int it = 0; it < kSteps; ++it) {
            float f[2] = {0.0f, 0.0f}, df[2] = {0.0f, 0.0f};
            each([&](float4 y) {
                gain(y.x - top0, tau[0], f[0], df[0]);
                gain(y.z - top0, tau[0], f[0], df[0]);
                gain(y.y - top1, tau[1], f[1], df[1]);
                gain(y.w - top1, tau[1], f[1], df[1]);
            });
            bool end = true;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int k = 4; k; k >>= 1) {
                    f[e] += __shfl_xor_sync(~0u, f[e], k);
                    df[e] += __shfl_xor_sync(~0u, df[e], k);
                }
                if ((lane & 7) == 0) s_sum[warp][2 * t + e][0] = f[e], s_sum[warp][2 * t + e][1] = df[e];
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sf = 0.0f, sd = 0.0f;
                for (int w = 0; w < W; ++w) sf += s_sum[w][2 * t + e][0], sd += s_sum[w][2 * t + e][1];
                const float y = e ? top1 : top0;
                if (y > -INFINITY && y < INFINITY) end &= step(it, sf, sd, lo[e], hi[e], tau[e]);
            }
            if (__syncthreads_and(end)) break;
        }
        if (warp == 0 && (lane & 7) == 0) s_tau[2 * t] = tau[0], s_tau[2 * t + 1] = tau[1];
    }
    __syncthreads();
    if (tid < 8) {
        const float y = s_top[tid];                   // (NaN where a score is)
        const bool none = y == -INFINITY;
        tau_out[tid] = none ? INFINITY : __fadd_rd(y, s_tau[tid]);
        edge_out[tid] = none ? make_float2(0.0f, INFINITY) : make_float2(y, s_tau[tid]);
    }
}

// ---- host --------------------------------------------------------------------------
template <int NT>
constexpr int warps_of() { return NT == 1 ? 8 : 4; }
constexpr int ctas_of(int nt) { return nt == 1 ? 2 : 3; }        // an SM holds

// Row tiles (of 8) that a CTA takes at once.  Two share the reading and unpacking of the
// codes, which pays where the tiles keep all warps busy: nine or more a warp, by
// the rows that fill them.  Us with one and with two: 64 sequences of 1024 tokens, 8
// key heads of 16 rows, head size 64, 53.7 and 38.5; 8 of 8192, 32 rows, 60.6 and 46.3; 32
// of 4096, 16 rows, head size 128, 98.6 and 94.8.  With fewer the smaller grain wins:
// 8 of 4096, 12 rows, 30.2 and 39.7; 1 of 4096, 14.1 and 19.7.
int row_tiles(const Shape& s, int keep) {
    const int64_t rows = keep ? s.G : (int64_t)s.T * s.G, blocks = (int64_t)(keep ? keep : s.width) * (s.P / kBlock);
    const int64_t tiles = (int64_t)(keep ? s.B * s.T : s.B) * s.H * ((blocks + kTile - 1) / kTile);
    return rows > 8 && tiles * rows >= 16ll * 9 * kSms * 3 * 4 ? 2 : 1;
}

Plan make_plan(const Shape& s, int keep) {
    Plan p;
    const int nt = row_tiles(s, keep);
    p.U = keep ? s.B * s.T : s.B;
    p.R = keep ? s.G : s.T * s.G;
    p.tiles = (p.R + 8 * nt - 1) / (8 * nt);
    p.keep = keep;
    p.cap = ((keep ? keep : s.width) * (s.P / kBlock) + kTile - 1) / kTile;
    const int64_t items = (int64_t)p.U * p.tiles * s.H, slots = (int64_t)kSms * ctas_of(nt);
    const int warps = nt == 1 ? 8 : 4;
    // An item is taken by one CTA, or by a cluster whose CTAs join their sums over
    // its shared memory: as many CTAs as have a tile a warp, and as the SMs hold for all
    // items at once.  Or else all items are cut into equal runs, one a CTA, at the price
    // of a second kernel: about five rounds, a round being a tile to each warp.  So they
    // are cut where that takes fewer rounds, lengths taken to be three quarters of
    // what the table holds.  Head size 128, 8 key heads of 4 query heads, us by CTA, by
    // cluster of the size taken, and by runs:
    //    1 sequence   of   512 tokens  9.4,  9.2, 12.3;  4096  32.4, 11.5, 14.0;  16384  111.2, 21.5, 16.9
    //    8 sequences  of  1024 tokens 13.1, 11.3, 16.7;  4096  33.5, 21.2, 24.5;  32768  219.6, 90.2, 85.9
    //   64 sequences  of  1024 tokens 36.1, -, 41.3;     4096  94.8, -, 95.6;      8192  172.1, -, 163.2
    const auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    p.cluster = 1;
    while (p.cluster < 8 && items * 2 * p.cluster <= slots && p.cap > p.cluster * warps) p.cluster *= 2;
    const int64_t whole = ceil_div(items * p.cluster, slots) * ceil_div(p.cap, p.cluster * warps);
    const int64_t runs = items * p.cap * (keep ? 4 : 3) / (4 * slots * warps) + 5;
    p.split = items < 8 * slots && whole > runs;      // (many items even out, and runs count them all)
    // The values of an entmax row are those of few tiles: taken to be a quarter at most,
    // items that fill the SMs at once are left whole more often, and need no join (with
    // all three kernels, 8 sequences of 32768 tokens, 8 key heads, 75.5 us, 79.2 with the
    // values cut as the scores; 32 of 4096 74.9, 78.1; but 1 of 32768, 64 CTAs, 77.2, 75.8).
    const bool fill = items * p.cluster <= slots && 2 * items * p.cluster > slots;
    p.values = p.split && s.alpha != 1.0f && fill && whole <= 4 * runs ? p.cluster : 0;
    if (p.split) p.cluster = 1;
    p.tile = kTile * kBlock;
    p.item_cost = keep ? kListedCost : kItemCost;
    p.least = nt == 1 ? 16 : 12;
    p.vec = 0;
    p.page_shift = 0;
    while (kBlock << p.page_shift < s.P) ++p.page_shift;
    return p;
}

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

// Offsets of the workspace's parts; its size.
size_t lay_out(const Shape& s, const Plan& p, void* base, Space* w) {
    const int nt = row_tiles(s, p.keep), rows = 8 * nt;
    const int64_t items = (int64_t)p.U * p.tiles * s.H, slots = 2ll * kSms * ctas_of(nt);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* q = (char*)base + at;
        at += up256(bytes);
        return q;
    };
    Space x{};
    if (p.split) {
        x.run = (int64_t*)take(((size_t)p.U + 1) * 8);
        x.part = (float*)take((size_t)slots * rows * s.d * 4);
        x.part_ml = (float*)take((size_t)slots * 2 * rows * 4);
    }
    if (s.alpha != 1.0f) {
        x.score = (float4*)take((size_t)items * p.cap * kTile * nt * 512);
        x.top = (float*)take((size_t)items * p.cap * rows * 4);
        x.tau = (float*)take((size_t)items * rows * 4);
        x.edge = (float2*)take((size_t)items * rows * 8);
    }
    if (w) *w = x;
    return at;
}

template <int D, int NT, int MODE>
cudaError_t launch_walk(const Args& a, cudaStream_t st) {
    constexpr int W = warps_of<NT>();
    const int smem = (int)sizeof(Smem<D, NT, W>);
    auto kernel = walk_kernel<D, NT, W, MODE>;
    static Allowed allowed;
    cudaError_t e = allow_shared(kernel, smem, allowed);
    if (e != cudaSuccess) return e;
    const int64_t items = (int64_t)a.p.U * a.p.tiles * a.s.H;
    const unsigned grid = a.p.split ? kSms * ctas_of(NT) : (unsigned)(items * a.p.cluster);
    return launch_clusters(a.p.cluster, kernel, grid, W * 32, smem, st, a);
}

template <int D, int NT>
cudaError_t attend_as(const Args& a, cudaStream_t st) {
    const int64_t items = (int64_t)a.p.U * a.p.tiles * a.s.H;
    if (items * 8 * NT > 0x7fffffff) return cudaErrorInvalidConfiguration;
    cudaError_t e;
    if (a.s.alpha == 1.0f) {
        e = launch_walk<D, NT, kSoftmax>(a, st);
    } else {
        e = launch_walk<D, NT, kScores>(a, st);
        if (e != cudaSuccess) return e;
        static Allowed allowed;
        e = allow_shared(threshold_kernel<NT>, kTauSmem, allowed);
        if (e != cudaSuccess) return e;
        e = launch(threshold_kernel<NT>, (unsigned)(items * NT), kTauThreads, kTauSmem, st, a);
        if (e != cudaSuccess) return e;
        if (a.p.values) {
            Args v = a;
            v.p.split = 0;
            v.p.cluster = a.p.values;
            return launch_walk<D, NT, kValues>(v, st);
        }
        e = launch_walk<D, NT, kValues>(a, st);
    }
    if (e != cudaSuccess || !a.p.split) return e;
    // eight warps share a row's parts where items are few (2 sequences of 131072 tokens, 4
    // key heads, with the walk: 51.1 us, 53.5 by four), else four (48 of up to 8192, 8 key
    // heads: 52.3 by eight, 50.0)
    if (items * 8 <= 4 * kSms) return launch(combine_kernel<D, 8 * NT, NT, 8>, (unsigned)(items * 8), 256, 0, st, a);
    return launch(combine_kernel<D, 8 * NT, NT, 4>, (unsigned)(items * 8), 128, 0, st, a);
}

}  // namespace

// Lane 0 waits, with the kernels' bounded wait, for an arrival that nobody makes; then it
// completes the barrier itself, so that nothing is pending when the block ends.
__global__ void wait_probe_kernel(int naps, int* err) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        sm100::mbar_init(&bar, 1);
        sm100::fence_barrier_init();
        wait_full(&bar, 0, naps, err);
        sm100::mbar_arrive(&bar);
    }
    __syncwarp();
}

cudaError_t wait_probe(int naps, int* err, cudaStream_t st) {
    wait_probe_kernel<<<1, 32, 0, st>>>(naps, err);
    note_launch();
    return cudaGetLastError();
}

size_t attend_workspace(const Shape& s, int keep) {
    if (chunk_takes(s, keep)) return chunk_workspace(s);
    return lay_out(s, make_plan(s, keep), nullptr, nullptr);
}

cudaError_t attend(const Shape& s, const void* Q, Strides qs, const uint8_t* pool, const int32_t* table,
                   const int32_t* lengths, const int32_t* list, int keep, void* O, void* ws, int* err,
                   cudaStream_t st) {
    if (chunk_takes(s, keep)) return chunk_attend(s, Q, qs, pool, table, lengths, O, ws, err, st);
    Args a;
    a.s = s;
    a.p = make_plan(s, keep);
    lay_out(s, a.p, ws, &a.w);
    a.qs = qs;
    a.Q = (const __nv_bfloat16*)Q;
    a.pool = pool;
    a.table = table;
    a.lengths = lengths;
    a.list = list;
    a.O = (__nv_bfloat16*)O;
    a.err = err;
    a.p.vec = (reinterpret_cast<uintptr_t>(Q) & 15) == 0 && qs.b % 8 == 0 && qs.t % 8 == 0 && qs.h % 8 == 0;
    const bool two = row_tiles(s, keep) == 2;
    switch (s.d) {
        case 32: return two ? attend_as<32, 2>(a, st) : attend_as<32, 1>(a, st);
        case 64: return two ? attend_as<64, 2>(a, st) : attend_as<64, 1>(a, st);
        case 96: return two ? attend_as<96, 2>(a, st) : attend_as<96, 1>(a, st);
        default: return two ? attend_as<128, 2>(a, st) : attend_as<128, 1>(a, st);
    }
}

}  // namespace cache
}  // namespace asa
