// asa_cache_capi.cu -- the extern "C" entry points of the 4-bit paged cache:
// argument checks, workspaces and launches.  Nothing is allocated or
// synchronised here; errors come back as status codes.
#include "asa_cache.h"

#include <climits>
#include <cmath>

namespace {

using asa::cache::Shape;
using asa::cache::Strides;

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The training kernels' spins, sixteen to a nap (five seconds by default).
int naps_of(long long spins) { return (int)((spins >> 4) + 1 < (1 << 30) ? (spins >> 4) + 1 : (1 << 30)); }

int check(const asa_cache_params* p, Shape* s, bool queries) {
    if (!p) return ASA_ERR_INVALID;
    if (p->B < 0 || p->T < 0 || p->kv_heads < 1 || p->num_pages < 0 || p->table_width < 0)
        return ASA_ERR_INVALID;
    if (p->d < 1 || p->page_size < 1) return ASA_ERR_INVALID;
    if (p->dtype != ASA_DTYPE_F32 && p->dtype != ASA_DTYPE_BF16) return ASA_ERR_INVALID;
    if (queries) {
        if (p->heads < 1 || p->heads % p->kv_heads) return ASA_ERR_INVALID;
        if (!std::isfinite(p->sm_scale) || !std::isfinite(p->alpha)) return ASA_ERR_INVALID;
        if (p->alpha != 1.0f && !(p->alpha >= 1.05f && p->alpha <= 3.0f)) return ASA_ERR_INVALID;
    }
    if (p->d % 32 || p->d > 128) return ASA_ERR_UNSUPPORTED;
    if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
        return ASA_ERR_UNSUPPORTED;
    const long long rows = (long long)p->B * p->T;
    // positions and (row, page) numbers are 32-bit integers in the kernels
    if ((long long)p->table_width * p->page_size > INT_MAX / 2 || rows > INT_MAX / 2 ||
        rows * (queries ? p->heads : p->kv_heads) > INT_MAX / 4 ||
        (long long)p->num_pages * p->kv_heads > INT_MAX / 2)
        return ASA_ERR_UNSUPPORTED;
    s->B = p->B;
    s->T = p->T;
    s->H = p->kv_heads;
    s->HQ = queries ? p->heads : p->kv_heads;
    s->G = s->HQ / s->H;
    s->d = p->d;
    s->P = p->page_size;
    s->pages = p->num_pages;
    s->width = p->table_width;
    s->dtype = p->dtype;
    s->scale = p->sm_scale;
    s->alpha = p->alpha;
    s->naps = naps_of(p->timeout_spins > 0 ? p->timeout_spins : (1LL << 22));
    s->rec = asa::cache::record_bytes(p->d, p->page_size);
    return ASA_OK;
}

bool lacks(const void* ws, size_t bytes, size_t need) { return need && (bytes < need || !ws || !aligned(ws, 16)); }

Strides strides(const int64_t v[3]) { return Strides{v[0], v[1], v[2]}; }

// Times what is launched while it lives, when profiling is on.
struct Scope {
    void* at;
    Scope(const char* label, cudaStream_t st) : at(asa::profile_open(label, st)) {}
    ~Scope() { asa::profile_close(at); }
};

}  // namespace

extern "C" {

long long asa_cache_record_bytes(int d, int page_size) {
    if (d < 1 || d % 32 || d > 128 || page_size < 16 || page_size % 16) return 0;
    return asa::cache::record_bytes(d, page_size);
}

int asa_cache_workspace_bytes(const asa_cache_params* p, int keep, size_t* attend_bytes,
                              size_t* select_bytes) {
    Shape s;
    int rc = check(p, &s, true);
    if (rc) return rc;
    if (keep < 0) return ASA_ERR_INVALID;
    if (attend_bytes) *attend_bytes = asa::cache::attend_workspace(s, keep);
    if (select_bytes) *select_bytes = asa::cache::select_workspace(s);
    return ASA_OK;
}

int asa_cache_wait_probe(long long spins, asa_stream_t stream) {
    if (spins < 1) return ASA_ERR_INVALID;
    int* w = asa::cache_error_word();
    if (!w) return ASA_ERR_CUDA;
    return asa::cuda_status_of(asa::cache::wait_probe(naps_of(spins), w, (cudaStream_t)stream));
}

int asa_cache_write(const asa_cache_params* p, const void* K, const void* V, const int64_t k_strides[3],
                    const int64_t v_strides[3], void* pool, void* bounds, const int32_t* block_table,
                    const int32_t* start, const int32_t* count, asa_stream_t stream) {
    Shape s;
    int rc = check(p, &s, false);
    if (rc) return rc;
    if (!s.B || !s.T) return ASA_OK;
    if (!K || !V || !k_strides || !v_strides || !start || (s.width && !block_table) ||
        (s.pages && (!pool || !bounds)))
        return ASA_ERR_INVALID;
    if (!aligned(pool, 16) || !aligned(bounds, 16)) return ASA_ERR_INVALID;
    cudaStream_t st = (cudaStream_t)stream;
    Scope ps("cache_write", st);
    return asa::cuda_status_of(asa::cache::write(s, K, V, strides(k_strides), strides(v_strides),
                                                 (uint8_t*)pool, (int8_t*)bounds, block_table, start,
                                                 count, asa::cache_error_word(), st));
}

int asa_cache_read(const asa_cache_params* p, const void* pool, const int32_t* block_table,
                   const int32_t* start, const int32_t* count, void* K, void* V, asa_stream_t stream) {
    Shape s;
    int rc = check(p, &s, false);
    if (rc) return rc;
    if (!s.B || !s.T) return ASA_OK;
    if (!K || !V || !start || (s.width && !block_table) || (s.pages && !pool)) return ASA_ERR_INVALID;
    if (!aligned(pool, 16) || !aligned(K, 16) || !aligned(V, 16)) return ASA_ERR_INVALID;
    cudaStream_t st = (cudaStream_t)stream;
    Scope ps("cache_read", st);
    return asa::cuda_status_of(asa::cache::read(s, (const uint8_t*)pool, block_table, start, count, K, V,
                                                asa::cache_error_word(), st));
}

int asa_cache_bounds(const asa_cache_params* p, const void* bounds, const int32_t* pages, int n,
                     float* upper, float* lower, asa_stream_t stream) {
    Shape s;
    int rc = check(p, &s, false);
    if (rc) return rc;
    if (n < 0 || (long long)n * s.H > INT_MAX / 2) return ASA_ERR_INVALID;
    if (!n) return ASA_OK;
    if (!pages || !upper || !lower || (s.pages && !bounds)) return ASA_ERR_INVALID;
    if (!aligned(bounds, 16)) return ASA_ERR_INVALID;
    cudaStream_t st = (cudaStream_t)stream;
    Scope ps("cache_bounds", st);
    return asa::cuda_status_of(asa::cache::read_bounds(s, (const int8_t*)bounds, pages, n, upper, lower,
                                                       asa::cache_error_word(), st));
}

int asa_cache_select(const asa_cache_params* p, const void* Q, const int64_t q_strides[3],
                     const void* bounds, const int32_t* block_table, const int32_t* lengths, int keep,
                     int32_t* pages, void* ws, size_t ws_bytes, asa_stream_t stream) {
    Shape s;
    int rc = check(p, &s, true);
    if (rc) return rc;
    if (keep < 1) return ASA_ERR_INVALID;
    if (s.G > 256) return ASA_ERR_UNSUPPORTED;           // a query's heads are held in shared memory
    if (!s.B || !s.T) return ASA_OK;
    if ((long long)s.B * s.T * s.H * keep > (1LL << 40)) return ASA_ERR_UNSUPPORTED;
    if (!Q || !q_strides || !lengths || !pages || (s.width && !block_table) || (s.pages && !bounds))
        return ASA_ERR_INVALID;
    if (!aligned(bounds, 16)) return ASA_ERR_INVALID;
    if (lacks(ws, ws_bytes, asa::cache::select_workspace(s))) return ASA_ERR_WORKSPACE;
    cudaStream_t st = (cudaStream_t)stream;
    Scope ps("cache_select", st);
    return asa::cuda_status_of(asa::cache::select(s, Q, strides(q_strides), (const int8_t*)bounds,
                                                  block_table, lengths, keep, pages, ws,
                                                  asa::cache_error_word(), st));
}

int asa_cache_attention(const asa_cache_params* p, const void* Q, const int64_t q_strides[3],
                        const void* pool, const int32_t* block_table, const int32_t* lengths,
                        const int32_t* pages, int keep, void* O, void* ws, size_t ws_bytes,
                        asa_stream_t stream) {
    Shape s;
    int rc = check(p, &s, true);
    if (rc) return rc;
    if (keep < 0 || (pages && keep < 1) || (!pages && keep)) return ASA_ERR_INVALID;
    if ((long long)keep * s.P > INT_MAX / 2) return ASA_ERR_UNSUPPORTED;
    if (!s.B || !s.T) return ASA_OK;
    if (!Q || !q_strides || !lengths || !O || (s.width && !block_table) || (s.pages && !pool))
        return ASA_ERR_INVALID;
    if (!aligned(pool, 16) || !aligned(O, 16)) return ASA_ERR_INVALID;
    if (lacks(ws, ws_bytes, asa::cache::attend_workspace(s, keep))) return ASA_ERR_WORKSPACE;
    cudaStream_t st = (cudaStream_t)stream;
    Scope ps(s.alpha == 1.0f ? "cache_attention" : "cache_entmax", st);
    return asa::cuda_status_of(asa::cache::attend(s, Q, strides(q_strides), (const uint8_t*)pool,
                                                  block_table, lengths, pages, keep, O, ws,
                                                  asa::cache_error_word(), st));
}

}  // extern "C"
