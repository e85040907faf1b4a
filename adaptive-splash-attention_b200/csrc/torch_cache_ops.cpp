// torch_cache_ops.cpp -- the 4-bit paged cache's operators registered with
// PyTorch's dispatcher, a thin layer over the C ABI of libasa.so.
//
//   splash_attention::cache_write(K, V, pool!, bounds!, block_table, start, count?)
//   splash_attention::cache_read(pool, bounds, block_table, start, T, count?, out_f32) -> (K, V)
//   splash_attention::cache_bounds(bounds, pages) -> (upper, lower)
//   splash_attention::cache_select(Q, pool, bounds, block_table, lengths, keep) -> pages
//   splash_attention::cache_attention(Q, pool, bounds, block_table, lengths, pages?, sm_scale, alpha) -> O
//
// Outputs and workspaces come from PyTorch's caching allocator; launches go on
// the current stream of the tensors' device.  Bad shapes raise ValueError, bad
// types TypeError, everything else RuntimeError.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <climits>
#include <string>

#include "../../include/asa.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void check(int rc, const char* what) {
    if (rc == ASA_OK) return;
    std::string msg = std::string(what) + ": " + asa_status_string(rc) + " (asa_status " + std::to_string(rc) + ")";
    if (rc == ASA_ERR_CUDA) msg += std::string(": ") + asa_last_cuda_error();
    TORCH_CHECK(false, msg);
}

int int_of(int64_t v, const char* what) {
    TORCH_CHECK_VALUE(v >= 0 && v <= INT_MAX, "splash_attention: ", what, " is out of range");
    return (int)v;
}

// The page size that a pool of records and a head dim imply.
int64_t page_size_of(const Tensor& pool, int64_t d) {
    TORCH_CHECK_TYPE(pool.scalar_type() == at::kByte, "splash_attention: the cache's pool must be uint8");
    TORCH_CHECK_VALUE(pool.dim() == 3 && d > 0 && d % 32 == 0 && d <= 128,
                      "splash_attention: the pool must be [pages, kv_heads, record], head_dim 32, 64, 96 or 128");
    const int64_t P = pool.size(2) * 4 / (5 * d);
    TORCH_CHECK_VALUE((P == 16 || P == 32 || P == 64 || P == 128) && asa_cache_record_bytes((int)d, (int)P) == pool.size(2),
                      "splash_attention: the pool's records do not fit head_dim ", d);
    TORCH_CHECK_VALUE(pool.is_contiguous(), "splash_attention: the cache's pool must be contiguous");
    return P;
}

void check_bounds(const Tensor& bounds, int64_t d) {
    TORCH_CHECK_TYPE(bounds.scalar_type() == at::kChar, "splash_attention: the cache's bounds must be int8");
    TORCH_CHECK_VALUE(bounds.dim() == 3 && bounds.size(2) == 2 * d + ASA_CACHE_BOUNDS_PAD && bounds.is_contiguous(),
                      "splash_attention: the bounds must be contiguous [pages, kv_heads, 2 * head_dim + 16]");
}

void same_device(const Tensor& a, const Tensor& b, const char* name) {
    TORCH_CHECK(a.device() == b.device(), "splash_attention: ", name, " must be on ", a.device());
}

// Positions, lengths and tables as contiguous int32 on the cache's device.  Numbers that
// int32 does not hold become its ends, which lie outside every table and pool, not others.
Tensor index(const Tensor& t, const Tensor& like, c10::IntArrayRef shape, const char* name) {
    TORCH_CHECK_TYPE(at::isIntegralType(t.scalar_type(), false), "splash_attention: ", name, " must hold integers");
    same_device(like, t, name);
    TORCH_CHECK_VALUE(t.dim() == (int64_t)shape.size(), "splash_attention: ", name, " must have ", shape.size(), " dimensions");
    for (size_t i = 0; i < shape.size(); ++i)
        TORCH_CHECK_VALUE(shape[i] < 0 || t.size(i) == shape[i], "splash_attention: ", name, " has shape ", t.sizes());
    const auto type = t.scalar_type();
    if (type == at::kInt) return t.contiguous();
    const bool wide = type == at::kLong || type == at::kUInt32 || type == at::kUInt64;
    return (wide ? t.to(at::kLong).clamp(INT_MIN, INT_MAX) : t).to(at::kInt).contiguous();
}

const int32_t* ints(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

asa_stream_t stream_of(const Tensor& t) {
    return (asa_stream_t)c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

struct Strided {      // a [B, T, heads, d] tensor whose channels are contiguous
    Tensor t;
    int64_t s[3];
    explicit Strided(const Tensor& x) : t(x.size(3) == 1 || x.stride(3) == 1 ? x : x.contiguous()) {
        for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
    }
};

asa_cache_params params(int64_t B, int64_t T, int64_t heads, int64_t kv_heads, int64_t d, int64_t page, int64_t pages,
                        int64_t width) {
    asa_cache_params p{};
    p.B = int_of(B, "the batch");
    p.T = int_of(T, "T");
    p.heads = int_of(heads, "heads");
    p.kv_heads = int_of(kv_heads, "kv_heads");
    p.d = int_of(d, "head_dim");
    p.page_size = int_of(page, "page_size");
    p.num_pages = int_of(pages, "pages");
    p.table_width = int_of(width, "the block table's width");
    p.dtype = ASA_DTYPE_BF16;
    p.sm_scale = 1.0f;
    p.alpha = 1.0f;
    return p;
}

int dtype_code(at::ScalarType t) {
    TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16, "splash_attention: unsupported dtype ", t,
                     " (float32 or bfloat16)");
    return t == at::kFloat ? ASA_DTYPE_F32 : ASA_DTYPE_BF16;
}

void write_cuda(const Tensor& K, const Tensor& V, const Tensor& pool, const Tensor& bounds, const Tensor& block_table,
                const Tensor& start, const OptTensor& count) {
    TORCH_CHECK_VALUE(K.dim() == 4 && V.sizes() == K.sizes(),
                      "splash_attention: K and V must be [B, T, kv_heads, head_dim], of one shape");
    TORCH_CHECK_TYPE(K.scalar_type() == V.scalar_type(), "splash_attention: K and V must have one dtype");
    const int code = dtype_code(K.scalar_type());
    const int64_t B = K.size(0), T = K.size(1), H = K.size(2), d = K.size(3);
    const int64_t P = page_size_of(pool, d);
    check_bounds(bounds, d);
    TORCH_CHECK_VALUE(pool.size(1) == H && bounds.size(1) == H && pool.size(0) == bounds.size(0),
                      "splash_attention: the cache's pool and bounds must have K's heads and one number of pages");
    same_device(K, V, "V");
    same_device(K, pool, "the pool");
    same_device(K, bounds, "the bounds");
    const Tensor tab = index(block_table, K, {B, -1}, "block_table"), st = index(start, K, {B}, "start");
    Tensor cnt;
    if (count.has_value() && count->defined()) cnt = index(*count, K, {B}, "count");
    c10::cuda::CUDAGuard guard(K.device());
    const Strided k(K), v(V);
    asa_cache_params p = params(B, T, H, H, d, P, pool.size(0), tab.size(1));
    p.dtype = code;
    check(asa_cache_write(&p, k.t.data_ptr(), v.t.data_ptr(), k.s, v.s, pool.data_ptr(), bounds.data_ptr(), ints(tab),
                          ints(st), ints(cnt), stream_of(K)),
          "asa_cache_write");
}

int64_t head_dim_of(const Tensor& bounds) {
    TORCH_CHECK_VALUE(bounds.dim() == 3 && bounds.size(2) > ASA_CACHE_BOUNDS_PAD,
                      "splash_attention: the bounds must be [pages, kv_heads, 2 * head_dim + 16]");
    return (bounds.size(2) - ASA_CACHE_BOUNDS_PAD) / 2;
}

std::tuple<Tensor, Tensor> read_cuda(const Tensor& pool, const Tensor& bounds, const Tensor& block_table,
                                     const Tensor& start, int64_t T, const OptTensor& count, bool out_f32) {
    const int64_t d = head_dim_of(bounds);
    const int64_t P = page_size_of(pool, d), H = pool.size(1);
    TORCH_CHECK_VALUE(start.dim() == 1, "splash_attention: start must be [B]");
    const int64_t B = start.size(0);
    TORCH_CHECK_VALUE(T >= 0, "splash_attention: T must not be negative");
    const Tensor tab = index(block_table, pool, {B, -1}, "block_table"), st = index(start, pool, {B}, "start");
    Tensor cnt;
    if (count.has_value() && count->defined()) cnt = index(*count, pool, {B}, "count");
    c10::cuda::CUDAGuard guard(pool.device());
    const auto opt = pool.options().dtype(out_f32 ? at::kFloat : at::kBFloat16);
    Tensor K = at::empty({B, T, H, d}, opt), V = at::empty({B, T, H, d}, opt);
    asa_cache_params p = params(B, T, H, H, d, P, pool.size(0), tab.size(1));
    p.dtype = out_f32 ? ASA_DTYPE_F32 : ASA_DTYPE_BF16;
    check(asa_cache_read(&p, pool.data_ptr(), ints(tab), ints(st), ints(cnt), K.data_ptr(), V.data_ptr(), stream_of(pool)),
          "asa_cache_read");
    return {K, V};
}

std::tuple<Tensor, Tensor> bounds_cuda(const Tensor& bounds, const Tensor& pages) {
    const int64_t d = head_dim_of(bounds), H = bounds.size(1);
    check_bounds(bounds, d);
    const Tensor ids = index(pages, bounds, {-1}, "pages");
    c10::cuda::CUDAGuard guard(bounds.device());
    const auto opt = bounds.options().dtype(at::kFloat);
    Tensor upper = at::empty({ids.size(0), H, d}, opt), lower = at::empty({ids.size(0), H, d}, opt);
    asa_cache_params p = params(1, 1, H, H, d, 16, bounds.size(0), 0);
    check(asa_cache_bounds(&p, bounds.data_ptr(), ints(ids), int_of(ids.size(0), "the number of pages"),
                           upper.data_ptr<float>(), lower.data_ptr<float>(), stream_of(bounds)),
          "asa_cache_bounds");
    return {upper, lower};
}

void check_queries(const Tensor& Q, int64_t kv_heads) {
    TORCH_CHECK_VALUE(Q.dim() == 4, "splash_attention: q must be [B, T, heads, head_dim]");
    TORCH_CHECK_TYPE(Q.scalar_type() == at::kBFloat16, "splash_attention: q must be bfloat16, got ", Q.scalar_type());
    TORCH_CHECK_VALUE(kv_heads > 0 && Q.size(2) > 0 && Q.size(2) % kv_heads == 0, "splash_attention: q's ", Q.size(2),
                      " heads are not a multiple of the cache's ", kv_heads);
}

Tensor select_cuda(const Tensor& Q, const Tensor& pool, const Tensor& bounds, const Tensor& block_table,
                   const Tensor& lengths, int64_t keep) {
    TORCH_CHECK_VALUE(bounds.dim() == 3 && Q.dim() == 4, "splash_attention: q must be [B, T, heads, head_dim]");
    const int64_t B = Q.size(0), T = Q.size(1), d = Q.size(3), H = bounds.size(1);
    check_queries(Q, H);
    check_bounds(bounds, d);
    const int64_t page_size = page_size_of(pool, d);
    same_device(Q, bounds, "the bounds");
    TORCH_CHECK_VALUE(keep >= 1 && keep <= INT_MAX, "splash_attention: keep must be at least 1");
    const Tensor tab = index(block_table, Q, {B, -1}, "block_table"), len = index(lengths, Q, {B}, "lengths");
    c10::cuda::CUDAGuard guard(Q.device());
    const Strided q(Q);
    asa_cache_params p = params(B, T, Q.size(2), H, d, page_size, bounds.size(0), tab.size(1));
    Tensor out = at::empty({B, T, H, keep}, Q.options().dtype(at::kInt));
    size_t bytes = 0;
    check(asa_cache_workspace_bytes(&p, 0, nullptr, &bytes), "asa_cache_workspace_bytes");
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, Q.options().dtype(at::kByte));
    check(asa_cache_select(&p, q.t.data_ptr(), q.s, bounds.data_ptr(), ints(tab), ints(len), (int)keep,
                           out.data_ptr<int32_t>(), bytes ? ws.data_ptr() : nullptr, bytes, stream_of(Q)),
          "asa_cache_select");
    return out;
}

Tensor attention_cuda(const Tensor& Q, const Tensor& pool, const Tensor& bounds, const Tensor& block_table,
                      const Tensor& lengths, const OptTensor& pages, double sm_scale, double alpha) {
    TORCH_CHECK_VALUE(pool.dim() == 3, "splash_attention: the pool must be [pages, kv_heads, record]");
    check_queries(Q, pool.size(1));
    const int64_t B = Q.size(0), T = Q.size(1), HQ = Q.size(2), d = Q.size(3), H = pool.size(1);
    TORCH_CHECK_VALUE(head_dim_of(bounds) == d, "splash_attention: q's head_dim ", d, " is not the cache's");
    const int64_t P = page_size_of(pool, d);
    same_device(Q, pool, "the pool");
    TORCH_CHECK_VALUE(alpha == 1.0 || (alpha >= 1.05 && alpha <= 3.0), "splash_attention: alpha must be 1 (softmax) or in [1.05, 3]");
    const Tensor tab = index(block_table, Q, {B, -1}, "block_table"), len = index(lengths, Q, {B}, "lengths");
    Tensor list;
    int keep = 0;
    if (pages.has_value() && pages->defined()) {
        list = index(*pages, Q, {B, T, H, -1}, "pages");
        keep = int_of(list.size(3), "pages");
        TORCH_CHECK_VALUE(keep > 0, "splash_attention: pages must list at least one page");
    }
    c10::cuda::CUDAGuard guard(Q.device());
    const Strided q(Q);
    asa_cache_params p = params(B, T, HQ, H, d, P, pool.size(0), tab.size(1));
    p.sm_scale = (float)sm_scale;
    p.alpha = (float)alpha;
    Tensor O = at::empty({B, T, HQ, d}, Q.options());
    size_t bytes = 0;
    check(asa_cache_workspace_bytes(&p, keep, &bytes, nullptr), "asa_cache_workspace_bytes");
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, Q.options().dtype(at::kByte));
    check(asa_cache_attention(&p, q.t.data_ptr(), q.s, pool.data_ptr(), ints(tab), ints(len), ints(list), keep,
                              O.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes, stream_of(Q)),
          "asa_cache_attention");
    return O;
}

// Writing, above the kernels: the cache's version counters count it, as autograd and
// compilers expect of an operator that changes its arguments.
void write_counted(c10::DispatchKeySet keys, const Tensor& K, const Tensor& V, const Tensor& pool, const Tensor& bounds,
                   const Tensor& block_table, const Tensor& start, const OptTensor& count) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("splash_attention::cache_write", "")
                               .typed<void(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                           const Tensor&, const OptTensor&)>();
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        op.redispatch(keys & c10::after_ADInplaceOrView_keyset, K, V, pool, bounds, block_table, start, count);
    }
    for (const Tensor* t : {&pool, &bounds})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void write_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                const OptTensor&) {}

std::tuple<Tensor, Tensor> read_meta(const Tensor& pool, const Tensor& bounds, const Tensor&, const Tensor& start,
                                     int64_t T, const OptTensor&, bool out_f32) {
    const int64_t d = head_dim_of(bounds);
    const auto opt = pool.options().dtype(out_f32 ? at::kFloat : at::kBFloat16);
    return {at::empty({start.size(0), T, pool.size(1), d}, opt), at::empty({start.size(0), T, pool.size(1), d}, opt)};
}

std::tuple<Tensor, Tensor> bounds_meta(const Tensor& bounds, const Tensor& pages) {
    const auto opt = bounds.options().dtype(at::kFloat);
    const int64_t d = (bounds.size(2) - ASA_CACHE_BOUNDS_PAD) / 2;
    return {at::empty({pages.size(0), bounds.size(1), d}, opt), at::empty({pages.size(0), bounds.size(1), d}, opt)};
}

Tensor select_meta(const Tensor& Q, const Tensor&, const Tensor& bounds, const Tensor&, const Tensor&, int64_t keep) {
    return at::empty({Q.size(0), Q.size(1), bounds.size(1), keep}, Q.options().dtype(at::kInt));
}

Tensor attention_meta(const Tensor& Q, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                      double, double) {
    return at::empty(Q.sizes(), Q.options());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(splash_attention, m) {
    m.def("cache_write(Tensor K, Tensor V, Tensor(a!) pool, Tensor(b!) bounds, Tensor block_table, Tensor start, "
          "Tensor? count) -> ()");
    m.def("cache_read(Tensor pool, Tensor bounds, Tensor block_table, Tensor start, int T, Tensor? count, bool out_f32) "
          "-> (Tensor, Tensor)");
    m.def("cache_bounds(Tensor bounds, Tensor pages) -> (Tensor, Tensor)");
    m.def("cache_select(Tensor Q, Tensor pool, Tensor bounds, Tensor block_table, Tensor lengths, int keep) -> Tensor");
    m.def("cache_attention(Tensor Q, Tensor pool, Tensor bounds, Tensor block_table, Tensor lengths, Tensor? pages, "
          "float sm_scale, float alpha) -> Tensor");
}

TORCH_LIBRARY_IMPL(splash_attention, CUDA, m) {
    m.impl("cache_write", &write_cuda);
    m.impl("cache_read", &read_cuda);
    m.impl("cache_bounds", &bounds_cuda);
    m.impl("cache_select", &select_cuda);
    m.impl("cache_attention", &attention_cuda);
}

TORCH_LIBRARY_IMPL(splash_attention, Meta, m) {
    m.impl("cache_write", &write_meta);
    m.impl("cache_read", &read_meta);
    m.impl("cache_bounds", &bounds_meta);
    m.impl("cache_select", &select_meta);
    m.impl("cache_attention", &attention_meta);
}

// A cache is read by inference: its operators pass autograd by (outputs carry no
// gradient), which also spares a call the boxed fallback for operators without one.
TORCH_LIBRARY_IMPL(splash_attention, Autograd, m) {
    for (const char* name : {"cache_write", "cache_read", "cache_bounds", "cache_select", "cache_attention"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}
TORCH_LIBRARY_IMPL(splash_attention, ADInplaceOrView, m) {
    m.impl("cache_write", TORCH_FN(write_counted));
    for (const char* name : {"cache_read", "cache_bounds", "cache_select", "cache_attention"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}
