// asa_cache.h -- launch-side declarations of the 4-bit paged key/value cache's
// kernels (asa_cache_*.cu), and the layout both sides share.  Not part of the
// public ABI; include/asa.h describes the formats.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/asa.h"

namespace asa {

void note_launch(int n = 1);
int* cache_error_word();               // asa_capi.cu
int cuda_status_of(cudaError_t e);
void* profile_open(const char* label, cudaStream_t st);
void profile_close(void* scope);

namespace cache {

constexpr int kBlock = 16;       // tokens of a block: the unit a record is laid out in
constexpr int kGroup = 32;       // channels that share a scale and an offset
constexpr float kF16Max = 65504.0f;
// The formats multiply by the nearest fp32 numbers to 1/15 and 1/127.
constexpr float kFifteenth = 1.0f / 15.0f;
constexpr float k127th = 1.0f / 127.0f;

// One call's sizes, checked on the host.
struct Shape {
    int B, T, HQ, H, G, d, P;        // G = HQ / H query heads a key head; P tokens a page
    int pages, width;                // the pool's pages; entries of a block table row
    int dtype;
    float scale, alpha;
    int naps;                        // bound on device-side waits, in naps of 20 us at most
    int64_t rec;                     // bytes of one page's record of one key head
};

__host__ __device__ constexpr int row_bytes(int d) { return d / 2; }
__host__ __device__ constexpr int par_bytes(int d) { return d / 8; }             // 2 * d/32 fp16
__host__ __device__ constexpr int block_bytes(int d) { return kBlock * (row_bytes(d) + par_bytes(d)); }
__host__ __device__ constexpr int64_t record_bytes(int d, int P) { return 2ll * (P / kBlock) * block_bytes(d); }
__host__ __device__ constexpr int bounds_bytes(int d) { return 2 * d + ASA_CACHE_BOUNDS_PAD; }

struct Strides { int64_t b, t, h; };

// The cache's kernels follow one another closely (a step is four to six of them), so
// each may be set up on the SMs while the one before it drains: a kernel first waits
// for the memory of all before it, then lets the next be set up.
#ifdef __CUDACC__
__device__ __forceinline__ void follow() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// Allows a kernel `bytes` of dynamic shared memory, once a device (`done`: the kernel's own).
struct Allowed { std::atomic<unsigned long long> devices{0}; };
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, Allowed& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.devices.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.devices.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
template <typename... P, typename... A>
cudaError_t launch_clusters(int cluster, void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st,
                            A&&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(block);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = cluster > 1 ? 2 : 1;
    note_launch();
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, A&&... args) {
    return launch_clusters(1, kernel, grid, block, smem, st, args...);
}
#endif

cudaError_t write(const Shape& s, const void* K, const void* V, Strides ks, Strides vs, uint8_t* pool,
                  int8_t* bounds, const int32_t* table, const int32_t* start, const int32_t* count,
                  int* err, cudaStream_t st);
cudaError_t read(const Shape& s, const uint8_t* pool, const int32_t* table, const int32_t* start,
                 const int32_t* count, void* K, void* V, int* err, cudaStream_t st);
cudaError_t read_bounds(const Shape& s, const int8_t* bounds, const int32_t* pages, int n, float* upper,
                        float* lower, int* err, cudaStream_t st);

size_t select_workspace(const Shape& s);
cudaError_t select(const Shape& s, const void* Q, Strides qs, const int8_t* bounds, const int32_t* table,
                   const int32_t* lengths, int keep, int32_t* pages, void* ws, int* err, cudaStream_t st);

cudaError_t wait_probe(int naps, int* err, cudaStream_t st);

size_t attend_workspace(const Shape& s, int keep);
cudaError_t attend(const Shape& s, const void* Q, Strides qs, const uint8_t* pool, const int32_t* table,
                   const int32_t* lengths, const int32_t* list, int keep, void* O, void* ws, int* err,
                   cudaStream_t st);

}  // namespace cache
}  // namespace asa
