// Page copies of a paged KV cache (fork, compaction) and the page tables' new numbers.
#include "kv.cuh"
#include "launch.h"

namespace b200q {

__device__ int g_pages_status = 0;
static std::atomic<bool> g_launched{false}; // nothing to read before

constexpr int kCopyThreads = 256;

struct CopyArgs {
    uint8_t * pool[2 * kCopyLayers]; // k, v of each layer
    const int32_t * src, * dst;
    int64_t page_bytes;
    int64_t bytes; // of a page that hold values, a multiple of 16
    int32_t n_pages, chunks;
};

// One block copies one chunk of one page: every load of the block is issued before its first store.  Bound by HBM: 301
// pages of 64 tokens x 24 layers, 1.9 GB read and written, 289 us = 6.54 TB/s, the rate of a plain copy.
constexpr int kCopyUnroll = 4;
constexpr int kCopyChunk = kCopyThreads * 16 * kCopyUnroll;
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int chunk = blockIdx.x % a.chunks, i = blockIdx.x / a.chunks;
    const int s = a.src[i], d = a.dst[i];
    if (s < 0 || s >= a.n_pages || d < 0 || d >= a.n_pages) {
        if (threadIdx.x == 0) {
            note_bad_page(&g_pages_status);
        }
        return;
    }
    uint8_t * pool = a.pool[blockIdx.y];
    const uint4 * from = reinterpret_cast<const uint4 *>(pool + (size_t)s * a.page_bytes);
    uint4 * to = reinterpret_cast<uint4 *>(pool + (size_t)d * a.page_bytes);
    const int64_t n16 = a.bytes / 16, at = (int64_t)chunk * (kCopyChunk / 16) + threadIdx.x;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; j++) {
        if (at + j * kCopyThreads < n16) {
            v[j] = __ldcs(from + at + j * kCopyThreads);
        }
    }
#pragma unroll
    for (int j = 0; j < kCopyUnroll; j++) {
        if (at + j * kCopyThreads < n16) {
            __stcs(to + at + j * kCopyThreads, v[j]);
        }
    }
}

__global__ void __launch_bounds__(256) remap_kernel(const int32_t * table, int table_stride, int width,
                                                    const int32_t * __restrict__ map, int n_pages, int32_t * out,
                                                    int out_stride) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < width) {
        const int32_t p = table[(size_t)blockIdx.y * table_stride + i];
        out[(size_t)blockIdx.y * out_stride + i] = p >= 0 && p < n_pages ? map[p] : p;
    }
}

static cudaLaunchConfig_t chained(cudaStream_t s, dim3 grid, int threads, cudaLaunchAttribute * attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

static int64_t page_value_bytes(const KvDev & c) { return (int64_t)c.n_kv * c.head_dim * kv_elem_bytes(c.type) << c.page_shift; }
int kv_copy_chunks(const KvDev & c) { return (int)((page_value_bytes(c) + kCopyChunk - 1) / kCopyChunk); }

cudaError_t launch_kv_copy_pages(cudaStream_t s, const KvDev & c, void * const * pools, int n_pools, const int32_t * src,
                                 const int32_t * dst, int n) {
    g_launched = true;
    CopyArgs a = {};
    for (int i = 0; i < n_pools; i++) {
        a.pool[i] = static_cast<uint8_t *>(pools[i]);
    }
    a.src = src;
    a.dst = dst;
    a.page_bytes = c.page_bytes;
    a.bytes = page_value_bytes(c);
    a.n_pages = c.n_pages;
    a.chunks = kv_copy_chunks(c);
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = chained(s, dim3((unsigned)n * a.chunks, (unsigned)n_pools), kCopyThreads, attr);
    return cudaLaunchKernelEx(&cfg, copy_pages_kernel, a);
}

cudaError_t launch_kv_remap(cudaStream_t s, const int32_t * table, int table_stride, int n_seq, int width,
                            const int32_t * map, int n_pages, int32_t * out, int out_stride) {
    for (int s0 = 0; s0 < n_seq; s0 += 65535) { // grid y holds 65535 rows
        const int m = n_seq - s0 < 65535 ? n_seq - s0 : 65535;
        cudaLaunchAttribute attr[1];
        const cudaLaunchConfig_t cfg = chained(s, dim3((unsigned)((width + 255) / 256), (unsigned)m), 256, attr);
        const cudaError_t e = cudaLaunchKernelEx(&cfg, remap_kernel, table + (size_t)s0 * table_stride, table_stride, width,
                                                 map, n_pages, out + (size_t)s0 * out_stride, out_stride);
        if (e != cudaSuccess) {
            return e;
        }
    }
    return cudaSuccess;
}

cudaError_t read_pages_status(int * status, bool clear) {
    if (!g_launched) {
        *status = 0;
        return cudaSuccess;
    }
    cudaError_t e = cudaMemcpyFromSymbol(status, g_pages_status, sizeof(int));
    if (e == cudaSuccess && clear && *status != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_pages_status, &zero, sizeof(int));
    }
    return e;
}

} // namespace b200q
