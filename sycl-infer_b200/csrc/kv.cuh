// Paged KV cache and step batch as the kernels see them, and what they share: the rows of a sequence,
// the keys they see, the page of a key, conversion to the cache's element types.
#pragma once
#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200q {

constexpr int kF16 = B200Q_KV_F16, kBF16 = B200Q_KV_BF16, kE4M3 = B200Q_KV_E4M3;

struct KvDev {
    uint8_t * k, * v;
    int64_t page_bytes; // from one page to the next
    int32_t type, n_pages, page_shift, n_kv, head_dim;
    float k_scale, v_scale;
};

struct BatchDev {
    const int32_t * page_table, * q_start, * kv_len;
    int32_t table_stride, n_seq, n_tok, max_q;
};

constexpr int kCopyLayers = 64; // layers of one page-copy launch

// defined beside their kernels
cudaError_t launch_rope_table(cudaStream_t s, const b200q_rope & r, double * table);
cudaError_t launch_rope_append(cudaStream_t s, const double * table, int n_rot, int interleaved, const float * q,
                               int q_stride, int n_head, const float * k, int k_stride, const float * v, int v_stride,
                               float * q_out, int q_out_stride, const KvDev & kv, const BatchDev & b);
cudaError_t launch_kv_copy_pages(cudaStream_t s, const KvDev & c, void * const * pools, int n_pools, const int32_t * src,
                                 const int32_t * dst, int n);
int kv_copy_chunks(const KvDev & c); // blocks that copy one page
cudaError_t launch_kv_remap(cudaStream_t s, const int32_t * table, int table_stride, int n_seq, int width,
                            const int32_t * map, int n_pages, int32_t * out, int out_stride);

__host__ __device__ inline int kv_elem_bytes(uint32_t type) { return type == kE4M3 ? 1 : 2; }

#ifdef __CUDACC__

// Rows and cache length of a sequence, made safe: whatever the caller's arrays hold, rows stay inside
// [0, n_tok) and keys inside the page table.
struct SeqRows {
    int row0;  // first row
    int n_row; // rows the sequence owns
    int n_run; // rows that are computed (at most max_q)
    int n;     // keys in the cache, the new ones included; at most 2^30
};
__device__ __forceinline__ SeqRows seq_rows(const BatchDev & b, int page_shift, int s) {
    SeqRows r;
    const int a = b.q_start[s], e = b.q_start[s + 1], n = b.kv_len[s];
    r.row0 = min(max(a, 0), b.n_tok);
    const int end = min(max(e, r.row0), b.n_tok);
    r.n_row = end - r.row0;
    r.n_run = min(r.n_row, b.max_q);
    const long long cap = min((long long)b.table_stride << page_shift, 1LL << 30); // tile arithmetic stays in 32 bits
    r.n = (int)min((long long)max(n, 0), cap);
    return r;
}

// A page id outside the pool: the rest of the call is right.  Never in place of a wait that ran out, after which nothing is.
__device__ __forceinline__ void note_bad_page(int * status) { atomicCAS(status, 0, B200Q_EINVAL); }

template <int T> struct KvElem;
template <> struct KvElem<kF16> {
    static constexpr int BYTES = 2;
    // round to nearest even; finite values beyond the range become the largest finite one, as do infinities
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        a = isnan(a) ? a : fminf(fmaxf(a, -65504.0f), 65504.0f);
        b = isnan(b) ? b : fminf(fmaxf(b, -65504.0f), 65504.0f);
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <> struct KvElem<kBF16> {
    static constexpr int BYTES = 2;
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const float top = 3.3895313892515355e38f;
        a = isnan(a) ? a : fminf(fmaxf(a, -top), top);
        b = isnan(b) ? b : fminf(fmaxf(b, -top), top);
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <> struct KvElem<kE4M3> {
    static constexpr int BYTES = 1;
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { // 16 bits used
        return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    }
};

#endif

} // namespace b200q
