// What the attention kernels share: arguments, the keys that a sequence's rows see, 16-bit splitting.
#pragma once
#include <type_traits>

#include "kv.cuh"
#include "launch.h"

namespace b200q {

struct AttnDev {
    const float * q;
    float * out;
    int32_t q_stride, out_stride, n_head, group; // group: query heads of a KV head
    KvDev kv;
    BatchDev b;
    float scale_log2; // softmax scale x log2(e) x k_scale
    float v_scale;
    int32_t window, n_sink;
    float * parts;       // scratch: what CTAs leave of units that they share
    uint32_t * counters; // scratch: arrivals at a unit that workers share, by the worker that has its start; zero between calls
    int32_t vec;         // rows of q and out can be read and written 16 bytes at a time
};

// More query rows of a (sequence, KV head) than this take the prompt kernel (attn_prompt.cu).
constexpr int kDecodeRows = 16;
constexpr int kMaxSeqs = 4096; // of one step

// The scratch begins with this many counters, whatever the call: calls of different shapes may use one scratch in turn,
// and no call's parts ever lie where another keeps its counters.
constexpr int kAttnCounters = 2048;

cudaError_t launch_attn_prompt(cudaStream_t s, AttnDev a);
size_t attn_prompt_part_bytes(int head_dim);
cudaError_t read_attn_prompt_status(int * status, bool clear);
cudaError_t launch_attn_decode(cudaStream_t s, const AttnDev & a);
size_t attn_decode_part_bytes(int n_head, int n_kv, int head_dim, int n_seq, int max_q);

#ifdef __CUDACC__

// Tiles of `kt` keys that some of a unit's rows see, whose first row is at position pos_first and whose last key is n - 1:
// those of the first n_sink keys, then those from the oldest key in any row's window to the newest.  At least one,
// so that rows that see nothing are still written.
struct KeyTiles {
    int n;          // keys 0 .. n-1 exist for the unit
    int oldest;     // oldest key in any row's window
    int sink_tiles; // tiles of the list that belong to the sinks alone
    int t_lo;       // tile of `oldest`
    int count;
};
__device__ __forceinline__ KeyTiles key_tiles(int pos_first, int n, int kt, int window, int n_sink) {
    KeyTiles k;
    k.n = n;
    k.oldest = window ? max(0, pos_first - window + 1) : 0;
    k.oldest = min(k.oldest, n);
    k.t_lo = k.oldest / kt;
    k.sink_tiles = min((min(n_sink, n) + kt - 1) / kt, k.t_lo);
    k.count = max(1, k.sink_tiles + (n + kt - 1) / kt - k.t_lo);
    return k;
}
// Which of the 16 keys from k0 on some row sees, as bits.
__device__ __forceinline__ uint32_t keys_seen(const KeyTiles & k, int k0, int n_sink) {
    if (k0 >= k.n) {
        return 0;
    }
    uint32_t seen = k0 + 16 <= k.n ? 0xFFFFu : 0xFFFFu >> (k0 + 16 - k.n);
    if (k0 < k.oldest) {
        uint32_t keep = k.oldest - k0 >= 16 ? 0u : 0xFFFFu << (k.oldest - k0);
        keep |= n_sink - k0 >= 16 ? 0xFFFFu : (n_sink > k0 ? 0xFFFFu >> (16 - (n_sink - k0)) : 0u);
        seen &= keep;
    }
    return seen;
}
__device__ __forceinline__ int key_tile(const KeyTiles & k, int i) { return i < k.sink_tiles ? i : i - k.sink_tiles + k.t_lo; }

__device__ __forceinline__ float exp2_fast(float x) { // 2 ulp, 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The power of two that brings `top` into [2^14, 2^15), kept within fp32's exponents; 0 for zero, infinity and NaN.
__device__ __forceinline__ int pow2_to_top(float top) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255u);
    return e == 0 || e == 255 ? 0 : min(14 - (e - 127), 100);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); } // -126..127

// (x, y) as a sum of N pairs of 16-bit numbers, the largest first
template <int T, int N> __device__ __forceinline__ void split_pair(float x, float y, uint32_t (&part)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (T == kBF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
            part[i] = *reinterpret_cast<const uint32_t *>(&h);
            x -= __uint_as_float(part[i] << 16);
            y -= __uint_as_float(part[i] & 0xFFFF0000u);
        } else {
            const __half2 h = __floats2half2_rn(x, y);
            part[i] = *reinterpret_cast<const uint32_t *>(&h);
            const float2 f = __half22float2(h);
            x -= f.x;
            y -= f.y;
        }
    }
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) { // the low 16 bits; exact
    uint32_t r;
    asm("{.reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t;}" : "=r"(r) : "r"(v));
    return r;
}

#endif

} // namespace b200q
