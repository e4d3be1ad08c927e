// Rotary positions and the append of K and V to a paged cache, in one pass over the q|k|v call's output.
//
//   (a, b) -> (a c - b s, a s + b c),  c + i s = factor * exp(2 pi i frac(pos * turns_i))
//   stored = saturate(round(x / scale)) at the token's place in its page
//
// The angle is kept in turns and in 64 bits until its whole turns are taken off: pos * turns is then off by
// less than 2^-53 * 2^31 turns, where 32 bits would lose every digit of the fast pairs at far positions.
// sincospi runs in 64 bits and is rounded once, so cos and sin are the fp32 numbers nearest to the true ones
// (but for ties that 64 bits cannot tell apart); the rotation is three correctly rounded fp32
// operations without contraction, so what lands in a cache of few bits does not hang on the
// compiler's choice.  One block turns one token's cos and sin once for all the heads that it handles.
#include "kv.cuh"
#include "launch.h"

namespace b200q {

__device__ int g_append_status = 0;

constexpr int kRopeThreads = 256;
constexpr int kMaxRot = 128;

__global__ void rope_table_kernel(const __grid_constant__ b200q_rope r, double * __restrict__ table) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int half = r.n_rot / 2, i = threadIdx.x;
    const double two_pi = 6.283185307179586476925286766559;
    if (i < half) {
        double theta = exp2(-2.0 * i / r.n_rot * log2((double)r.base));
        if (r.freq_factors) {
            theta /= (double)r.freq_factors[i];
        }
        double keep = 0.0;
        if (r.ext_factor != 0.0f) {
            const double den = 2.0 * log((double)r.base);
            const double lo = fmax(0.0, floor(r.n_rot * log(r.n_ctx_orig / (two_pi * r.beta_fast)) / den));
            const double hi = fmin(r.n_rot - 1.0, ceil(r.n_rot * log(r.n_ctx_orig / (two_pi * r.beta_slow)) / den));
            keep = r.ext_factor * (1.0 - fmin(1.0, fmax(0.0, (i - lo) / fmax(0.001, hi - lo))));
        }
        table[i] = theta * ((double)r.freq_scale * (1.0 - keep) + keep) / two_pi;
    }
    if (i == 0) {
        table[half] = (double)r.attn_factor * (r.ext_factor != 0.0f ? 1.0 + 0.1 * log(1.0 / (double)r.freq_scale) : 1.0);
    }
}

struct AppendArgs {
    const double * table;
    const float * q, * k, * v;
    float * q_out;
    int q_stride, k_stride, v_stride, q_out_stride;
    int n_head, n_kv, head_dim, n_rot, interleaved;
    int heads_per_block; // of the n_head + 2 n_kv heads of a token
    KvDev kv;
    BatchDev b;
};

// VEC = 4: a thread handles pairs four at a time (half layout: two float4 loads half a rotation apart; interleaved:
// one float4 holds two pairs); VEC = 1: any alignment and any even n_rot.
template <int T, int VEC> __global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    __shared__ int s_seq;
    asm volatile("griddepcontrol.launch_dependents;");
    const int t = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) {
        s_seq = -1;
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // the sequence that owns row t: every thread looks at its share of the ranges, all loads at once
    for (int s = tid; s < a.b.n_seq; s += kRopeThreads) {
        if (a.b.q_start[s] <= t && t < a.b.q_start[s + 1]) {
            s_seq = s;
        }
    }
    __syncthreads();
    const int seq = s_seq;
    if (seq < 0) {
        return; // behind the last sequence
    }
    const SeqRows r = seq_rows(a.b, a.kv.page_shift, seq);
    const int i = t - r.row0;
    const int pos = r.n - r.n_row + i;
    if (i < 0 || i >= r.n_run || pos < 0) {
        return;
    }
    if (a.table && tid < a.n_rot / 2) {
        const double turns = (double)pos * a.table[tid];
        double s, c;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        const double f = a.table[a.n_rot / 2];
        cs[tid] = make_float2((float)(c * f), (float)(s * f));
    }
    int page = -1;
    if (a.k) {
        page = a.b.page_table[(size_t)seq * a.b.table_stride + (pos >> a.kv.page_shift)];
        if (page < 0 || page >= a.kv.n_pages) {
            page = -1;
            if (tid == 0 && blockIdx.y == 0) {
                atomicExch(&g_append_status, B200Q_EINVAL);
            }
        }
    }
    __syncthreads();
    const int D = a.head_dim, per = D / VEC / (VEC == 4 ? 1 : 2); // work items of a head
    const int rot = a.table ? a.n_rot : 0;
    const int n_q = a.q ? a.n_head : 0, n_all = n_q + (a.k ? 2 * a.n_kv : 0);
    const int h0 = blockIdx.y * a.heads_per_block, h1 = min(h0 + a.heads_per_block, n_all);
    const int in_page = pos & ((1 << a.kv.page_shift) - 1);
    for (int w = h0 * per + tid; w < h1 * per; w += kRopeThreads) {
        const int h = w / per, e = w - h * per;
        const bool is_q = h < n_q, is_v = h >= n_q + a.n_kv;
        const int kh = is_q ? 0 : (is_v ? h - n_q - a.n_kv : h - n_q);
        if (!is_q && page < 0) {
            continue;
        }
        const float * x = is_q ? a.q + (size_t)t * a.q_stride + (size_t)h * D
                               : (is_v ? a.v + (size_t)t * a.v_stride : a.k + (size_t)t * a.k_stride) + (size_t)kh * D;
        const int turned = is_v ? 0 : rot;
        float * y = a.q_out + (size_t)t * a.q_out_stride + (size_t)h * D;
        uint8_t * z = nullptr;
        float inv = 1.0f;
        if (!is_q) {
            z = (is_v ? a.kv.v : a.kv.k) + (size_t)page * a.kv.page_bytes +
                (((size_t)kh << a.kv.page_shift) + in_page) * D * KvElem<T>::BYTES;
            inv = is_v ? a.kv.v_scale : a.kv.k_scale;
        }
        if constexpr (VEC == 4) {
            // the item's eight values as two runs of four: (d0.., d1..)
            int d0, d1, c0;
            const int half = turned / 2;
            float4 u, v;
            if (a.interleaved || 4 * e >= turned) { // four neighbouring values, alone
                d0 = 4 * e;
                u = *reinterpret_cast<const float4 *>(x + d0);
                if (d0 < turned) {
                    c0 = d0 / 2;
                    const float2 A = cs[c0], B = cs[c0 + 1];
                    u = make_float4(__fsub_rn(__fmul_rn(u.x, A.x), __fmul_rn(u.y, A.y)),
                                    __fadd_rn(__fmul_rn(u.x, A.y), __fmul_rn(u.y, A.x)),
                                    __fsub_rn(__fmul_rn(u.z, B.x), __fmul_rn(u.w, B.y)),
                                    __fadd_rn(__fmul_rn(u.z, B.y), __fmul_rn(u.w, B.x)));
                }
                if (is_q) {
                    *reinterpret_cast<float4 *>(y + d0) = u;
                } else {
                    const uint32_t lo = KvElem<T>::pack2(__fdiv_rn(u.x, inv), __fdiv_rn(u.y, inv));
                    const uint32_t hi = KvElem<T>::pack2(__fdiv_rn(u.z, inv), __fdiv_rn(u.w, inv));
                    if constexpr (T == kE4M3) {
                        *reinterpret_cast<uint32_t *>(z + d0) = lo | hi << 16;
                    } else {
                        *reinterpret_cast<uint2 *>(z + d0 * 2) = make_uint2(lo, hi);
                    }
                }
                continue;
            }
            // half layout: items of the first half do both halves, those of the second nothing
            d0 = 4 * e;
            if (d0 >= half) {
                continue;
            }
            d1 = d0 + half;
            u = *reinterpret_cast<const float4 *>(x + d0);
            v = *reinterpret_cast<const float4 *>(x + d1);
            const float uu[4] = {u.x, u.y, u.z, u.w}, vv[4] = {v.x, v.y, v.z, v.w};
            float ra[4], rb[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 A = cs[d0 + j];
                ra[j] = __fsub_rn(__fmul_rn(uu[j], A.x), __fmul_rn(vv[j], A.y));
                rb[j] = __fadd_rn(__fmul_rn(uu[j], A.y), __fmul_rn(vv[j], A.x));
            }
            if (is_q) {
                *reinterpret_cast<float4 *>(y + d0) = make_float4(ra[0], ra[1], ra[2], ra[3]);
                *reinterpret_cast<float4 *>(y + d1) = make_float4(rb[0], rb[1], rb[2], rb[3]);
            } else {
                uint32_t p[4];
                p[0] = KvElem<T>::pack2(__fdiv_rn(ra[0], inv), __fdiv_rn(ra[1], inv));
                p[1] = KvElem<T>::pack2(__fdiv_rn(ra[2], inv), __fdiv_rn(ra[3], inv));
                p[2] = KvElem<T>::pack2(__fdiv_rn(rb[0], inv), __fdiv_rn(rb[1], inv));
                p[3] = KvElem<T>::pack2(__fdiv_rn(rb[2], inv), __fdiv_rn(rb[3], inv));
                if constexpr (T == kE4M3) {
                    *reinterpret_cast<uint32_t *>(z + d0) = p[0] | p[1] << 16;
                    *reinterpret_cast<uint32_t *>(z + d1) = p[2] | p[3] << 16;
                } else {
                    *reinterpret_cast<uint2 *>(z + d0 * 2) = make_uint2(p[0], p[1]);
                    *reinterpret_cast<uint2 *>(z + d1 * 2) = make_uint2(p[2], p[3]);
                }
            }
        } else {
            // one pair an item: rotated pairs first, then neighbours of the part that is not rotated
            const int half = turned / 2;
            const int d0 = e < half ? (a.interleaved ? 2 * e : e) : 2 * e;
            const int d1 = e < half && !a.interleaved ? e + half : d0 + 1;
            float u = x[d0], v = x[d1];
            if (e < half) {
                const float2 A = cs[e];
                const float ra = __fsub_rn(__fmul_rn(u, A.x), __fmul_rn(v, A.y));
                v = __fadd_rn(__fmul_rn(u, A.y), __fmul_rn(v, A.x));
                u = ra;
            }
            if (is_q) {
                y[d0] = u;
                y[d1] = v;
            } else {
                const uint32_t p = KvElem<T>::pack2(__fdiv_rn(u, inv), __fdiv_rn(v, inv));
                if constexpr (T == kE4M3) {
                    z[d0] = (uint8_t)p;
                    z[d1] = (uint8_t)(p >> 8);
                } else {
                    reinterpret_cast<uint16_t *>(z)[d0] = (uint16_t)p;
                    reinterpret_cast<uint16_t *>(z)[d1] = (uint16_t)(p >> 16);
                }
            }
        }
    }
}

template <int T> static cudaError_t launch_append_t(cudaStream_t s, AppendArgs & a, bool vec) {
    const int heads = (a.q ? a.n_head : 0) + (a.k ? 2 * a.n_kv : 0);
    // few rows: a token's heads over several blocks, so that the SMs share the work; many rows: one block a
    // token, which forms the angles once
    int per = heads;
    while (per > 8 && (long long)a.b.n_tok * ((heads + per - 1) / per) < 4 * kSMs) {
        per = (per + 1) / 2;
    }
    a.heads_per_block = per;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.b.n_tok, (unsigned)((heads + per - 1) / per));
    cfg.blockDim = dim3(kRopeThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return vec ? cudaLaunchKernelEx(&cfg, rope_append_kernel<T, 4>, a) : cudaLaunchKernelEx(&cfg, rope_append_kernel<T, 1>, a);
}

cudaError_t launch_rope_append(cudaStream_t s, const double * table, int n_rot, int interleaved, const float * q,
                               int q_stride, int n_head, const float * k, int k_stride, const float * v, int v_stride,
                               float * q_out, int q_out_stride, const KvDev & kv, const BatchDev & b) {
    AppendArgs a = {};
    a.table = table;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out_stride = q_out_stride;
    a.n_head = n_head;
    a.n_kv = kv.n_kv;
    a.head_dim = kv.head_dim;
    a.n_rot = n_rot;
    a.interleaved = interleaved;
    a.kv = kv;
    a.b = b;
    auto ok = [](const void * p, int stride) { return !p || (!((uintptr_t)p & 15) && !(stride & 3)); };
    const bool vec = ok(q, q_stride) && ok(k, k_stride) && ok(v, v_stride) && ok(q_out, q_out_stride) &&
                     (!table || n_rot % (interleaved ? 4 : 8) == 0);
    switch (kv.type) {
    case kF16: return launch_append_t<kF16>(s, a, vec);
    case kBF16: return launch_append_t<kBF16>(s, a, vec);
    default: return launch_append_t<kE4M3>(s, a, vec);
    }
}

cudaError_t launch_rope_table(cudaStream_t s, const b200q_rope & r, double * table) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(kMaxRot / 2);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rope_table_kernel, r, table);
}

cudaError_t read_append_status(int * status, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_append_status, sizeof(int));
    if (e == cudaSuccess && clear && *status != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_append_status, &zero, sizeof(int));
    }
    return e;
}

} // namespace b200q
