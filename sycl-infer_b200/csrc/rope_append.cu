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
//
// B200: one token 2.5 us on the device (a launch and three dependent loads); 2048 tokens of 40 + 8 heads of 128, 109 MB,
// 23.1 us = 4.7 TB/s: what is left is the blocks' own chain (row, sequence, page, angle), which ten blocks an SM hide in part.
#include "kv.cuh"
#include "launch.h"

namespace b200q {

__device__ int g_append_status = 0;
static std::atomic<bool> g_launched{false}; // nothing to read before

constexpr int kRopeThreads = 128;
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

// What a block reads first of its inputs, then of the batch: which row it is does not depend on the sequence that owns
// it, so the rows travel while the sequence, the page and the angles are found.
//
// VEC = 4: an item is eight values of a head as two float4: in the rotated part four pairs (half layout: the second float4
// lies half a rotation behind the first; interleaved: next to it), behind it, and in v, eight neighbours.  VEC = 1: an item is
// one pair, for any alignment and any even n_rot.
// Many small blocks hide each other's chain best.  2048 tokens / 900 in 48 chunks: 256 threads with two items each in flight
// 24.1 / 11.0 us, 128 threads with two 23.1 / 10.3, with one (ten blocks an SM) 23.1 / 9.1.
constexpr int kRopeBatch = 1; // items of a thread in flight

template <int T, int VEC> struct RopeItem {
    float u[VEC], v[VEC]; // values d0.. and d1..
    int d0, d1, pair;     // pair: first rotated pair, or -1
    bool is_q, is_v;
    int h;
};

template <int T, int VEC> __global__ void __launch_bounds__(kRopeThreads, 10) rope_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    __shared__ int s_seq;
    asm volatile("griddepcontrol.launch_dependents;");
    const int t = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) {
        s_seq = -1;
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int D = a.head_dim, per = D / (2 * VEC); // items of a head
    const int rot = a.table ? a.n_rot : 0;
    const int n_q = a.q ? a.n_head : 0, n_all = n_q + (a.k ? 2 * a.n_kv : 0);
    const int w0 = blockIdx.y * a.heads_per_block * per, w1 = min((blockIdx.y + 1) * a.heads_per_block, n_all) * per;
    auto read = [&](int w, RopeItem<T, VEC> & x) {
        const int h = w / per, e = w - h * per;
        x.is_q = h < n_q;
        x.is_v = h >= n_q + a.n_kv;
        x.h = x.is_q ? h : (x.is_v ? h - n_q - a.n_kv : h - n_q);
        const int turned = x.is_v ? 0 : rot, half = turned / 2;
        x.pair = VEC * e < half ? VEC * e : -1;
        if (x.pair >= 0 && !a.interleaved) {
            x.d0 = VEC * e;
            x.d1 = x.d0 + half;
        } else {
            x.d0 = 2 * VEC * e;
            x.d1 = x.d0 + VEC;
        }
        const float * p = (x.is_q ? a.q + (size_t)t * a.q_stride : (x.is_v ? a.v + (size_t)t * a.v_stride : a.k + (size_t)t * a.k_stride)) + (size_t)x.h * D;
        if constexpr (VEC == 4) {
            const float4 u = *reinterpret_cast<const float4 *>(p + x.d0), v = *reinterpret_cast<const float4 *>(p + x.d1);
            x.u[0] = u.x, x.u[1] = u.y, x.u[2] = u.z, x.u[3] = u.w;
            x.v[0] = v.x, x.v[1] = v.y, x.v[2] = v.z, x.v[3] = v.w;
        } else {
            x.u[0] = p[x.d0];
            x.v[0] = p[x.d1];
        }
    };
    RopeItem<T, VEC> item[kRopeBatch];
    auto read_batch = [&](int w) {
#pragma unroll
        for (int i = 0; i < kRopeBatch; i++) {
            if (w + i * kRopeThreads < w1) {
                read(w + i * kRopeThreads, item[i]);
            }
        }
    };
    read_batch(w0 + tid);
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
    const int i_tok = t - r.row0;
    const int pos = r.n - r.n_row + i_tok;
    if (i_tok < 0 || i_tok >= r.n_run || pos < 0) {
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
                note_bad_page(&g_append_status);
            }
        }
    }
    __syncthreads();
    const int in_page = pos & ((1 << a.kv.page_shift) - 1);
    auto finish = [&](RopeItem<T, VEC> & x) {
        if (x.pair >= 0) {
            auto turn = [](float & p, float & q, const float2 c) {
                const float rp = __fsub_rn(__fmul_rn(p, c.x), __fmul_rn(q, c.y));
                q = __fadd_rn(__fmul_rn(p, c.y), __fmul_rn(q, c.x));
                p = rp;
            };
            if (VEC == 1 || !a.interleaved) {
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    turn(x.u[j], x.v[j], cs[x.pair + j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    turn(x.u[j], x.u[(j + 1) % VEC], cs[x.pair + j / 2]);
                    turn(x.v[j], x.v[(j + 1) % VEC], cs[x.pair + VEC / 2 + j / 2]);
                }
            }
        }
        if (x.is_q) {
            float * y = a.q_out + (size_t)t * a.q_out_stride + (size_t)x.h * D;
            if constexpr (VEC == 4) {
                *reinterpret_cast<float4 *>(y + x.d0) = make_float4(x.u[0], x.u[1], x.u[2], x.u[3]);
                *reinterpret_cast<float4 *>(y + x.d1) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
            } else {
                y[x.d0] = x.u[0];
                y[x.d1] = x.v[0];
            }
            return;
        }
        if (page < 0) {
            return;
        }
        const float scale = x.is_v ? a.kv.v_scale : a.kv.k_scale;
        uint8_t * z = (x.is_v ? a.kv.v : a.kv.k) + (size_t)page * a.kv.page_bytes +
                      (((size_t)x.h << a.kv.page_shift) + in_page) * D * KvElem<T>::BYTES;
        auto pack = [&](float p, float q) { return KvElem<T>::pack2(__fdiv_rn(p, scale), __fdiv_rn(q, scale)); };
        if constexpr (VEC == 4) {
            const uint32_t p0 = pack(x.u[0], x.u[1]), p1 = pack(x.u[2], x.u[3]), p2 = pack(x.v[0], x.v[1]), p3 = pack(x.v[2], x.v[3]);
            if constexpr (T == kE4M3) {
                *reinterpret_cast<uint32_t *>(z + x.d0) = p0 | p1 << 16;
                *reinterpret_cast<uint32_t *>(z + x.d1) = p2 | p3 << 16;
            } else {
                *reinterpret_cast<uint2 *>(z + x.d0 * 2) = make_uint2(p0, p1);
                *reinterpret_cast<uint2 *>(z + x.d1 * 2) = make_uint2(p2, p3);
            }
        } else {
            const uint32_t p = pack(x.u[0], x.v[0]);
            if constexpr (T == kE4M3) {
                z[x.d0] = (uint8_t)p;
                z[x.d1] = (uint8_t)(p >> 8);
            } else {
                reinterpret_cast<uint16_t *>(z)[x.d0] = (uint16_t)p;
                reinterpret_cast<uint16_t *>(z)[x.d1] = (uint16_t)(p >> 16);
            }
        }
    };
    for (int w = w0 + tid; w < w1; w += kRopeBatch * kRopeThreads) {
        if (w != w0 + tid) {
            read_batch(w);
        }
#pragma unroll
        for (int i = 0; i < kRopeBatch; i++) {
            if (w + i * kRopeThreads < w1) {
                finish(item[i]);
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
    g_launched = true;
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
                     (!table || n_rot % 8 == 0);
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
    if (!g_launched) {
        *status = 0;
        return cudaSuccess;
    }
    cudaError_t e = cudaMemcpyFromSymbol(status, g_append_status, sizeof(int));
    if (e == cudaSuccess && clear && *status != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_append_status, &zero, sizeof(int));
    }
    return e;
}

} // namespace b200q
