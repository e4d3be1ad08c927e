// Attention of a few new tokens per sequence over the paged cache.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp2(c q_r . k_j - m_r),  c = scale log2(e), m_r the largest exponent
//
// One pass over the visible keys with a running maximum and sum.  What bounds it is the one read of K and V
// from HBM, so everything else is arranged around keeping that stream deep and even:
//
// * Units.  A unit is (sequence, KV head, block of query rows); its rows are the new tokens' query heads that share the
//   KV head, so that K and V are read once for all of them.  The units' key tiles in order form one list,
//   and the CTAs take equal contiguous shares of it, whatever the lengths: a long sequence is split
//   over many CTAs, short ones are several to a CTA.  Lengths are read on the device.
// * Streams.  Each warp takes every fourth tile of the CTA's share of a unit and owns a ring of three 8 KB
//   stages that it fills by itself with 16-byte asynchronous copies: no block barrier inside the stream, and the ring runs
//   on over the units' borders, so that the next unit's keys travel while the last one is joined.
// * Products on mma.sync m16n8k16: with at most 16 query rows the tensor work is a few per cent of the time that the
//   tile's bytes take, and a 128-row tcgen05 tile would be empty.  fp32 accuracy at 16-bit operands: q and p are
//   split into two 16-bit parts, x = hi + lo.  Up to eight rows, the sixteen rows of the one product are the
//   eight hi and the eight lo rows, and the two halves of the accumulators are added; more rows take two products.
//   bf16 caches: 16 bits of q and p (off by at most 2^-18 of the value); fp16 and e4m3 caches (e4m3 becomes fp16 exactly):
//   22 bits, with q scaled per row by a power of two to the top of fp16's range and p by 2^14, so that small parts do
//   not fall below fp16's smallest step.
// * Join.  The four warps' (m, l, o) are joined in shared memory in a fixed order; where a unit spans CTAs, each
//   leaves its part in the scratch and the CTA that finishes last joins the parts in order, so results do not depend
//   on who that is.
#include "async.cuh"
#include "attn.cuh"

namespace b200q {

__device__ int g_attn_status = 0;

constexpr int kDecWarps = 4;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecStages = 3;
constexpr int kDecStageBytes = 8192; // K and V halves of one tile
constexpr int kDecPerSM = 2;

// 16-byte chunk `c` of row `r` in a tile of ROWB-byte rows.  16-bit rows are read by ldmatrix (eight rows of one
// chunk column): chunk ^ row.  8-bit rows are read as fragments, for K four chunks of two neighbouring rows, for V
// two chunks of every second row, both without bank conflicts.
template <int T, int ROWB> __device__ __forceinline__ uint32_t tile_off(int r, int c) {
    if constexpr (T != kE4M3) {
        return (uint32_t)(r * ROWB + ((c ^ (r & 7)) << 4));
    } else if constexpr (ROWB == 128) {
        return (uint32_t)(r * 128 + ((c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2))) << 4));
    } else {
        const int line = r >> 1;
        return (uint32_t)(line * 128 + (((((r & 1) << 2) + c) ^ ((line & 3) << 1)) << 4));
    }
}

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t (&v)[4]) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void lds64(uint32_t a, uint32_t & x, uint32_t & y) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x), "=r"(y) : "r"(a) : "memory");
}
// copies 16 bytes, or fills with zeros where `take` is false
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void * src, bool take) {
    const int n = take ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (T == kBF16) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// The unit that a CTA works on, and its share of the unit's tiles.
struct Segment {
    int s, h, rb;        // sequence, KV head, row block
    int t_begin, t_end;  // tiles of the unit's list
    int t_unit;          // tiles of the whole unit
};

struct SeqTiles {
    SeqRows r;
    KeyTiles k;
    int blocks; // row blocks with rows
};
template <int KT, int ROWS> __device__ __forceinline__ SeqTiles seq_tiles(const AttnDev & a, int s) {
    SeqTiles q;
    q.r = seq_rows(a.b, a.kv.page_shift, s);
    q.k = key_tiles(q.r, KT, a.window, a.n_sink);
    q.blocks = (q.r.n_run * a.group + ROWS - 1) / ROWS;
    return q;
}

// H8: at most eight rows a unit, hi and lo parts side by side in one product; otherwise sixteen rows, two products.
template <int T, int D, bool H8> __global__ void __launch_bounds__(kDecThreads, kDecPerSM) attn_decode_kernel(const __grid_constant__ AttnDev a) {
    constexpr int EB = KvElem<T>::BYTES, ROWB = D * EB, KT = kDecStageBytes / 2 / ROWB;
    constexpr int ROWS = H8 ? 8 : 16, KS = D / 16, NT = D / 8;
    constexpr int CPR = ROWB / 16;             // 16-byte chunks of a row
    constexpr int RPI = 32 / CPR;              // rows that one copy instruction of the warp covers
    constexpr int OV = H8 ? 2 : 4;             // o values of a thread per 8 columns
    constexpr float kPBias = T == kBF16 ? 0.0f : 14.0f;
    constexpr int PART = (NT * OV + 1) * 32;   // floats of a part: o, then (m, l) of the up to sixteen rows
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_sum[kDecWarps], s_before;
    __shared__ int s_seq, s_last;
    __shared__ int2 s_meta[kDecWarps][kDecStages];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * kDecStages * kDecStageBytes;
    float * join = reinterpret_cast<float *>(smem + kDecWarps * kDecStages * kDecStageBytes); // two parts

    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- the CTA's share [c0, c1) of the list of all units' tiles
    auto block_sum = [&](long long v, long long & before) { // inclusive over threads; returns the block's sum
        long long x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long y = __shfl_up_sync(~0u, x, d);
            x += lane >= d ? y : 0;
        }
        __syncthreads();
        if (lane == 31) {
            s_sum[warp] = x;
        }
        __syncthreads();
        long long all = 0, mine = 0;
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) {
            mine += w < warp ? s_sum[w] : 0;
            all += s_sum[w];
        }
        before = mine + x - v;
        return all;
    };
    auto seq_total = [&](int s) -> long long {
        if (s >= a.b.n_seq) {
            return 0;
        }
        const SeqTiles q = seq_tiles<KT, ROWS>(a, s);
        return (long long)q.blocks * q.k.count * a.kv.n_kv;
    };
    long long total = 0, before;
    for (int s0 = 0; s0 < a.b.n_seq; s0 += kDecThreads) {
        total += block_sum(seq_total(s0 + tid), before);
    }
    if (total == 0) {
        return;
    }
    const long long want = (total + a.min_tiles - 1) / a.min_tiles;
    const long long nw = want < gridDim.x ? want : gridDim.x;
    if (blockIdx.x >= nw) {
        return;
    }
    const long long c0 = blockIdx.x * total / nw, c1 = (blockIdx.x + 1) * total / nw;
    {
        long long run = 0;
        for (int s0 = 0; s0 < a.b.n_seq; s0 += kDecThreads) {
            const long long v = seq_total(s0 + tid);
            const long long all = block_sum(v, before);
            if (v > 0 && c0 >= run + before && c0 < run + before + v) {
                s_seq = s0 + tid;
                s_before = run + before;
            }
            run += all;
            if (run > c0) {
                break;
            }
        }
        __syncthreads();
    }
    // the first unit
    Segment first;
    {
        first.s = s_seq;
        const SeqTiles q = seq_tiles<KT, ROWS>(a, first.s);
        long long at = c0 - s_before;
        const int u = (int)(at / q.k.count);
        first.h = u / q.blocks;
        first.rb = u % q.blocks;
        first.t_unit = q.k.count;
        first.t_begin = (int)(at - (long long)u * q.k.count);
        const long long left = c1 - c0, here = q.k.count - first.t_begin;
        first.t_end = first.t_begin + (int)(left < here ? left : here);
    }
    // the next unit after `g`, `left` tiles of the share still to come (> 0)
    auto advance = [&](Segment & x, long long left, SeqTiles & q) {
        if (++x.rb == q.blocks) {
            x.rb = 0;
            if (++x.h == a.kv.n_kv) {
                x.h = 0;
                do {
                    x.s++;
                    q = seq_tiles<KT, ROWS>(a, x.s);
                } while (q.blocks == 0 && x.s + 1 < a.b.n_seq);
            }
        }
        x.t_unit = q.k.count;
        x.t_begin = 0;
        x.t_end = (int)(left < q.k.count ? left : q.k.count);
    };

    // ---- the warp's stream: issue() copies the warp's next tile into a stage and says whether there was one
    Segment ps = first;
    SeqTiles pq = seq_tiles<KT, ROWS>(a, ps.s);
    long long p_left = c1 - c0; // tiles from the start of ps on
    int p_tile = ps.t_begin + warp;
    int n_issued = 0;
    auto issue = [&]() {
        while (p_tile >= ps.t_end) {
            p_left -= ps.t_end - ps.t_begin;
            if (p_left <= 0) {
                cp_async_commit();
                return;
            }
            advance(ps, p_left, pq);
            p_tile = ps.t_begin + warp;
        }
        const int stage = n_issued % kDecStages;
        const int tile = key_tile(pq.k, p_tile);
        const int key0 = tile * KT;
        // pages of the tile's groups of 16 keys, one a lane
        constexpr int GROUPS = KT / 16;
        int page = -1;
        bool bad = false;
        if (lane < GROUPS) {
            const int k0 = key0 + lane * 16;
            // a group none of whose keys any row sees needs no page
            if (k0 < pq.r.n && (k0 + 15 >= pq.k.oldest || k0 < a.n_sink)) {
                page = a.b.page_table[(size_t)ps.s * a.b.table_stride + (k0 >> a.kv.page_shift)];
                if (page < 0 || page >= a.kv.n_pages) {
                    page = -1;
                    bad = true;
                }
            }
        }
        if (bad) {
            atomicExch(&g_attn_status, B200Q_EINVAL);
        }
        const uint32_t valid = __ballot_sync(~0u, page >= 0);
        if (lane == 0) {
            s_meta[warp][stage] = make_int2(tile, (int)valid);
        }
        const uint32_t dk = ring + stage * kDecStageBytes, dv = dk + kDecStageBytes / 2;
        const int c = lane % CPR, r0 = lane / CPR;
#pragma unroll
        for (int i = 0; i < KT / RPI; i++) {
            const int r = i * RPI + r0, key = key0 + r;
            const int pg = __shfl_sync(~0u, page, (i * RPI) / 16);
            const bool take = pg >= 0 && key < pq.r.n && (key >= pq.k.oldest || key < a.n_sink);
            const size_t off = (size_t)max(pg, 0) * a.kv.page_bytes +
                               (((size_t)ps.h << a.kv.page_shift) + (key & ((1 << a.kv.page_shift) - 1))) * ROWB + c * 16;
            const uint32_t so = tile_off<T, ROWB>(r, c);
            cp_async16_or_zero(dk + so, a.kv.k + off, take);
            cp_async16_or_zero(dv + so, a.kv.v + off, take);
        }
        cp_async_commit();
        n_issued++;
        p_tile += kDecWarps;
    };
#pragma unroll
    for (int i = 0; i < kDecStages - 1; i++) {
        issue();
    }

    // ---- the units, one after the other
    Segment sg = first;
    SeqTiles sq = seq_tiles<KT, ROWS>(a, sg.s);
    long long left = c1 - c0, at = c0;
    int done = 0;
    for (;;) {
        // rows: a thread holds row g, and with sixteen rows row g + 8 too
        int row_tok[2], row_head[2], pos[2];
        bool live[2];
        const int n_rows = sq.r.n_run * a.group;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int r = sg.rb * ROWS + g + 8 * x;
            live[x] = (x == 0 || !H8) && r < n_rows;
            const int i = live[x] ? r / a.group : 0;
            row_tok[x] = sq.r.row0 + i;
            row_head[x] = sg.h * a.group + (live[x] ? r - i * a.group : 0);
            pos[x] = live[x] ? sq.r.n - sq.r.n_row + i : -1;
        }
        // q as fragments: qa[k step][0] (H8: hi rows above lo rows; else the hi parts), [1] the lo parts
        uint32_t qa[KS][H8 ? 1 : 2][4];
        float cq[2] = {a.scale_log2, a.scale_log2};
        {
            float qv[KS][2][4]; // [k step][row][slots 2t, 2t+1, 2t+8, 2t+9]
#pragma unroll
            for (int x = 0; x < (H8 ? 1 : 2); x++) {
                const float * q = a.q + (size_t)row_tok[x] * a.q_stride + (size_t)row_head[x] * D;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    // the values that the k step's slots of this thread stand for: see the K fragments below
                    const int d0 = T == kE4M3 ? (ks / 4) * 64 + t4 * 16 + (ks % 4) * 4 : ks * 16 + 2 * t4;
                    const int d1 = T == kE4M3 ? d0 + 2 : d0 + 8;
                    qv[ks][x][0] = live[x] ? __ldg(q + d0) : 0.0f;
                    qv[ks][x][1] = live[x] ? __ldg(q + d0 + 1) : 0.0f;
                    qv[ks][x][2] = live[x] ? __ldg(q + d1) : 0.0f;
                    qv[ks][x][3] = live[x] ? __ldg(q + d1 + 1) : 0.0f;
                }
            }
            if constexpr (T != kBF16) {
#pragma unroll
                for (int x = 0; x < (H8 ? 1 : 2); x++) {
                    float top = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            top = fmaxf(top, fabsf(qv[ks][x][j]));
                        }
                    }
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                    const int e = pow2_to_top(top);
                    const float up = exp2_int(e);
                    cq[x] *= exp2_int(-e);
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            qv[ks][x][j] *= up;
                        }
                    }
                }
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if constexpr (H8) {
                    split2<T>(qv[ks][0][0], qv[ks][0][1], qa[ks][0][0], qa[ks][0][1]);
                    split2<T>(qv[ks][0][2], qv[ks][0][3], qa[ks][0][2], qa[ks][0][3]);
                } else {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        split2<T>(qv[ks][x][0], qv[ks][x][1], qa[ks][0][x], qa[ks][1][x]);
                        split2<T>(qv[ks][x][2], qv[ks][x][3], qa[ks][0][2 + x], qa[ks][1][2 + x]);
                    }
                }
            }
        }
        float o[NT][4];
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NT; j++) {
            o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        }
        const int pos_first = sq.r.n - sq.r.n_row, pos_last = pos_first + sq.r.n_run - 1;

        for (int i = sg.t_begin + warp; i < sg.t_end; i += kDecWarps) {
            issue();
            cp_async_wait<kDecStages - 1>();
            __syncwarp();
            const int stage = done % kDecStages;
            done++;
            const int2 meta = s_meta[warp][stage];
            const int key0 = meta.x * KT;
            const uint32_t sk = ring + stage * kDecStageBytes, sv = sk + kDecStageBytes / 2;
            // ---- s = q . k
            float sc[KT / 8][4];
#pragma unroll
            for (int n = 0; n < KT / 8; n++) {
                sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
                if constexpr (T != kE4M3) {
#pragma unroll
                    for (int ks = 0; ks < KS; ks += 2) {
                        uint32_t kb[4];
                        ldsm4(sk + tile_off<T, ROWB>(n * 8 + (lane & 7), ks * 2 + (lane >> 3)), kb);
#pragma unroll
                        for (int y = 0; y < (H8 ? 1 : 2); y++) {
                            mma16816<T>(sc[n], qa[ks][y], kb[0], kb[1]);
                            mma16816<T>(sc[n], qa[ks + 1][y], kb[2], kb[3]);
                        }
                    }
                } else {
                    // 16 values of key g: words 0..3 are the slots of four k steps
#pragma unroll
                    for (int c = 0; c < D / 64; c++) {
                        uint32_t kb[4];
                        lds128(sk + tile_off<T, ROWB>(n * 8 + g, c * 4 + t4), kb);
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const uint32_t b0 = e4m3x2_to_f16x2(kb[w]), b1 = e4m3x2_to_f16x2(kb[w] >> 16);
#pragma unroll
                            for (int y = 0; y < (H8 ? 1 : 2); y++) {
                                mma16816<T>(sc[n], qa[c * 4 + w][y], b0, b1);
                            }
                        }
                    }
                }
            }
            // ---- masks, running maximum
            if constexpr (H8) { // hi row + lo row
#pragma unroll
                for (int n = 0; n < KT / 8; n++) {
                    sc[n][0] += sc[n][2];
                    sc[n][1] += sc[n][3];
                }
            }
            constexpr uint32_t kAll = (KT / 16 >= 32) ? ~0u : (1u << (KT / 16)) - 1u;
            const bool whole = (uint32_t)meta.y == kAll && key0 + KT - 1 <= pos_first &&
                               (a.window == 0 || key0 > pos_last - a.window || key0 + KT <= a.n_sink);
#pragma unroll
            for (int x = 0; x < (H8 ? 1 : 2); x++) {
                float top = -INFINITY;
                const int low = a.window ? pos[x] - a.window + 1 : 0;
#pragma unroll
                for (int n = 0; n < KT / 8; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float v = sc[n][2 * x + e] * cq[x];
                        if (!whole) {
                            const int key = key0 + n * 8 + 2 * t4 + e;
                            const bool seen = key <= pos[x] && (key >= low || key < a.n_sink) && ((meta.y >> (n / 2)) & 1);
                            v = seen ? v : -INFINITY;
                        }
                        sc[n][2 * x + e] = v;
                        top = fmaxf(top, v);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const float mn = fmaxf(m[x], top);
                if (__any_sync(~0u, mn > m[x])) {
                    const float f = mn > m[x] ? exp2f(m[x] - mn) : 1.0f; // m = -inf: 0
                    l[x] *= f;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        if constexpr (H8) {
                            o[j][0] *= f, o[j][1] *= f, o[j][2] *= f, o[j][3] *= f;
                        } else {
                            o[j][2 * x] *= f, o[j][2 * x + 1] *= f;
                        }
                    }
                    m[x] = mn;
                }
                const float base = (m[x] == -INFINITY ? 0.0f : m[x]) - kPBias;
#pragma unroll
                for (int n = 0; n < KT / 8; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float p = exp2_fast(sc[n][2 * x + e] - base);
                        sc[n][2 * x + e] = p;
                        l[x] += p;
                    }
                }
            }
            // ---- o += p v
#pragma unroll
            for (int kk = 0; kk < KT / 16; kk++) {
                uint32_t pa[H8 ? 1 : 2][4];
                if constexpr (H8) {
                    split2<T>(sc[2 * kk][0], sc[2 * kk][1], pa[0][0], pa[0][1]);
                    split2<T>(sc[2 * kk + 1][0], sc[2 * kk + 1][1], pa[0][2], pa[0][3]);
                } else {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        split2<T>(sc[2 * kk][2 * x], sc[2 * kk][2 * x + 1], pa[0][x], pa[1][x]);
                        split2<T>(sc[2 * kk + 1][2 * x], sc[2 * kk + 1][2 * x + 1], pa[0][2 + x], pa[1][2 + x]);
                    }
                }
                if constexpr (T != kE4M3) {
#pragma unroll
                    for (int j = 0; j < NT; j += 2) {
                        uint32_t vb[4];
                        ldsm4t(sv + tile_off<T, ROWB>(kk * 16 + (lane & 15), j + (lane >> 4)), vb);
#pragma unroll
                        for (int y = 0; y < (H8 ? 1 : 2); y++) {
                            mma16816<T>(o[j], pa[y], vb[0], vb[1]);
                            mma16816<T>(o[j + 1], pa[y], vb[2], vb[3]);
                        }
                    }
                } else {
                    // keys 2t, 2t+1, 2t+8, 2t+9, NT values each from value NT g on: column g of o[j] is value NT g + j
                    uint32_t w[4][NT / 4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const int r = kk * 16 + 2 * t4 + (y & 1) + (y >> 1) * 8;
                        if constexpr (D == 128) {
                            lds128(sv + tile_off<T, ROWB>(r, g), w[y]);
                        } else {
                            lds64(sv + tile_off<T, ROWB>(r, g >> 1) + (g & 1) * 8, w[y][0], w[y][1]);
                        }
                    }
#pragma unroll
                    for (int q4 = 0; q4 < NT / 4; q4++) {
                        const uint32_t b0l = __byte_perm(w[0][q4], w[1][q4], 0x5140), b0h = __byte_perm(w[0][q4], w[1][q4], 0x7362);
                        const uint32_t b1l = __byte_perm(w[2][q4], w[3][q4], 0x5140), b1h = __byte_perm(w[2][q4], w[3][q4], 0x7362);
                        const uint32_t b0[4] = {e4m3x2_to_f16x2(b0l), e4m3x2_to_f16x2(b0l >> 16), e4m3x2_to_f16x2(b0h), e4m3x2_to_f16x2(b0h >> 16)};
                        const uint32_t b1[4] = {e4m3x2_to_f16x2(b1l), e4m3x2_to_f16x2(b1l >> 16), e4m3x2_to_f16x2(b1h), e4m3x2_to_f16x2(b1h >> 16)};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
#pragma unroll
                            for (int y = 0; y < (H8 ? 1 : 2); y++) {
                                mma16816<T>(o[q4 * 4 + e], pa[y], b0[e], b1[e]);
                            }
                        }
                    }
                }
            }
            __syncwarp(); // the stage may be filled again
        }

        // ---- join: v[] are the thread's o values, (m, l) of its rows
        float v[NT * OV];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            if constexpr (H8) {
                v[2 * j] = o[j][0] + o[j][2];
                v[2 * j + 1] = o[j][1] + o[j][3];
            } else {
                v[4 * j] = o[j][0], v[4 * j + 1] = o[j][1], v[4 * j + 2] = o[j][2], v[4 * j + 3] = o[j][3];
            }
        }
#pragma unroll
        for (int x = 0; x < 2; x++) {
            l[x] += __shfl_xor_sync(~0u, l[x], 1);
            l[x] += __shfl_xor_sync(~0u, l[x], 2);
        }
        auto put = [&](float * p) {
#pragma unroll
            for (int j = 0; j < NT * OV; j++) {
                p[j * 32 + lane] = v[j];
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                p[NT * OV * 32 + x * 16 + g] = m[x]; // the same from all four threads of the row
                p[NT * OV * 32 + x * 16 + 8 + g] = l[x];
            }
        };
        auto take = [&](const float * p) { // joins another part to the thread's
            float f[2], h[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const float m2 = p[NT * OV * 32 + x * 16 + g], l2 = p[NT * OV * 32 + x * 16 + 8 + g];
                const float mn = fmaxf(m[x], m2);
                f[x] = m[x] == mn ? 1.0f : exp2f(m[x] - mn);
                h[x] = m2 == mn ? 1.0f : exp2f(m2 - mn);
                m[x] = mn;
                l[x] = l[x] * f[x] + l2 * h[x];
            }
#pragma unroll
            for (int j = 0; j < NT * OV; j++) {
                const int x = H8 ? 0 : (j >> 1) & 1;
                v[j] = v[j] * f[x] + p[j * 32 + lane] * h[x];
            }
        };
        auto join_warps = [&]() { // warp 0 ends with all
            __syncthreads();
            if (warp >= 2) {
                put(join + (warp - 2) * PART);
            }
            __syncthreads();
            if (warp < 2) {
                take(join + warp * PART);
            }
            __syncthreads();
            if (warp == 1) {
                put(join);
            }
            __syncthreads();
            if (warp == 0) {
                take(join);
            }
        };
        join_warps();
        bool write = true;
        if (sg.t_end - sg.t_begin != sg.t_unit) {
            // the unit spans CTAs: its tiles are [u0, u0 + t_unit) of the list
            const long long u0 = at - sg.t_begin;
            auto owner = [&](long long x) { return (int)(((x + 1) * nw - 1) / total); };
            const int b0 = owner(u0), b1 = owner(u0 + sg.t_unit - 1);
            // of a CTA's two slots the second holds the unit that starts in its share and runs on behind it
            if (warp == 0) {
                put(a.parts + ((size_t)blockIdx.x * 2 + (sg.t_begin == 0 ? 1 : 0)) * PART);
                __threadfence();
                __syncwarp();
                if (lane == 0) {
                    const int unit = (sg.s * a.kv.n_kv + sg.h) * a.row_blocks + sg.rb;
                    const uint32_t was = atomicAdd(a.counters + unit, 1u);
                    s_last = was == (uint32_t)(b1 - b0);
                    if (s_last) {
                        a.counters[unit] = 0; // as the next call wants it
                        __threadfence();
                    }
                }
            }
            __syncthreads();
            write = s_last;
            if (write) {
                m[0] = m[1] = -INFINITY;
                l[0] = l[1] = 0.0f;
#pragma unroll
                for (int j = 0; j < NT * OV; j++) {
                    v[j] = 0.0f;
                }
                for (int b = b0 + warp; b <= b1; b += kDecWarps) {
                    take(a.parts + ((size_t)b * 2 + (b == b0 ? 1 : 0)) * PART);
                }
                join_warps();
            }
        }
        if (write && warp == 0) {
#pragma unroll
            for (int x = 0; x < (H8 ? 1 : 2); x++) {
                if (live[x]) {
                    const float f = l[x] > 0.0f || isnan(l[x]) ? a.v_scale / l[x] : 0.0f; // no visible key: zeros
                    float * out = a.out + (size_t)row_tok[x] * a.out_stride + (size_t)row_head[x] * D;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int d = T == kE4M3 ? NT * (2 * t4 + e) + j : j * 8 + 2 * t4 + e;
                            out[d] = v[OV * j + 2 * x + e] * f;
                        }
                    }
                }
            }
        }
        left -= sg.t_end - sg.t_begin;
        at += sg.t_end - sg.t_begin;
        if (left <= 0) {
            break;
        }
        advance(sg, left, sq);
    }
    cp_async_wait<0>();
}

template <int T, int D, bool H8> static cudaError_t launch_t(cudaStream_t s, const AttnDev & a, int grid) {
    constexpr int PART = (D / 8 * (H8 ? 2 : 4) + 1) * 32;
    constexpr int smem = kDecWarps * kDecStages * kDecStageBytes + 2 * PART * 4;
    const cudaError_t e = ensure_dynamic_smem((const void *)attn_decode_kernel<T, D, H8>, smem);
    if (e != cudaSuccess) {
        return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kDecThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_decode_kernel<T, D, H8>, a);
}

constexpr int kDecGrid = kSMs * kDecPerSM;

static int dec_rows(int group, int max_q) { return group * max_q <= 8 ? 8 : 16; }

size_t attn_decode_units(int n_head, int n_kv, int n_seq, int max_q) {
    const int rows = dec_rows(n_head / n_kv, max_q);
    return (size_t)n_seq * n_kv * (((size_t)max_q * (n_head / n_kv) + rows - 1) / rows);
}
size_t attn_decode_part_bytes(int n_head, int n_kv, int head_dim, int max_q) {
    const int rows = dec_rows(n_head / n_kv, max_q);
    return (size_t)kDecGrid * 2 * ((size_t)head_dim / 8 * (rows == 8 ? 2 : 4) + 1) * 32 * sizeof(float);
}

cudaError_t launch_attn_decode(cudaStream_t s, AttnDev a) {
    const int rows = dec_rows(a.group, a.b.max_q);
    a.row_blocks = (a.b.max_q * a.group + rows - 1) / rows;
    a.min_tiles = kDecWarps;
    auto go = [&](auto t, auto d) -> cudaError_t {
        constexpr int T = decltype(t)::value, D = decltype(d)::value;
        return rows == 8 ? launch_t<T, D, true>(s, a, kDecGrid) : launch_t<T, D, false>(s, a, kDecGrid);
    };
    auto dim = [&](auto t) {
        return a.kv.head_dim == 64 ? go(t, std::integral_constant<int, 64>{}) : go(t, std::integral_constant<int, 128>{});
    };
    switch (a.kv.type) {
    case kF16: return dim(std::integral_constant<int, kF16>{});
    case kBF16: return dim(std::integral_constant<int, kBF16>{});
    default: return dim(std::integral_constant<int, kE4M3>{});
    }
}

cudaError_t read_attn_status(int * status, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_attn_status, sizeof(int));
    if (e == cudaSuccess && clear && *status != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(int));
    }
    return e;
}

} // namespace b200q
