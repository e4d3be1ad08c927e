// Attention of a few new tokens per sequence over the paged cache.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp2(c q_r . k_j - m_r),  c = scale log2(e), m_r the largest exponent
//
// One pass over the visible keys with a running maximum and sum.  What bounds it is the one read of K and V
// from HBM, so everything else is arranged around keeping that stream deep and even:
//
// * Units.  A unit is (sequence, KV head, block of query rows); its rows are the new tokens' query heads that share the
//   KV head, so that K and V are read once for all of them.  The units' key tiles in order form one list that is
//   cut over the SMs whatever the lengths, which are read on the device: a long sequence is split over many, short ones
//   share one.
// * Streams.  Each warp owns a ring of 8 KB stages that it fills by itself with 16-byte asynchronous copies: no block
//   barrier inside the stream, and with shares of several units the ring runs on over their borders, so that the next
//   unit's keys travel while the last one is finished.
// * Teams.  With many units every warp is a worker with an equal share of the list (TEAM 1).  With few, each CTA takes one
//   piece of one unit, its eight warps every eighth tile, and joins in shared memory (TEAM 8): a unit is left in few parts and
//   nobody works through two joins (1 x 517 keys: 8.9 us against 12.9 us with equal shares, where a CTA that got the
//   end of one unit and the start of the next finished last).
// * Products on mma.sync m16n8k16: with at most 16 query rows the tensor work hides behind the bytes, and a 128-row
//   tcgen05 tile would be empty.  fp32 accuracy at 16-bit operands: q and p are split into 16-bit parts, two for
//   fp16 and e4m3 caches (e4m3 becomes fp16 exactly; 22 bits, with q scaled per row by a power of two to the top of
//   fp16's range and p by 2^14, so that small parts do not fall below fp16's smallest step), three for bf16 (24 bits).
//   Up to eight rows, the sixteen rows of one product are the eight first and the eight second parts.  The tensor
//   cores' fp32 sums drop bits at every step, always towards zero, so a long chain drifts: each tile's product starts from
//   zero, smallest parts first, and is added to the running o in a rounded fp32 addition (which the rescaling to the new
//   maximum needs anyway).
// * Join.  Where a unit spans workers, each leaves its (m, l, o) in the scratch and the one that finishes last joins the
//   parts in order, so results do not depend on who that is.
//
// B200: 1 x 131071 keys bf16 (537 MB) 93 us, of which the stream takes 72 (7.5 TB/s), the start 4, the spread of the
// CTAs' ends and the last join the rest; 32 x 200..8192 keys f16 (595 MB) 107 us, 5.5 TB/s: the shares are equal, the SMs' rates
// are not (ends from 70 to 99 us); 192 x window 1024 e4m3 62 us: widening 8-bit keys in registers is what it issues.
#include "async.cuh"
#include "attn.cuh"

namespace b200q {

__device__ int g_attn_status = 0;
static std::atomic<bool> g_launched{false}; // nothing to read before

constexpr int kDecStageBytes = 8192; // K and V halves of one tile
constexpr int kDecTeam = 8;          // warps of a CTA that work on one piece
// TEAM 1: four warps a CTA, two CTAs an SM with rings of three stages; eight rows of 64 values leave registers for a third
// CTA, with rings of two (192 x window 1024 keys e4m3: 70 -> 63 us; with 128 values it spills: 73 -> 76 us).
// TEAM 8: one CTA an SM.
__host__ __device__ constexpr int dec_warps(int team) { return team == 1 ? 4 : team; }
__host__ __device__ constexpr int dec_per_sm(int dim, bool h8, int team) { return team > 1 ? 1 : (h8 && dim == 64 ? 3 : 2); }
__host__ __device__ constexpr int dec_stages(int dim, bool h8, int team) { return team == 1 && h8 && dim == 64 ? 2 : 3; }

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
__device__ __forceinline__ void lds64(uint32_t a, uint32_t (&v)[2]) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a) : "memory");
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

// The unit that a worker is at, and its share of the unit's tiles.
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
    q.k = key_tiles(q.r.n - q.r.n_row, q.r.n, KT, a.window, a.n_sink);
    q.blocks = (q.r.n_run * a.group + ROWS - 1) / ROWS;
    return q;
}

// Floats of a part in the scratch or in shared memory: o as the warp's threads hold it, then (m, l) of up to 16 rows.
__host__ __device__ constexpr int part_floats(int dim, bool h8) { return (dim / 8 * (h8 ? 2 : 4) + 1) * 32; }

// H8: at most eight rows a unit, first and second parts side by side in one product; otherwise sixteen rows.
template <int T, int D, bool H8, int TEAM>
__global__ void __launch_bounds__(dec_warps(TEAM) * 32, dec_per_sm(D, H8, TEAM)) attn_decode_kernel(const __grid_constant__ AttnDev a) {
    constexpr int EB = KvElem<T>::BYTES, ROWB = D * EB, KT = kDecStageBytes / 2 / ROWB;
    constexpr int ROWS = H8 ? 8 : 16, KS = D / 16, NT = D / 8;
    constexpr int PARTS = T == kBF16 ? 3 : 2;  // 16-bit parts of q and p
    constexpr int NA = H8 ? PARTS - 1 : PARTS; // A operands: with H8 the first holds two parts
    constexpr int CPR = ROWB / 16;             // 16-byte chunks of a row
    constexpr int RPI = 32 / CPR;              // rows that one copy instruction of the warp covers
    constexpr int GROUPS = KT / 16;            // groups of 16 keys: contiguous in a page
    constexpr int OV = H8 ? 2 : 4;             // o values of a thread per 8 columns
    constexpr int RX = H8 ? 1 : 2;             // rows of a thread
    constexpr float kPBias = T == kBF16 ? 0.0f : 14.0f;
    constexpr int PART = part_floats(D, H8);
    constexpr int WARPS = dec_warps(TEAM), THREADS = WARPS * 32, STAGES = dec_stages(D, H8, TEAM);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_sum[WARPS], s_before[WARPS];
    __shared__ int s_seq[WARPS], s_last;
    __shared__ int2 s_meta[WARPS][STAGES];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * STAGES * kDecStageBytes;
    float * join = reinterpret_cast<float *>(smem + WARPS * STAGES * kDecStageBytes); // TEAM 8: four parts

    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- the worker's share [c0, c1) of the list of all units' tiles
    auto block_sum = [&](long long v, long long & before) { // before: sum over the threads below; returns the block's sum
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
        for (int w = 0; w < WARPS; w++) {
            mine += w < warp ? s_sum[w] : 0;
            all += s_sum[w];
        }
        before = mine + x - v;
        return all;
    };
    // TEAM 8 counts the units along: few, by the rule that chooses it
    constexpr int kUnitBit = 40;
    auto seq_total = [&](int s) -> long long {
        if (s >= a.b.n_seq) {
            return 0;
        }
        const SeqTiles q = seq_tiles<KT, ROWS>(a, s);
        const long long units = (long long)q.blocks * a.kv.n_kv;
        return units * q.k.count + (TEAM > 1 ? units << kUnitBit : 0);
    };
    const long long v_first = seq_total(tid);
    long long before_first, before;
    long long total = block_sum(v_first, before_first);
    const long long sum_first = total;
    for (int s0 = THREADS; s0 < a.b.n_seq; s0 += THREADS) {
        total += block_sum(seq_total(s0 + tid), before);
    }
    if (total == 0) {
        return;
    }
    // TEAM 1: the list is cut into equal shares, one a warp, wherever the cuts fall; worker w's share starts at
    // w * each + min(w, more).  TEAM 8: every unit is cut into pieces of equal length, at most `each` tiles, so that a CTA
    // has one piece of one unit and its way to the end is as short as can be.
    constexpr int WORKERS = WARPS / TEAM; // of a CTA
    long long nw, each, more = 0, v_team = 0, sum_team = 0, before_team = 0;
    auto pieces = [&](const SeqTiles & q) { return (int)((q.k.count + each - 1) / each); };
    auto seq_workers = [&](int s) -> long long { // TEAM 8
        if (s >= a.b.n_seq) {
            return 0;
        }
        const SeqTiles q = seq_tiles<KT, ROWS>(a, s);
        return (long long)q.blocks * a.kv.n_kv * pieces(q);
    };
    if constexpr (TEAM == 1) {
        const long long most = (long long)gridDim.x * WORKERS;
        nw = total < most ? total : most;
        each = total / nw;
        more = total - each * nw;
    } else {
        const long long units = total >> kUnitBit;
        total &= (1LL << kUnitBit) - 1;
        // Pieces of `each` tiles are at most total / each + units in number: no more than CTAs, one for each at most (units
        // are fewer than CTAs: kTeamUnits, one row block each).
        each = (total + gridDim.x - units - 1) / (gridDim.x - units);
        each = each > TEAM ? each : TEAM; // a tile for every warp
        v_team = seq_workers(tid);
        sum_team = nw = block_sum(v_team, before_team);
        for (int s0 = THREADS; s0 < a.b.n_seq; s0 += THREADS) {
            nw += block_sum(seq_workers(s0 + tid), before);
        }
    }
    if ((long long)blockIdx.x * WORKERS >= nw) {
        return;
    }
    auto share = [&](int w) { return w * each + (w < more ? w : more); };
    const int w_first = TEAM == 1 ? 0 : warp; // the warp's first tile of a segment
    const int copy_row = lane / CPR, copy_chunk = lane % CPR;
    const int worker = blockIdx.x * WORKERS + warp / TEAM;
    // ---- where the worker starts
    {
        long long run = 0;
        for (int s0 = 0; s0 < a.b.n_seq; s0 += THREADS) {
            long long v, all;
            if constexpr (TEAM == 1) {
                v = v_first, all = sum_first, before = before_first;
                if (s0 > 0) {
                    v = seq_total(s0 + tid);
                    all = block_sum(v, before);
                }
            } else {
                v = v_team, all = sum_team, before = before_team;
                if (s0 > 0) {
                    v = seq_workers(s0 + tid);
                    all = block_sum(v, before);
                }
            }
            long long c_last = 0;
#pragma unroll
            for (int w = 0; w < WORKERS; w++) {
                const long long c = TEAM == 1 ? share(blockIdx.x * WORKERS + w) : worker;
                if (v > 0 && c >= run + before && c < run + before + v) {
                    s_seq[w] = s0 + tid;
                    s_before[w] = run + before;
                }
                c_last = c;
            }
            run += all;
            if (run > c_last) {
                break;
            }
        }
        __syncthreads();
    }
    if (TEAM == 1 && worker >= nw) {
        return; // no block barrier from here on
    }
    // the first unit
    const long long c0 = TEAM == 1 ? share(worker) : 0, c1 = TEAM == 1 ? share(worker + 1) : 1;
    Segment first;
    int piece = 0, n_pieces = 1; // TEAM 8
    SeqTiles pq;
    {
        first.s = s_seq[warp / TEAM];
        pq = seq_tiles<KT, ROWS>(a, first.s);
        first.t_unit = pq.k.count;
        if constexpr (TEAM == 1) {
            const long long at = c0 - s_before[warp / TEAM];
            const int u = (int)(at / pq.k.count);
            first.h = u / pq.blocks;
            first.rb = u % pq.blocks;
            first.t_begin = (int)(at - (long long)u * pq.k.count);
            const long long left = c1 - c0, here = pq.k.count - first.t_begin;
            first.t_end = first.t_begin + (int)(left < here ? left : here);
        } else {
            n_pieces = pieces(pq);
            const int at = (int)(worker - s_before[0]), u = at / n_pieces;
            piece = at - u * n_pieces;
            first.h = u / pq.blocks;
            first.rb = u % pq.blocks;
            first.t_begin = (int)((long long)piece * pq.k.count / n_pieces);
            first.t_end = (int)((long long)(piece + 1) * pq.k.count / n_pieces);
        }
    }
    // the unit after x, with `left` tiles of the share still to come (> 0)
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

    // ---- the warp's stream: issue() copies the warp's next tile into the next stage
    Segment ps = first;
    const SeqTiles fq = pq;
    long long p_left = c1 - c0; // tiles from the start of ps on
    int p_tile = ps.t_begin + w_first;
    int p_stage = 0;
    auto issue = [&]() {
        while (p_tile >= ps.t_end) {
            p_left -= ps.t_end - ps.t_begin;
            if (TEAM > 1 || p_left <= 0) { // a piece is all that a team has
                cp_async_commit();
                return;
            }
            advance(ps, p_left, pq);
            p_tile = ps.t_begin + w_first;
        }
        const int tile = key_tile(pq.k, p_tile);
        const int key0 = tile * KT;
        // lane i looks after the tile's group i: where its 16 rows lie, which of them some row sees
        unsigned long long src = 0;
        uint32_t seen = 0;
        if (lane < GROUPS) {
            const int k0 = key0 + lane * 16;
            seen = keys_seen(pq.k, k0, a.n_sink);
            if (seen) {
                const int page = a.b.page_table[(size_t)ps.s * a.b.table_stride + (k0 >> a.kv.page_shift)];
                if (page >= 0 && page < a.kv.n_pages) {
                    src = (unsigned long long)page * a.kv.page_bytes +
                          (((unsigned long long)ps.h << a.kv.page_shift) + (k0 & ((1 << a.kv.page_shift) - 1))) * ROWB;
                } else {
                    seen = 0;
                    note_bad_page(&g_attn_status);
                }
            }
        }
        const uint32_t valid = __ballot_sync(~0u, seen != 0), full = __ballot_sync(~0u, seen == 0xFFFFu);
        if (lane == 0) {
            s_meta[warp][p_stage] = make_int2(key0, (int)valid);
        }
        const uint32_t dk = ring + p_stage * kDecStageBytes, dv = dk + kDecStageBytes / 2;
#pragma unroll
        for (int gr = 0; gr < GROUPS; gr++) {
            const unsigned long long off = __shfl_sync(~0u, src, gr) + lane * 16;
            const uint8_t * fk = a.kv.k + off, * fv = a.kv.v + off;
            if ((full >> gr) & 1) {
#pragma unroll
                for (int i = 0; i < 16 / RPI; i++) {
                    const uint32_t so = tile_off<T, ROWB>(gr * 16 + i * RPI + copy_row, copy_chunk);
                    cp_async16(dk + so, fk + i * 512);
                    cp_async16(dv + so, fv + i * 512);
                }
            } else { // rows that nobody sees (their memory may hold anything) become zeros
                const uint32_t rows = __shfl_sync(~0u, seen, gr);
#pragma unroll
                for (int i = 0; i < 16 / RPI; i++) {
                    const uint32_t so = tile_off<T, ROWB>(gr * 16 + i * RPI + copy_row, copy_chunk);
                    const bool take = (rows >> (i * RPI + copy_row)) & 1;
                    cp_async16_or_zero(dk + so, take ? fk + i * 512 : a.kv.k, take);
                    cp_async16_or_zero(dv + so, take ? fv + i * 512 : a.kv.v, take);
                }
            }
        }
        cp_async_commit();
        p_stage = p_stage + 1 == STAGES ? 0 : p_stage + 1;
        p_tile += TEAM;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) {
        issue();
    }

    // ---- the units, one after the other
    Segment sg = first;
    SeqTiles sq = fq;
    long long left = c1 - c0, at = c0;
    int stage = 0;
    for (;;) {
        // rows: a thread holds row g, and with sixteen rows row g + 8 too
        int row_tok[RX], row_head[RX], pos[RX];
        bool live[RX];
        const int n_rows = sq.r.n_run * a.group;
#pragma unroll
        for (int x = 0; x < RX; x++) {
            const int r = sg.rb * ROWS + g + 8 * x;
            live[x] = r < n_rows;
            const int i = live[x] ? r / a.group : 0;
            row_tok[x] = sq.r.row0 + i;
            row_head[x] = sg.h * a.group + (live[x] ? r - i * a.group : 0);
            pos[x] = live[x] ? sq.r.n - sq.r.n_row + i : -1;
        }
        // q as A operands.  H8: qa[.][0] has the first parts in rows 0..7 and the second in 8..15, qa[.][1] the third parts
        // in rows 0..7; otherwise qa[.][y] has part y of the sixteen rows.
        uint32_t qa[KS][NA][4];
        float cq[RX];
        {
            float qv[KS][RX][4]; // [k step][row][slots 2t, 2t+1, 2t+8, 2t+9]
#pragma unroll
            for (int x = 0; x < RX; x++) {
                const float * q = a.q + (size_t)row_tok[x] * a.q_stride + (size_t)row_head[x] * D;
                cq[x] = a.scale_log2;
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
                if constexpr (T != kBF16) {
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
#pragma unroll
                for (int x = 0; x < RX; x++) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint32_t part[PARTS];
                        split_pair<T>(qv[ks][x][2 * half], qv[ks][x][2 * half + 1], part);
                        if constexpr (H8) {
                            qa[ks][0][2 * half] = part[0];
                            qa[ks][0][2 * half + 1] = part[1];
                            if constexpr (PARTS == 3) {
                                qa[ks][NA - 1][2 * half] = part[2];
                                qa[ks][NA - 1][2 * half + 1] = 0;
                            }
                        } else {
#pragma unroll
                            for (int y = 0; y < PARTS; y++) {
                                qa[ks][y][2 * half + x] = part[y];
                            }
                        }
                    }
                }
            }
        }
        float v[NT * OV]; // o: H8 columns 2t, 2t+1 of row g; otherwise the same of row g + 8 behind them
        float m[RX], l[RX];
#pragma unroll
        for (int x = 0; x < RX; x++) {
            m[x] = -INFINITY;
            l[x] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NT * OV; j++) {
            v[j] = 0.0f;
        }
        const int pos_first = sq.r.n - sq.r.n_row, pos_last = pos_first + sq.r.n_run - 1;

        for (int i = sg.t_begin + w_first; i < sg.t_end; i += TEAM) {
            issue();
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            const int2 meta = s_meta[warp][stage];
            const int key0 = meta.x;
            const uint32_t sk = ring + stage * kDecStageBytes, sv = sk + kDecStageBytes / 2;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            // ---- s = q . k, the smallest parts first
            float sc[KT / 8][4];
#pragma unroll
            for (int n = 0; n < KT / 8; n++) {
                sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
                uint32_t kb[KS][2];
                if constexpr (T != kE4M3) {
#pragma unroll
                    for (int ks = 0; ks < KS; ks += 2) {
                        uint32_t w[4];
                        ldsm4(sk + tile_off<T, ROWB>(n * 8 + (lane & 7), ks * 2 + (lane >> 3)), w);
                        kb[ks][0] = w[0], kb[ks][1] = w[1], kb[ks + 1][0] = w[2], kb[ks + 1][1] = w[3];
                    }
                } else {
                    // 16 values of key g: words 0..3 are the slots of four k steps
#pragma unroll
                    for (int c = 0; c < D / 64; c++) {
                        uint32_t w[4];
                        lds128(sk + tile_off<T, ROWB>(n * 8 + g, c * 4 + t4), w);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            kb[c * 4 + e][0] = e4m3x2_to_f16x2(w[e]);
                            kb[c * 4 + e][1] = e4m3x2_to_f16x2(w[e] >> 16);
                        }
                    }
                }
#pragma unroll
                for (int y = NA - 1; y >= 0; y--) {
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        mma16816<T>(sc[n], qa[ks][y], kb[ks][0], kb[ks][1]);
                    }
                }
                if constexpr (H8) { // first part's row + second part's row
                    sc[n][0] += sc[n][2];
                    sc[n][1] += sc[n][3];
                }
            }
            // ---- masks (only tiles on a border), running maximum, p
            constexpr uint32_t kAll = (1u << GROUPS) - 1u;
            const bool whole = (uint32_t)meta.y == kAll && key0 + KT - 1 <= pos_first &&
                               (a.window == 0 || key0 > pos_last - a.window || key0 + KT <= a.n_sink);
            float f[RX];
            if (!whole) {
#pragma unroll
                for (int x = 0; x < RX; x++) {
                    const int low = a.window ? pos[x] - a.window + 1 : 0;
#pragma unroll
                    for (int n = 0; n < KT / 8; n++) {
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int key = key0 + n * 8 + 2 * t4 + e;
                            const bool seen = key <= pos[x] && (key >= low || key < a.n_sink) && ((meta.y >> (n / 2)) & 1);
                            sc[n][2 * x + e] = seen ? sc[n][2 * x + e] : -INFINITY;
                        }
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < RX; x++) {
                float top = fmaxf(sc[0][2 * x], sc[0][2 * x + 1]);
#pragma unroll
                for (int n = 1; n < KT / 8; n++) {
                    top = fmaxf(top, fmaxf(sc[n][2 * x], sc[n][2 * x + 1]));
                }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const float mn = fmaxf(m[x], top * cq[x]);
                f[x] = m[x] == mn ? 1.0f : exp2_fast(m[x] - mn); // nothing seen yet: exp2(-inf) = 0
                m[x] = mn;
                const float base = kPBias - (mn == -INFINITY ? 0.0f : mn);
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < KT / 8; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float p = exp2_fast(fmaf(sc[n][2 * x + e], cq[x], base));
                        sc[n][2 * x + e] = p;
                        sum += p;
                    }
                }
                l[x] = fmaf(l[x], f[x], sum);
            }
            // ---- o = f o + p v, the smallest parts first
            uint32_t pa[GROUPS][NA][4];
#pragma unroll
            for (int kk = 0; kk < GROUPS; kk++) {
#pragma unroll
                for (int x = 0; x < RX; x++) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint32_t part[PARTS];
                        split_pair<T>(sc[2 * kk + half][2 * x], sc[2 * kk + half][2 * x + 1], part);
                        if constexpr (H8) {
                            pa[kk][0][2 * half] = part[0];
                            pa[kk][0][2 * half + 1] = part[1];
                            if constexpr (PARTS == 3) {
                                pa[kk][NA - 1][2 * half] = part[2];
                                pa[kk][NA - 1][2 * half + 1] = 0;
                            }
                        } else {
#pragma unroll
                            for (int y = 0; y < PARTS; y++) {
                                pa[kk][y][2 * half + x] = part[y];
                            }
                        }
                    }
                }
            }
            constexpr int JC = T == kE4M3 ? 4 : 2; // blocks of eight columns that are taken together
            // e4m3: keys 2t, 2t+1, 2t+8, 2t+9, NT values each from value NT g on: column g of block j is value NT g + j
            uint32_t raw[T == kE4M3 ? GROUPS : 1][4][NT / 4];
            if constexpr (T == kE4M3) {
#pragma unroll
                for (int kk = 0; kk < GROUPS; kk++) {
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const int r = kk * 16 + 2 * t4 + (y & 1) + (y >> 1) * 8;
                        if constexpr (D == 128) {
                            lds128(sv + tile_off<T, ROWB>(r, g), raw[kk][y]);
                        } else {
                            lds64(sv + tile_off<T, ROWB>(r, g >> 1) + (g & 1) * 8, raw[kk][y]);
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NT; j += JC) {
                float c[JC][4];
                uint32_t vb[GROUPS][JC][2];
#pragma unroll
                for (int e = 0; e < JC; e++) {
                    c[e][0] = c[e][1] = c[e][2] = c[e][3] = 0.0f;
                }
#pragma unroll
                for (int kk = 0; kk < GROUPS; kk++) {
                    if constexpr (T != kE4M3) {
                        uint32_t w[4];
                        ldsm4t(sv + tile_off<T, ROWB>(kk * 16 + (lane & 15), j + (lane >> 4)), w);
                        vb[kk][0][0] = w[0], vb[kk][0][1] = w[1], vb[kk][1][0] = w[2], vb[kk][1][1] = w[3];
                    } else {
                        const uint32_t w[4] = {raw[kk][0][j / 4], raw[kk][1][j / 4], raw[kk][2][j / 4], raw[kk][3][j / 4]};
                        const uint32_t b0l = __byte_perm(w[0], w[1], 0x5140), b0h = __byte_perm(w[0], w[1], 0x7362);
                        const uint32_t b1l = __byte_perm(w[2], w[3], 0x5140), b1h = __byte_perm(w[2], w[3], 0x7362);
                        vb[kk][0][0] = e4m3x2_to_f16x2(b0l), vb[kk][1 % JC][0] = e4m3x2_to_f16x2(b0l >> 16);
                        vb[kk][2 % JC][0] = e4m3x2_to_f16x2(b0h), vb[kk][3 % JC][0] = e4m3x2_to_f16x2(b0h >> 16);
                        vb[kk][0][1] = e4m3x2_to_f16x2(b1l), vb[kk][1 % JC][1] = e4m3x2_to_f16x2(b1l >> 16);
                        vb[kk][2 % JC][1] = e4m3x2_to_f16x2(b1h), vb[kk][3 % JC][1] = e4m3x2_to_f16x2(b1h >> 16);
                    }
                }
#pragma unroll
                for (int y = NA - 1; y >= 0; y--) {
#pragma unroll
                    for (int kk = 0; kk < GROUPS; kk++) {
#pragma unroll
                        for (int e = 0; e < JC; e++) {
                            mma16816<T>(c[e], pa[kk][y], vb[kk][e][0], vb[kk][e][1]);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < JC; e++) {
                    float * o = v + (j + e) * OV;
                    if constexpr (H8) {
                        o[0] = fmaf(o[0], f[0], c[e][0] + c[e][2]);
                        o[1] = fmaf(o[1], f[0], c[e][1] + c[e][3]);
                    } else {
                        o[0] = fmaf(o[0], f[0], c[e][0]);
                        o[1] = fmaf(o[1], f[0], c[e][1]);
                        o[OV - 2] = fmaf(o[OV - 2], f[RX - 1], c[e][2]);
                        o[OV - 1] = fmaf(o[OV - 1], f[RX - 1], c[e][3]);
                    }
                }
            }
            __syncwarp(); // the stage may be filled again
        }

        // ---- join
#pragma unroll
        for (int x = 0; x < RX; x++) {
            l[x] += __shfl_xor_sync(~0u, l[x], 1);
            l[x] += __shfl_xor_sync(~0u, l[x], 2);
        }
        auto put = [&](float * p) {
#pragma unroll
            for (int j = 0; j < NT * OV; j++) {
                p[j * 32 + lane] = v[j];
            }
#pragma unroll
            for (int x = 0; x < RX; x++) {
                p[NT * OV * 32 + x * 16 + g] = m[x]; // the same from all four threads of the row
                p[NT * OV * 32 + x * 16 + 8 + g] = l[x];
            }
        };
        // Joins another part to the thread's; parts in the scratch are other SMs' and come from L2.
        auto take = [&](const float * p, auto in_scratch) {
            auto value = [&](int i) {
                if constexpr (decltype(in_scratch)::value) {
                    return __ldcg(p + i);
                } else {
                    return p[i];
                }
            };
            float fa[RX], fb[RX];
#pragma unroll
            for (int x = 0; x < RX; x++) {
                const float m2 = value(NT * OV * 32 + x * 16 + g), l2 = value(NT * OV * 32 + x * 16 + 8 + g);
                const float mn = fmaxf(m[x], m2);
                fa[x] = m[x] == mn ? 1.0f : exp2_fast(m[x] - mn);
                fb[x] = m2 == mn ? 1.0f : exp2_fast(m2 - mn);
                m[x] = mn;
                l[x] = l[x] * fa[x] + l2 * fb[x];
            }
#pragma unroll
            for (int j = 0; j < NT * OV; j++) {
                const int x = H8 ? 0 : (j >> 1) & 1;
                v[j] = v[j] * fa[x] + value(j * 32 + lane) * fb[x];
            }
        };
        // The team's first warp ends with all: halves of the team put their parts where the warp that takes them has
        // taken from before, so that one barrier a step is enough.
        auto join_team = [&]() {
            if constexpr (TEAM > 1) {
#pragma unroll
                for (int half = TEAM / 2; half > 0; half >>= 1) {
                    if (warp >= half && warp < 2 * half) {
                        put(join + (2 * half == TEAM ? warp - half : warp) * PART);
                    }
                    __syncthreads();
                    if (warp < half) {
                        take(join + (2 * half == TEAM ? warp : warp + half) * PART, std::false_type{});
                    }
                }
            }
        };
        const bool lead = TEAM == 1 || warp == 0;
        join_team();
        bool write = true;
        if (sg.t_end - sg.t_begin != sg.t_unit) {
            // the unit spans workers
            int b0, b1;
            if constexpr (TEAM == 1) { // its tiles are [u0, u0 + t_unit) of the list
                const long long u0 = at - sg.t_begin;
                auto owner = [&](long long x) { // the worker whose share holds tile x
                    return (int)(x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each);
                };
                b0 = owner(u0), b1 = owner(u0 + sg.t_unit - 1);
            } else {
                b0 = worker - piece, b1 = b0 + n_pieces - 1;
            }
            // of a worker's two slots (TEAM 8: one) the second holds the unit that starts in its share and runs on behind it
            auto slot = [&](int b, bool starts) { return a.parts + (TEAM == 1 ? (size_t)b * 2 + (starts ? 1 : 0) : (size_t)b) * PART; };
            if (lead) {
                put(slot(worker, sg.t_begin == 0));
                __threadfence();
                __syncwarp();
                uint32_t last = 0;
                if (lane == 0) {
                    uint32_t * counter = a.counters + b0; // one unit at most starts in a worker's share and runs on behind it
                    last = atomicAdd(counter, 1u) == (uint32_t)(b1 - b0);
                    if (last) {
                        *counter = 0; // as the next call wants it
                        __threadfence();
                    }
                    if constexpr (TEAM > 1) {
                        s_last = (int)last;
                    }
                }
                write = __shfl_sync(~0u, last, 0);
                __syncwarp(); // what lane 0's fence made visible, for all lanes: the shuffle orders no memory
            }
            if constexpr (TEAM > 1) {
                __syncthreads();
                write = s_last;
            }
            if (write) {
#pragma unroll
                for (int x = 0; x < RX; x++) {
                    m[x] = -INFINITY;
                    l[x] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < NT * OV; j++) {
                    v[j] = 0.0f;
                }
                for (int b = b0 + w_first; b <= b1; b += TEAM) {
                    take(slot(b, b == b0), std::true_type{});
                }
                join_team();
            }
        }
        if (write && lead) {
#pragma unroll
            for (int x = 0; x < RX; x++) {
                if (live[x]) {
                    const float r = l[x] > 0.0f || isnan(l[x]) ? a.v_scale / l[x] : 0.0f; // no visible key: zeros
                    float * out = a.out + (size_t)row_tok[x] * a.out_stride + (size_t)row_head[x] * D;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int d = T == kE4M3 ? NT * (2 * t4 + e) + j : j * 8 + 2 * t4 + e;
                            out[d] = v[OV * j + 2 * x + e] * r;
                        }
                    }
                }
            }
        }
        left -= sg.t_end - sg.t_begin;
        at += sg.t_end - sg.t_begin;
        if (TEAM > 1 || left <= 0) {
            break;
        }
        advance(sg, left, sq);
    }
    cp_async_wait<0>();
}

template <int T, int D, bool H8, int TEAM> static cudaError_t launch_t(cudaStream_t s, const AttnDev & a) {
    constexpr int smem = dec_warps(TEAM) * dec_stages(D, H8, TEAM) * kDecStageBytes + (TEAM > 1 ? TEAM / 2 * part_floats(D, H8) * 4 : 0);
    const cudaError_t e = ensure_dynamic_smem((const void *)attn_decode_kernel<T, D, H8, TEAM>, smem);
    if (e != cudaSuccess) {
        return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(kSMs * dec_per_sm(D, H8, TEAM)));
    cfg.blockDim = dim3(dec_warps(TEAM) * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_decode_kernel<T, D, H8, TEAM>, a);
}

// How a call is cut.  Few units: teams, so that a unit is left in few parts (B200, f16, 128 values, 8 KV heads, up to 8192
// keys: 2, 4, 8 sequences 14, 17, 31 us with teams of eight, 71, 41, 48 us with warps alone; 9 sequences 33 against 47 us, 12
// sequences 59 against 54: the border lies at half as many units as SMs).
// Rows: as many as there are, up to eight or up to sixteen; e4m3 in many units takes eight in any case, since its
// conversions and not its bytes bound it and many sequences have fewer rows than the largest (192 x window 1024 keys,
// 4 to 12 rows: 88 -> 70 us; sixteen rows in all: 116 against 117 us).
struct DecodeCut {
    int rows;
    bool team;
};
static_assert(kSMs * 3 * dec_warps(1) <= kAttnCounters, "a counter for every worker");
constexpr size_t kTeamUnits = kSMs / 2 + 1;
static DecodeCut decode_cut(int type, int group, int n_kv, int n_seq, int max_q) {
    DecodeCut c;
    const int all = group * max_q;
    c.rows = all <= 8 ? 8 : 16;
    c.team = (size_t)n_seq * n_kv < kTeamUnits;
    if (type == kE4M3 && !c.team) {
        c.rows = 8;
    }
    return c;
}

// for every cut that a call of this shape can get (the cache's type is not known here)
size_t attn_decode_part_bytes(int n_head, int n_kv, int head_dim, int n_seq, int max_q) {
    size_t most = 0;
    for (int type : {kF16, kE4M3}) {
        const DecodeCut c = decode_cut(type, n_head / n_kv, n_kv, n_seq, max_q);
        const int team = c.team ? kDecTeam : 1;
        const size_t slots = (size_t)kSMs * dec_per_sm(head_dim, c.rows == 8, team) * (c.team ? 1 : 2 * dec_warps(1));
        const size_t bytes = slots * part_floats(head_dim, c.rows == 8) * sizeof(float);
        most = bytes > most ? bytes : most;
    }
    return most;
}

cudaError_t launch_attn_decode(cudaStream_t s, const AttnDev & a) {
    g_launched = true;
    const DecodeCut c = decode_cut(a.kv.type, a.group, a.kv.n_kv, a.b.n_seq, a.b.max_q);
    auto go = [&](auto t, auto d) -> cudaError_t {
        constexpr int T = decltype(t)::value, D = decltype(d)::value;
        if (c.team) {
            return c.rows == 8 ? launch_t<T, D, true, kDecTeam>(s, a) : launch_t<T, D, false, kDecTeam>(s, a);
        }
        if constexpr (T == kE4M3) {
            return launch_t<T, D, true, 1>(s, a);
        } else {
            return c.rows == 8 ? launch_t<T, D, true, 1>(s, a) : launch_t<T, D, false, 1>(s, a);
        }
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
    if (!g_launched) {
        *status = 0;
        return cudaSuccess;
    }
    cudaError_t e = cudaMemcpyFromSymbol(status, g_attn_status, sizeof(int));
    if (e == cudaSuccess && clear && *status != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(int));
    }
    return e;
}

} // namespace b200q
