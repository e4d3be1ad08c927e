// Attention of many new tokens per sequence (prompts, chunks of prompts, long drafts) over the paged cache.
//
// The same sums as attn_decode.cu with the query rows in tiles of 128 on the fifth-generation tensor cores.
//
// * Units.  A unit is (sequence, KV head, 256 query rows): the rows are (token, query head of the group) pairs, so that K
//   and V are read once for all heads that share them, and run as two tiles of 128 rows that take turns: while the
//   tensor core multiplies for one, the other's softmax runs.  The units' key tiles of 128 in order form one list of
//   which each of the 148 CTAs takes an equal share; what the causal mask or the window hides from a whole unit is not in
//   the list.  A unit that spans CTAs is joined over the scratch by the CTA that finishes last, in order.
// * Accuracy.  q and p are split into two 16-bit parts (22 bits for fp16 and e4m3 caches, 16 for bf16), so both products take
//   twice the tensor work, which is what bounds the kernel: 4 x 128 x 128 x D multiply-adds a tile against 4096 a clock.
//   The tensor cores' sums drop bits towards zero at every step; each tile's p v therefore starts from zero in tensor
//   memory, low parts first, and the softmax threads add it to o in registers, rounded, with the factor of the new
//   maximum.  No accumulator is ever rescaled in tensor memory.
// * Roles.  Warps 0-3 and 4-7: softmax of the two tiles, a thread a row (o: D registers); warp 8: one thread issues the
//   products; warps 9-11 bring K and V into shared memory in the 128-byte swizzled form (16-bit caches by asynchronous
//   copies, e4m3 widened to fp16 on the way), rows that nobody sees as zeros.
//   Tensor memory: s of both tiles (128 columns each; p's two parts take the place of s as it is consumed), p v of both.
// * Every wait is bounded, by a time in which the CTA's products have not moved on; when one runs out the status word is
//   set and all roles run to their end without waiting.
//
// B200: 512 tokens after 32001 keys f16 591 us alone, 710 us in a run of them at the power limit: 1.14 and 0.95 PFLOP/s of tensor
// work (the two parts), 69 % of the measured burst and 69 % of the sustained bf16 rate.  A step of two tiles takes
// 7600 clocks of which the tensor pipe works 54 %; the softmax of a tile takes 4500, two thirds of it loads from tensor memory
// that nothing hides (330 clocks each while products run).  Wider loads (64 columns) spill and lose: 672 us.  The same step is most of
// the other prompts: 2048 tokens bf16 125 us, of which a CTA's 18.6 steps of two tiles take 74 and what its 2.8 units cost beside
// them (q in, first scores, rows out: about 9 us each, one after the other) 25; window 512 over 64 values, e4m3, 142 us: 24 steps
// and 4.5 units, some 90 and 40.
// bf16 keys widened to fp16 by the producers, for 22 bits there too, made the prompt of 2048 tokens 270 us: not taken.
#include "async.cuh"
#include "attn.cuh"

namespace b200q {

__device__ int g_attn_prompt_status = 0;
static std::atomic<bool> g_launched{false}; // nothing to read before

constexpr int kPrThreads = 384;
constexpr int kPrRows = 256; // rows of a unit
constexpr int kPrKeys = 128; // keys of a tile
constexpr int kPrProducers = 96;
constexpr int kPrHeader = 512;

__host__ __device__ constexpr int pr_slots(int dim) { return dim == 128 ? 3 : 6; }
__host__ __device__ constexpr int pr_tile_bytes(int dim) { return 128 * dim * 2; } // 128 rows of 16-bit values
__host__ __device__ constexpr int pr_smem(int dim) { return (4 + pr_slots(dim)) * pr_tile_bytes(dim) + kPrHeader + 1024; }
// floats that a CTA leaves of one 128-row tile: o by column, then m and l
__host__ __device__ constexpr int pr_part_floats(int dim) { return (dim + 2) * 128; }

// D[tmem] (+)= A B, 16-bit operands, fp32 sums; issued by one thread.  A from shared or from tensor memory.  Descriptors
// come as the low words of their first product with the shared high word; AO, BO step them (in 16 bytes, or columns), so
// that the unrolled products of a tile need no more than these registers.
template <int AO, int BO>
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b32 al, bl;\n\t.reg .b64 ad, bd;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "add.u32 al, %1, %7;\n\tadd.u32 bl, %3, %8;\n\tmov.b64 ad, {al, %2};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %5, p;\n\t}" ::"r"(d),
                 "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "n"(AO), "n"(BO)
                 : "memory");
}
template <int AO, int BO>
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b32 at, bl;\n\t.reg .b64 bd;\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "add.u32 at, %1, %6;\n\tadd.u32 bl, %2, %7;\n\tmov.b64 bd, {bl, %3};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [at], bd, %4, p;\n\t}" ::"r"(d),
                 "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "n"(AO), "n"(BO)
                 : "memory");
}
// f(0), f(1), ... with the index as a constant
template <int N, int I = 0, class F> __device__ __forceinline__ void unrolled(F && f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        unrolled<N, I + 1>(f);
    }
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint64_t (&v)[8]) { // 16 columns, in pairs
    tmem_ld16(taddr, reinterpret_cast<uint32_t (&)[16]>(v));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&u)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]),
                 "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint64_t (&v)[8]) {
    const uint32_t * u = reinterpret_cast<const uint32_t *>(v);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
                 "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// pairs of fp32 in one register pair
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float first2(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float second2(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Shared-memory operand descriptor, 128-byte swizzle: rows of 128 bytes in atoms of eight, `lbo` and `sbo` the byte
// distances between atoms (see the uses).
__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
    d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
    d |= (uint64_t)1 << 46; // descriptor version of this architecture
    d |= (uint64_t)2 << 61; // 128-byte swizzle
    return d;
}
// kind::f16: fp32 sums, fp16 or bf16 operands, A K-major, B K-major or (b_mn) N-major, M = 128
__device__ __forceinline__ uint32_t idesc_f16(bool bf16, bool b_mn, int N) {
    uint32_t d = 0;
    d |= 1u << 4;
    d |= (uint32_t)bf16 << 7;
    d |= (uint32_t)bf16 << 10;
    d |= (uint32_t)b_mn << 16;
    d |= (uint32_t)(N >> 3) << 17;
    d |= (uint32_t)(128 >> 4) << 24;
    return d;
}
// 16-byte chunk c of row r in a tile of 128 rows of 16-bit values: blocks of 64 values, 128 bytes a row, swizzled
__device__ __forceinline__ uint32_t sw128_off(int r, int c) {
    return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// the 128 softmax threads of a tile
__device__ __forceinline__ void tile_sync(int t) {
    if (t == 0) {
        asm volatile("bar.sync 1, 128;" ::: "memory");
    } else {
        asm volatile("bar.sync 2, 128;" ::: "memory");
    }
}

// A unit's rows and keys.
struct PromptUnit {
    SeqRows r;
    KeyTiles k;
    int blocks; // row blocks of the sequence
    int rows;   // rows of this block, at most kPrRows
    int row0;   // first row among the sequence's (token, head) rows
};
// A CTA's share of the list is measured in tiles plus kPrUnitCost a unit (its q, its join, its rows out): tile i of a unit
// that starts at position `pos` of the list lies at pos + kPrUnitCost + i.
constexpr int kPrUnitCost = 3;
constexpr int kPrMinShare = 2; // smallest share in positions of the list (one that lies in a unit's fixed cost holds no tile)
struct PromptSeg {
    int s, h, rb;
    int t_begin, t_end;
    long long pos;
};
// CTA b's share starts at b * each + min(b, more).
struct PromptShare {
    long long each, more, end;
    __device__ __forceinline__ int owner(long long x) const { // the CTA whose share holds position x
        return (int)(x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each);
    }
};

struct PromptBars {
    uint32_t q_full, s_full, p_full, kv_full, kv_empty, drain; // arrays of 8-byte barriers
};

template <int T, int D> struct Prompt {
    static constexpr int TILE = pr_tile_bytes(D), SLOTS = pr_slots(D), KS = D / 16;
    static constexpr bool BF = T == kBF16;
    static constexpr float BIAS = BF ? 0.0f : 14.0f;

    const AttnDev & a;
    uint32_t base;    // shared memory: Q[tile][part], K/V slots, header
    uint32_t hdr;
    uint32_t tmem;
    volatile int * fail;
    volatile int * progress; // the product warp's last item
    PromptBars bars;
    PromptShare share;

    __device__ __forceinline__ uint32_t q_addr(int tile, int part) const { return base + (tile * 2 + part) * TILE; }
    __device__ __forceinline__ uint32_t slot_addr(int slot) const { return base + (4 + slot) * TILE; }

    // A bounded wait; after one has run out nobody waits any more.  While products are issued the time starts anew: the second
    // tile's warps wait for as long as the CTA works on units without one, which may be most of a long call.
    __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) const {
        if (*fail) {
            return;
        }
        if (mbar_wait_some(bar, parity)) {
            return;
        }
        int at;
        do {
            at = *progress;
            if (mbar_wait_some(bar, parity)) {
                return;
            }
        } while (*progress != at);
        atomicExch(&g_attn_prompt_status, B200Q_ETIMEOUT);
        *fail = 1;
    }

    __device__ __forceinline__ PromptUnit unit(int s, int rb) const {
        PromptUnit u;
        u.r = seq_rows(a.b, a.kv.page_shift, s);
        const int all = u.r.n_run * a.group;
        u.blocks = (all + kPrRows - 1) / kPrRows;
        u.row0 = rb * kPrRows;
        u.rows = min(all - u.row0, kPrRows);
        const int first = u.r.n - u.r.n_row;
        const int pos0 = first + u.row0 / a.group, pos1 = first + (u.row0 + max(u.rows, 1) - 1) / a.group;
        u.k = key_tiles(pos0, min(u.r.n, max(pos1 + 1, 0)), kPrKeys, a.window, a.n_sink);
        return u;
    }
    // to the next unit of the share; false: there is none
    __device__ __forceinline__ bool advance(PromptSeg & x, PromptUnit & u) const {
        x.pos += u.k.count + kPrUnitCost;
        if (x.pos + kPrUnitCost >= share.end) {
            return false;
        }
        // heads innermost: neighbouring CTAs read neighbouring heads of the same pages
        if (++x.h == a.kv.n_kv) {
            x.h = 0;
            if (++x.rb >= u.blocks) {
                x.rb = 0;
                do {
                    x.s++;
                    u = unit(x.s, 0);
                } while (u.blocks == 0 && x.s + 1 < a.b.n_seq);
            } else {
                u = unit(x.s, x.rb);
            }
        }
        x.t_begin = 0;
        x.t_end = (int)min((long long)u.k.count, share.end - x.pos - kPrUnitCost);
        return true;
    }

    // ---- warp 8, one thread: the products
    __device__ void multiply(PromptSeg x, PromptUnit u) const {
        const uint32_t id_qk = idesc_f16(BF, false, kPrKeys), id_pv = idesc_f16(BF, true, D);
        uint32_t p_par = 0, q_par = 0, item = 0; // a bit a tile: the phase that is waited for
        auto s_cols = [&](int t) { return tmem + (uint32_t)t * 128; };
        auto o_cols = [&](int t) { return tmem + 256 + (uint32_t)t * 128; };
        const uint64_t k_desc = smem_desc_sw128(0, 16, 1024);
        // V as stored is N-major: blocks of 64 values 16384 bytes apart, groups of eight keys 1024
        const uint64_t v_desc = smem_desc_sw128(0, 16384, 1024);
        const uint32_t k_hi = (uint32_t)(k_desc >> 32), v_hi = (uint32_t)(v_desc >> 32);
        auto scores = [&](int t, uint32_t slot) { // s = q k: low part first
            const uint32_t qd = (uint32_t)k_desc | q_addr(t, 0) >> 4, kd = (uint32_t)k_desc | slot_addr((int)slot) >> 4, to = s_cols(t);
            unrolled<2 * KS>([&](auto n) {
                constexpr int i = decltype(n)::value;
                // 16 values: 32 bytes of a 128-byte row, then the next block of 64
                constexpr int part = i < KS ? 1 : 0, ks = i % KS, off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
                mma_f16_ss<off + part * (TILE >> 4), off>(to, qd, k_hi, kd, k_hi, id_qk, i > 0);
            });
        };
        auto values = [&](int t, uint32_t slot) { // o = p v: low part first
            const uint32_t vd = (uint32_t)v_desc | slot_addr((int)slot) >> 4, p = s_cols(t), to = o_cols(t);
            unrolled<kPrKeys / 8>([&](auto n) {
                constexpr int i = decltype(n)::value;
                constexpr int part = i < kPrKeys / 16 ? 1 : 0, ks = i % (kPrKeys / 16);
                mma_f16_ts<ks * 16 + part * 8, ks * (2048 >> 4)>(to, p, vd, v_hi, id_pv, i > 0);
            });
        };
        auto full = [&](uint32_t it) { wait(bars.kv_full + 8 * (it % SLOTS), (it / SLOTS) & 1); };
        auto release = [&](uint32_t it) { mma_commit(bars.kv_empty + 8 * (it % SLOTS)); };
        for (;;) {
            const int tiles = u.rows > 128 ? 2 : 1, n = x.t_end - x.t_begin;
            // items of this segment: K 0, V 0, K 1, V 1, ...
            full(item);
            tc_fence_after();
            for (int t = 0; t < tiles; t++) {
                wait(bars.q_full + 8 * t, (q_par >> t) & 1);
                q_par ^= 1u << t;
                tc_fence_after();
                scores(t, item % SLOTS);
                mma_commit(bars.s_full + 8 * t);
            }
            release(item);
            for (int j = 0; j < n; j++) {
                const uint32_t iv = item + 2 * j + 1, ik = iv + 1;
                *progress = (int)iv;
                for (int t = 0; t < tiles; t++) {
                    wait(bars.p_full + 8 * t, (p_par >> t) & 1);
                    p_par ^= 1u << t;
                    if (t == 0) {
                        full(iv);
                    }
                    tc_fence_after();
                    values(t, iv % SLOTS);
                    if (t == tiles - 1) {
                        release(iv); // before the scores: the next tile's keys take this place
                    }
                    if (j + 1 < n) {
                        if (t == 0) {
                            full(ik);
                            tc_fence_after();
                        }
                        scores(t, ik % SLOTS);
                    }
                    mma_commit(bars.s_full + 8 * t);
                }
                if (j + 1 < n) {
                    release(ik);
                }
            }
            item += 2 * n;
            if (!advance(x, u)) {
                break;
            }
        }
        mma_commit(bars.drain); // tensor memory is given back only when every product is done
        mbar_wait(bars.drain, 0, &g_attn_prompt_status);
    }

    // ---- warps 9-11: K and V into shared memory
    __device__ void produce(PromptSeg x, PromptUnit u) const {
        constexpr int EB = KvElem<T>::BYTES, ROWB = D * EB;
        constexpr int PIECES = kPrKeys * ROWB / 512;    // runs of 32 chunks of 16 bytes: one a warp
        constexpr int PER_GROUP = 16 * ROWB / 512;      // of a group of 16 keys
        constexpr int MINE = (PIECES + 2) / 3;
        constexpr int CPR = ROWB / 16;
        const int w = (int)(threadIdx.x >> 5) - 9, lane = threadIdx.x & 31;
        uint32_t item = 0;
        int pending = -1; // slot whose copies are in flight
        volatile int * meta = reinterpret_cast<volatile int *>(__cvta_shared_to_generic(hdr + 256));
        uint32_t tile_n = 0;
        auto flush = [&](bool all) {
            if (pending >= 0) {
                if (all) {
                    cp_async_wait<0>();
                } else {
                    cp_async_wait<1>();
                }
                fence_proxy_async();
                mbar_arrive(bars.kv_full + 8 * pending);
                pending = -1;
            }
        };
        auto ready = [&](uint32_t bar, uint32_t parity) {
            uint32_t ok;
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok)
                         : "r"(bar), "r"(parity)
                         : "memory");
            return __all_sync(~0u, ok != 0);
        };
        // the tile's groups of 16 keys, one a lane: where its rows lie and which of them are seen.  Looked up a tile ahead of the
        // copies, with a hint to bring the group into L2.
        auto look = [&](int i, unsigned long long & src, uint32_t & seen) {
            src = 0;
            seen = 0;
            if (i < x.t_end && lane < kPrKeys / 16) {
                const int k0 = key_tile(u.k, i) * kPrKeys + lane * 16;
                seen = keys_seen(u.k, k0, a.n_sink);
                if (seen) {
                    const int page = a.b.page_table[(size_t)x.s * a.b.table_stride + (k0 >> a.kv.page_shift)];
                    if (page >= 0 && page < a.kv.n_pages) {
                        src = (unsigned long long)page * a.kv.page_bytes +
                              (((unsigned long long)x.h << a.kv.page_shift) + (k0 & ((1 << a.kv.page_shift) - 1))) * ROWB;
                        if (w == 0) {
                            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.kv.k + src), "n"(16 * ROWB) : "memory");
                            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.kv.v + src), "n"(16 * ROWB) : "memory");
                        }
                    } else {
                        seen = 0;
                        note_bad_page(&g_attn_prompt_status);
                    }
                }
            }
            __syncwarp();
        };
        const int row = lane / CPR, chunk = lane % CPR; // of a piece
        // the next unit's q towards L2 while this one runs: a token's heads of the group lie together
        auto hint_q = [&]() {
            PromptSeg y = x;
            PromptUnit v = u;
            if (w == 1 && a.vec && a.group * D * 4 <= 65536 && advance(y, v)) {
                const int t0 = v.row0 / a.group, t1 = (v.row0 + v.rows - 1) / a.group;
                for (int i = t0 + lane; i <= t1; i += 32) {
                    const float * q = a.q + (size_t)(v.r.row0 + i) * a.q_stride + (size_t)y.h * a.group * D;
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(q), "r"(a.group * D * 4) : "memory");
                }
            }
        };
        for (;;) {
            hint_q();
            unsigned long long src, src_next;
            uint32_t seen, seen_next;
            look(x.t_begin, src, seen);
            for (int j = x.t_begin; j < x.t_end; j++) {
                look(j + 1, src_next, seen_next);
                const uint32_t valid = __ballot_sync(~0u, seen != 0), full = __ballot_sync(~0u, seen == 0xFFFFu);
                if (w == 0 && lane == 0) {
                    meta[tile_n & 7] = (int)valid;
                }
                tile_n++;
                for (int kv = 0; kv < 2; kv++, item++) {
                    const int slot = (int)(item % SLOTS);
                    const uint32_t bar = bars.kv_empty + 8 * slot, parity = ((item / SLOTS) & 1) ^ 1;
                    if (pending >= 0 && !ready(bar, parity)) {
                        flush(true);
                    }
                    wait(bar, parity);
                    __syncwarp();
                    const uint8_t * pool = kv ? a.kv.v : a.kv.k;
                    const uint32_t dst = slot_addr(slot);
                    if constexpr (T != kE4M3) {
#pragma unroll 1
                        for (int gr = w; gr < kPrKeys / 16; gr += 3) {
                            const uint8_t * from = pool + __shfl_sync(~0u, src, gr) + lane * 16;
                            const uint32_t to = dst + (uint32_t)gr * 2048;
                            if ((full >> gr) & 1) {
#pragma unroll
                                for (int i = 0; i < PER_GROUP; i++) {
                                    cp_async16(to + sw128_off(i * (32 / CPR) + row, chunk), from + i * 512);
                                }
                            } else { // rows that nobody sees (their memory may hold anything) become zeros
                                const uint32_t rows = __shfl_sync(~0u, seen, gr);
#pragma unroll
                                for (int i = 0; i < PER_GROUP; i++) {
                                    const bool take = (rows >> (i * (32 / CPR) + row)) & 1;
                                    const int n = take ? 16 : 0;
                                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + sw128_off(i * (32 / CPR) + row, chunk)),
                                                 "l"(take ? from + i * 512 : pool), "r"(n)
                                                 : "memory");
                                }
                            }
                        }
                        cp_async_commit();
                        flush(false);
                        pending = slot;
                    } else {
                        uint4 raw[MINE];
#pragma unroll
                        for (int q = 0; q < MINE; q++) {
                            const int i = w + 3 * q;
                            const int gr = min(i / PER_GROUP, kPrKeys / 16 - 1);
                            const unsigned long long off = __shfl_sync(~0u, src, gr) + (i % PER_GROUP) * 512 + lane * 16;
                            const uint32_t rows = __shfl_sync(~0u, seen, gr);
                            const int r = i * (32 / CPR) + row;
                            raw[q] = make_uint4(0, 0, 0, 0);
                            if (i < PIECES && ((rows >> (r & 15)) & 1)) {
                                raw[q] = __ldg(reinterpret_cast<const uint4 *>(pool + off));
                            }
                        }
#pragma unroll
                        for (int q = 0; q < MINE; q++) {
                            const int i = w + 3 * q;
                            if (i < PIECES) {
                                const int r = i * (32 / CPR) + row, c = chunk * 2;
                                sts128(dst + sw128_off(r, c), e4m3x2_to_f16x2(raw[q].x), e4m3x2_to_f16x2(raw[q].x >> 16),
                                       e4m3x2_to_f16x2(raw[q].y), e4m3x2_to_f16x2(raw[q].y >> 16));
                                sts128(dst + sw128_off(r, c + 1), e4m3x2_to_f16x2(raw[q].z), e4m3x2_to_f16x2(raw[q].z >> 16),
                                       e4m3x2_to_f16x2(raw[q].w), e4m3x2_to_f16x2(raw[q].w >> 16));
                            }
                        }
                        fence_proxy_async();
                        mbar_arrive(bars.kv_full + 8 * slot);
                    }
                }
                src = src_next;
                seen = seen_next;
            }
            if (!advance(x, u)) {
                break;
            }
        }
        flush(true);
    }

    // ---- warps 0-3 and 4-7: softmax, a thread a row of its tile
    __device__ void softmax(PromptSeg x, PromptUnit u) const {
        const int tid = threadIdx.x & 127, t = (int)(threadIdx.x >> 7), lane = threadIdx.x & 31, warp_row = tid & ~31;
        const uint32_t lanes = (uint32_t)warp_row << 16;
        const uint32_t s_cols = tmem + lanes + (uint32_t)t * 128, o_cols = tmem + lanes + 256 + (uint32_t)t * 128;
        const volatile int * meta = reinterpret_cast<const volatile int *>(__cvta_shared_to_generic(hdr + 256));
        volatile int * last = reinterpret_cast<volatile int *>(__cvta_shared_to_generic(hdr + 320)) + t;
        uint32_t s_par = 0, tile_n = 0;
        constexpr int RPL = 128 / D; // rows that one coalesced access of the warp covers (32 lanes of four values)
        for (;;) {
            const int n = x.t_end - x.t_begin;
            const bool mine = t == 0 || u.rows > 128; // the second tile may be empty
            if (mine) {
                const int r0 = u.row0 + t * 128, r = r0 + tid, r_end = u.row0 + u.rows;
                const bool live = r < r_end;
                const int first = u.r.n - u.r.n_row;
                const int tok = live ? r / a.group : 0, head = x.h * a.group + (live ? r - tok * a.group : 0);
                const int pos = live ? first + tok : -1;
                const int pos_min = first + r0 / a.group, pos_max = first + min(r0 + 127, r_end - 1) / a.group;
                const uint32_t live_rows = __ballot_sync(~0u, live); // of the warp's 32
                // q in two parts to shared memory, rows read whole by the warp
                float cq = a.scale_log2;
                const long long q_at = (long long)(u.r.row0 + tok) * a.q_stride + (long long)head * D;
                const int d = lane % (32 / RPL) * 4;
#pragma unroll 1
                for (int i0 = 0; i0 < 32; i0 += 16 * RPL) {
                    float4 v[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int row = i0 + i * RPL + lane / (32 / RPL);
                        const float * q = a.q + __shfl_sync(~0u, q_at, row) + d;
                        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if ((live_rows >> row) & 1) {
                            if (a.vec) {
                                v[i] = __ldg(reinterpret_cast<const float4 *>(q));
                            } else {
                                v[i] = make_float4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int row = i0 + i * RPL + lane / (32 / RPL);
                        if constexpr (!BF) {
                            float top = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
                            for (int w = 16 / RPL; w > 0; w >>= 1) {
                                top = fmaxf(top, __shfl_xor_sync(~0u, top, w));
                            }
                            const int e = pow2_to_top(top);
                            const float up = exp2_int(e);
                            v[i] = make_float4(v[i].x * up, v[i].y * up, v[i].z * up, v[i].w * up);
                            // the thread of the row takes the factor back out of the scores
#pragma unroll
                            for (int k = 0; k < RPL; k++) {
                                const int back = __shfl_sync(~0u, e, k * (32 / RPL));
                                cq *= lane == i0 + i * RPL + k ? exp2_int(-back) : 1.0f;
                            }
                        }
                        uint32_t p0[2], p1[2];
                        split_pair<T>(v[i].x, v[i].y, p0);
                        split_pair<T>(v[i].z, v[i].w, p1);
                        const uint32_t to = sw128_off(warp_row + row, d / 8) + (uint32_t)(d & 4) * 2;
                        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(q_addr(t, 0) + to), "r"(p0[0]), "r"(p1[0]) : "memory");
                        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(q_addr(t, 1) + to), "r"(p0[1]), "r"(p1[1]) : "memory");
                    }
                }
                fence_proxy_async();
                mbar_arrive(bars.q_full + 8 * t);

                uint64_t o[D / 2]; // pairs of fp32
#pragma unroll
                for (int i = 0; i < D / 2; i++) {
                    o[i] = 0;
                }
                float m = -INFINITY, l = 0.0f, f = 1.0f;
                const int low = a.window ? pos - a.window + 1 : 0;
                // A load from tensor memory is waited for only when the next one has been issued.
                auto add_o = [&]() { // o = o f + the tile's p v
                    const uint64_t ff = pair2(f, f);
                    uint64_t v[2][8];
                    tmem_ld16(o_cols, v[0]);
#pragma unroll
                    for (int c = 0; c < D / 16; c++) {
                        tmem_ld_wait();
                        if (c + 1 < D / 16) {
                            tmem_ld16(o_cols + 16 * (c + 1), v[(c + 1) & 1]);
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            o[8 * c + i] = fma2(o[8 * c + i], ff, v[c & 1][i]);
                        }
                    }
                };
                auto next_s = [&]() {
                    wait(bars.s_full + 8 * t, s_par);
                    s_par ^= 1;
                    __syncwarp();
                    tc_fence_after();
                };
                for (int j = 0; j < n; j++) {
                    next_s();
                    const int key0 = key_tile(u.k, x.t_begin + j) * kPrKeys;
                    const uint32_t valid = (uint32_t)meta[(tile_n + j) & 7];
                    const bool whole = valid == 0xFFu && key0 + kPrKeys - 1 <= pos_min &&
                                       (a.window == 0 || key0 > pos_max - a.window || key0 + kPrKeys <= a.n_sink);
                    // columns that the row sees, of the 16 (one group) from column c on
                    auto seen = [&](int c) {
                        auto below = [](int k) { return k >= 16 ? 0xFFFFu : (k <= 0 ? 0u : (1u << k) - 1u); }; // bits 0 .. k-1
                        const uint32_t bits = below(pos + 1 - key0 - c) & (~below(low - key0 - c) | below(a.n_sink - key0 - c));
                        return (valid >> (c / 16)) & 1 ? bits : 0u;
                    };
                    float top = -INFINITY;
                    // On a border, most groups of 16 keys are still seen by all rows of the warp or by none: only the others
                    // take masks, and their masked scores go back, so that the second reading needs none.  The two
                    // kinds of tile have code of their own: the tests would cost whole tiles 5 %.
                    uint32_t some = 0xFFu, mixed = 0;
                    auto look = [&](int c, uint64_t (&v)[8], auto border) {
                        if constexpr (decltype(border)::value) {
                            if (!((some >> (c / 16)) & 1)) {
                                return;
                            }
                            if ((mixed >> (c / 16)) & 1) {
                                const uint32_t bits = seen(c);
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    v[i] = pair2((bits >> (2 * i)) & 1 ? first2(v[i]) : -INFINITY,
                                                 (bits >> (2 * i + 1)) & 1 ? second2(v[i]) : -INFINITY);
                                }
                                tmem_st16(s_cols + c, v);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            top = fmaxf(top, fmaxf(first2(v[i]), second2(v[i])));
                        }
                    };
                    auto maximum = [&](auto border) {
                        uint64_t v[2][8];
                        tmem_ld16(s_cols, v[0]);
#pragma unroll 1
                        for (int c = 0; c < kPrKeys; c += 32) {
                            tmem_ld_wait();
                            tmem_ld16(s_cols + c + 16, v[1]);
                            look(c, v[0], border);
                            tmem_ld_wait();
                            if (c + 32 < kPrKeys) {
                                tmem_ld16(s_cols + c + 32, v[0]);
                            }
                            look(c + 16, v[1], border);
                        }
                    };
                    if (whole) {
                        maximum(std::false_type{});
                    } else {
                        some = 0;
#pragma unroll 1
                        for (int g = 0; g < kPrKeys / 16; g++) {
                            const uint32_t bits = seen(16 * g);
                            some |= __any_sync(~0u, bits != 0) ? 1u << g : 0u;
                            mixed |= __all_sync(~0u, bits == 0xFFFFu) ? 0u : 1u << g;
                        }
                        maximum(std::true_type{});
                        tmem_st_wait();
                    }
                    const float mn = fmaxf(m, top * cq);
                    const float f_new = m == mn ? 1.0f : exp2_fast(m - mn);
                    const float off = BIAS - (mn == -INFINITY ? 0.0f : mn);
                    m = mn;
                    uint64_t sum = 0, sum1 = 0;
                    const uint64_t cc = pair2(cq, cq), oo = pair2(off, off);
                    auto weigh = [&](int c, const uint64_t (&v)[8], auto border) { // p of 16 keys takes the place of their s
                        uint32_t hi[8], lo[8];
                        if constexpr (decltype(border)::value) {
                            if (!((some >> (c / 16)) & 1)) {
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    hi[i] = 0;
                                }
                                tmem_st8(s_cols + c, hi);
                                tmem_st8(s_cols + c + 8, hi);
                                return;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const uint64_t e = fma2(v[i], cc, oo);
                            const float p0 = exp2_fast(first2(e)), p1 = exp2_fast(second2(e));
                            const uint64_t pp = pair2(p0, p1);
                            if (i & 1) {
                                sum1 = add2(sum1, pp);
                            } else {
                                sum = add2(sum, pp);
                            }
                            uint32_t part[2];
                            split_pair<T>(p0, p1, part);
                            hi[i] = part[0];
                            lo[i] = part[1];
                        }
                        tmem_st8(s_cols + c, hi);
                        tmem_st8(s_cols + c + 8, lo);
                    };
                    auto weights = [&](auto border) {
                        uint64_t v[2][8];
                        tmem_ld16(s_cols, v[0]);
#pragma unroll 1
                        for (int c = 0; c < kPrKeys; c += 32) {
                            tmem_ld_wait();
                            tmem_ld16(s_cols + c + 16, v[1]);
                            weigh(c, v[0], border);
                            tmem_ld_wait();
                            if (c + 32 < kPrKeys) {
                                tmem_ld16(s_cols + c + 32, v[0]);
                            }
                            weigh(c + 16, v[1], border);
                        }
                    };
                    if (whole) {
                        weights(std::false_type{});
                    } else {
                        weights(std::true_type{});
                    }
                    sum = add2(sum, sum1);
                    l = fmaf(l, f_new, first2(sum) + second2(sum));
                    if (j > 0) {
                        add_o(); // of the tile before: complete, its commit came before this tile's s
                    }
                    f = f_new;
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(bars.p_full + 8 * t);
                }
                next_s();
                add_o();
                tc_fence_before();

                bool write = true;
                if (n != u.k.count) { // the unit spans CTAs
                    const int b0 = share.owner(x.pos + kPrUnitCost), b1 = share.owner(x.pos + kPrUnitCost + u.k.count - 1);
                    // four columns of a thread lie together, a warp's 512 bytes side by side
                    auto part = [&](int b, bool second) {
                        return a.parts + ((size_t)(b * 2 + (second ? 1 : 0)) * 2 + t) * pr_part_floats(D) + tid * 4;
                    };
                    auto stats = [&](int b, bool second) {
                        return a.parts + ((size_t)(b * 2 + (second ? 1 : 0)) * 2 + t) * pr_part_floats(D) + D * 128 + tid;
                    };
                    // of a CTA's two places the second holds the unit that starts in its share and runs on behind it
                    const bool second = x.t_begin == 0;
                    float * to = part((int)blockIdx.x, second), * st = stats((int)blockIdx.x, second);
#pragma unroll
                    for (int i = 0; i < D / 4; i++) {
                        *reinterpret_cast<float4 *>(to + i * 512) = make_float4(first2(o[2 * i]), second2(o[2 * i]), first2(o[2 * i + 1]), second2(o[2 * i + 1]));
                    }
                    st[0] = m;
                    st[128] = l;
                    __threadfence();
                    tile_sync(t);
                    if (tid == 0) {
                        uint32_t * counter = a.counters + b0 * 2 + t; // one unit at most starts in a CTA's share and runs on behind it
                        const bool end = atomicAdd(counter, 1u) == (uint32_t)(b1 - b0);
                        if (end) {
                            *counter = 0; // as the next call wants it
                        }
                        __threadfence();
                        *last = end;
                    }
                    tile_sync(t);
                    write = *last;
                    if (write) {
                        m = -INFINITY;
                        for (int b = b0; b <= b1; b++) {
                            m = fmaxf(m, __ldcg(stats(b, b == b0)));
                        }
                        l = 0.0f;
#pragma unroll
                        for (int i = 0; i < D / 2; i++) {
                            o[i] = 0;
                        }
                        for (int b = b0; b <= b1; b++) {
                            const float * p = part(b, b == b0), * s2 = stats(b, b == b0);
                            const float m2 = __ldcg(s2);
                            const float w = m2 == m ? 1.0f : exp2_fast(m2 - m);
                            const uint64_t ww = pair2(w, w);
                            l = fmaf(__ldcg(s2 + 128), w, l);
#pragma unroll
                            for (int i = 0; i < D / 4; i++) {
                                const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + i * 512));
                                o[2 * i] = fma2(pair2(v.x, v.y), ww, o[2 * i]);
                                o[2 * i + 1] = fma2(pair2(v.z, v.w), ww, o[2 * i + 1]);
                            }
                        }
                    }
                }
                if (write) {
                    // through the tile's q space, whose products are done, so that rows leave whole; a warp takes back the 32
                    // rows that it put there
                    const float inv = l > 0.0f || isnan(l) ? a.v_scale / l : 0.0f; // no visible key: zeros
                    const uint64_t ii = pair2(inv, inv);
                    const uint32_t stage = q_addr(t, 0) + (uint32_t)warp_row * D * 4;
#pragma unroll
                    for (int i = 0; i < D / 4; i++) {
                        const uint64_t lo2 = mul2(o[2 * i], ii), hi2 = mul2(o[2 * i + 1], ii);
                        sts128(stage + (uint32_t)(lane * D * 4 + ((i ^ (lane & 7)) << 4)), (uint32_t)lo2, (uint32_t)(lo2 >> 32), (uint32_t)hi2,
                               (uint32_t)(hi2 >> 32));
                    }
                    __syncwarp();
                    const long long out_at = (long long)(u.r.row0 + tok) * a.out_stride + (long long)head * D;
#pragma unroll 8
                    for (int i = 0; i < 32; i += RPL) {
                        const int row = i + lane / (32 / RPL);
                        float v[4];
                        const uint32_t from = stage + (uint32_t)(row * D * 4 + (((d / 4) ^ (row & 7)) << 4));
                        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(from) : "memory");
                        float * out = a.out + __shfl_sync(~0u, out_at, row) + d;
                        if ((live_rows >> row) & 1) {
                            if (a.vec) {
                                *reinterpret_cast<float4 *>(out) = make_float4(v[0], v[1], v[2], v[3]);
                            } else {
                                out[0] = v[0], out[1] = v[1], out[2] = v[2], out[3] = v[3];
                            }
                        }
                    }
                    // The space takes the next unit's q, whose swizzled blocks of any warp lie over the rows of several: none
                    // before all four have sent theirs.
                    tile_sync(t);
                }
            }
            tile_n += (uint32_t)n;
            if (!advance(x, u)) {
                break;
            }
        }
    }
};

template <int T, int D> __global__ void __launch_bounds__(kPrThreads, 1) attn_prompt_kernel(const __grid_constant__ AttnDev a) {
    extern __shared__ uint8_t smem_raw[];
    using P = Prompt<T, D>;
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t * gen = smem_raw + (base - raw);
    constexpr uint32_t HDR = (4 + P::SLOTS) * P::TILE;
    const uint32_t hdr = base + HDR;
    // header: q_full[2] @0, s_full[2] @16, p_full[2] @32, drain @48, kv_full[6] @64, kv_empty[6] @128, seen groups of eight
    // tiles @256, last[2] @320, tensor memory address @328, fail @332, found share @336, sums @352,
    // progress @448
    P p{a, base, hdr, 0, reinterpret_cast<volatile int *>(gen + HDR + 332), reinterpret_cast<volatile int *>(gen + HDR + 448), {hdr, hdr + 16, hdr + 32, hdr + 64, hdr + 128, hdr + 48}, {0, 0, 0}};
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) {
        for (int t = 0; t < 2; t++) {
            mbar_init(p.bars.q_full + 8 * t, 128);
            mbar_init(p.bars.s_full + 8 * t, 1);
            mbar_init(p.bars.p_full + 8 * t, 128);
        }
        for (int s = 0; s < P::SLOTS; s++) {
            mbar_init(p.bars.kv_full + 8 * s, kPrProducers);
            mbar_init(p.bars.kv_empty + 8 * s, 1);
        }
        mbar_init(p.bars.drain, 1);
        *p.fail = 0;
        *p.progress = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        tmem_alloc(hdr + 328, 512);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- the CTA's share of the list: units by (sequence, row block, KV head).  The first blocks of the sequences
    // go through shared memory (the tiles' space, not yet in use), then the threads look at a (sequence, row block) each.
    int * first_block = reinterpret_cast<int *>(gen); // [n_seq + 1]
    volatile long long * s_sum = reinterpret_cast<volatile long long *>(gen + HDR + 352); // one a warp
    auto block_scan = [&](long long v, long long & before) { // sum over the threads below; returns the block's sum
        long long y = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long z = __shfl_up_sync(~0u, y, d);
            y += lane >= d ? z : 0;
        }
        __syncthreads();
        if (lane == 31) {
            s_sum[warp] = y;
        }
        __syncthreads();
        long long all = 0, mine = 0;
#pragma unroll
        for (int w = 0; w < kPrThreads / 32; w++) {
            mine += w < warp ? s_sum[w] : 0;
            all += s_sum[w];
        }
        before = mine + y - v;
        return all;
    };
    int n_pairs = 0;
    long long before;
    for (int s0 = 0; s0 < a.b.n_seq; s0 += kPrThreads) {
        const int s = s0 + tid;
        const int v = s < a.b.n_seq ? (seq_rows(a.b, a.kv.page_shift, s).n_run * a.group + kPrRows - 1) / kPrRows : 0;
        const int all = (int)block_scan(v, before);
        if (s < a.b.n_seq) {
            first_block[s] = n_pairs + (int)before;
        }
        n_pairs += all;
    }
    __syncthreads();
    auto find = [&](int pair, int & s, int & rb) { // the last sequence whose first block is not behind the pair
        int lo = 0, hi = a.b.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first_block[mid] <= pair) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        s = lo;
        rb = pair - first_block[lo];
    };
    long long total = 0;
    auto cost = [&](int pair, int & s, int & rb) { // of the pair's unit of one head
        if (pair >= n_pairs) {
            return 0;
        }
        find(pair, s, rb);
        return p.unit(s, rb).k.count + kPrUnitCost;
    };
    int s_first = 0, rb_first = 0;
    long long before_first = 0;
    const int v_first = cost(tid, s_first, rb_first);
    const long long all_first = block_scan(v_first, before_first);
    total = all_first * a.kv.n_kv;
    for (int p0 = kPrThreads; p0 < n_pairs; p0 += kPrThreads) {
        int s, rb;
        total += block_scan(cost(p0 + tid, s, rb), before) * a.kv.n_kv;
    }
    const long long want = (total + kPrMinShare - 1) / kPrMinShare;
    const long long nw = max(1LL, want < gridDim.x ? want : gridDim.x);
    p.share.each = total / nw;
    p.share.more = total - p.share.each * nw;
    const long long c0 = blockIdx.x * p.share.each + min((long long)blockIdx.x, p.share.more);
    p.share.end = c0 + p.share.each + (blockIdx.x < p.share.more ? 1 : 0);
    bool work = blockIdx.x < nw && p.share.end > c0;
    PromptSeg seg = {};
    volatile int * found = reinterpret_cast<volatile int *>(gen + HDR + 336); // s, rb, head, position in the unit
    if (work) {
        long long run = 0;
        for (int p0 = 0; p0 < n_pairs; p0 += kPrThreads) {
            int v = v_first, s = s_first, rb = rb_first;
            long long all = all_first;
            before = before_first;
            if (p0 > 0) {
                v = cost(p0 + tid, s, rb);
                all = block_scan(v, before);
            }
            const long long b = run + before * a.kv.n_kv;
            if (v > 0 && c0 >= b && c0 < b + (long long)v * a.kv.n_kv) {
                const long long in = c0 - b;
                found[0] = s;
                found[1] = rb;
                found[2] = (int)(in / v);
                found[3] = (int)(in % v);
            }
            run += all * a.kv.n_kv;
            if (run > c0) {
                break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    p.tmem = *reinterpret_cast<volatile uint32_t *>(gen + HDR + 328);
    PromptUnit u = {};
    if (work) {
        seg.s = found[0];
        seg.rb = found[1];
        seg.h = found[2];
        seg.pos = c0 - found[3];
        u = p.unit(seg.s, seg.rb);
        seg.t_begin = max(0, found[3] - kPrUnitCost);
        seg.t_end = (int)min((long long)u.k.count, p.share.end - seg.pos - kPrUnitCost);
        work = seg.t_end > seg.t_begin; // a share may end inside a unit's fixed cost, and has no tile then
    }
    if (work) {
        if (warp < 8) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
            p.softmax(seg, u);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
            if (warp > 8) {
                p.produce(seg, u);
            } else if (lane == 0) {
                p.multiply(seg, u);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tmem_dealloc(p.tmem, 512);
    }
}

template <int T, int D> static cudaError_t launch_t(cudaStream_t s, const AttnDev & a) {
    const cudaError_t e = ensure_dynamic_smem((const void *)attn_prompt_kernel<T, D>, pr_smem(D));
    if (e != cudaSuccess) {
        return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kSMs);
    cfg.blockDim = dim3(kPrThreads);
    cfg.dynamicSmemBytes = pr_smem(D);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_prompt_kernel<T, D>, a);
}

static_assert(kSMs * 2 <= kAttnCounters, "a counter for every CTA and tile");
size_t attn_prompt_part_bytes(int head_dim) { return (size_t)kSMs * 4 * pr_part_floats(head_dim) * sizeof(float); }

cudaError_t launch_attn_prompt(cudaStream_t s, AttnDev a) {
    g_launched = true;
    a.vec = !((uintptr_t)a.q & 15) && !((uintptr_t)a.out & 15) && !(a.q_stride & 3) && !(a.out_stride & 3);
    switch (a.kv.type) {
    case kF16: return a.kv.head_dim == 64 ? launch_t<kF16, 64>(s, a) : launch_t<kF16, 128>(s, a);
    case kBF16: return a.kv.head_dim == 64 ? launch_t<kBF16, 64>(s, a) : launch_t<kBF16, 128>(s, a);
    default: return a.kv.head_dim == 64 ? launch_t<kE4M3, 64>(s, a) : launch_t<kE4M3, 128>(s, a);
    }
}

cudaError_t read_attn_prompt_status(int * status, bool clear) {
    if (!g_launched) {
        *status = 0;
        return cudaSuccess;
    }
    cudaError_t e = cudaMemcpyFromSymbol(status, g_attn_prompt_status, sizeof(int));
    if (e == cudaSuccess && clear && *status != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_attn_prompt_status, &zero, sizeof(int));
    }
    return e;
}

} // namespace b200q
