// C ABI of the attention side: argument validation and dispatch of rope_append, attn and the page operators.
#include <cmath>
#include <cstring>

#include "attn.cuh"

namespace b200q {

static inline bool aligned(const void * p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

static int check_cache(const char * who, const b200q_kv_cache * c, KvDev & d) {
    if (!c || !c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) {
        set_error("%s: the cache's k and v must be non-null and 16-byte aligned", who);
        return B200Q_EINVAL;
    }
    if (c->type != B200Q_KV_F16 && c->type != B200Q_KV_BF16 && c->type != B200Q_KV_E4M3) {
        set_error("%s: unsupported cache type %u (supported: F16=1 BF16=30 E4M3=256)", who, c->type);
        return B200Q_EUNSUPPORTED;
    }
    if (c->head_dim != 64 && c->head_dim != 128) {
        set_error("%s: head_dim must be 64 or 128 (got %d)", who, c->head_dim);
        return B200Q_EUNSUPPORTED;
    }
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) {
        set_error("%s: page_size must be 16, 32, 64 or 128 (got %d)", who, c->page_size);
        return B200Q_EUNSUPPORTED;
    }
    const int eb = kv_elem_bytes(c->type);
    if (c->n_pages < 1 || c->n_kv < 1 || c->n_kv > 4096 ||
        c->page_stride < (int64_t)c->n_kv * c->page_size * c->head_dim || (c->page_stride * eb) % 16) {
        set_error("%s: bad cache shape (n_pages=%d n_kv=%d page_stride=%lld: at least n_kv * page_size * head_dim, a "
                  "multiple of 16 bytes)", who, c->n_pages, c->n_kv, (long long)c->page_stride);
        return B200Q_EINVAL;
    }
    if (!(c->k_scale > 0.0f) || !(c->v_scale > 0.0f) || std::isinf(c->k_scale) || std::isinf(c->v_scale)) {
        set_error("%s: k_scale and v_scale must be finite and positive", who);
        return B200Q_EINVAL;
    }
    d.k = static_cast<uint8_t *>(c->k);
    d.v = static_cast<uint8_t *>(c->v);
    d.page_bytes = c->page_stride * eb;
    d.type = (int32_t)c->type;
    d.n_pages = c->n_pages;
    d.page_shift = c->page_size == 16 ? 4 : (c->page_size == 32 ? 5 : (c->page_size == 64 ? 6 : 7));
    d.n_kv = c->n_kv;
    d.head_dim = c->head_dim;
    d.k_scale = c->k_scale;
    d.v_scale = c->v_scale;
    return B200Q_OK;
}

static int check_batch(const char * who, const b200q_kv_batch * b, BatchDev & d) {
    if (!b || !b->page_table || !b->q_start || !b->kv_len || !aligned(b->page_table, 4) || !aligned(b->q_start, 4) ||
        !aligned(b->kv_len, 4)) {
        set_error("%s: the batch's page_table, q_start and kv_len must be non-null and 4-byte aligned", who);
        return B200Q_EINVAL;
    }
    if (b->n_seq < 1 || b->n_tok < 0 || b->max_q < 1 || b->table_stride < 1) {
        set_error("%s: bad batch shape (n_seq=%d n_tok=%d max_q=%d table_stride=%d)", who, b->n_seq, b->n_tok, b->max_q,
                  b->table_stride);
        return B200Q_EINVAL;
    }
    if (b->n_seq > kMaxSeqs) {
        set_error("%s: a step holds up to %d sequences (got %d)", who, kMaxSeqs, b->n_seq);
        return B200Q_EUNSUPPORTED;
    }
    d.page_table = b->page_table;
    d.q_start = b->q_start;
    d.kv_len = b->kv_len;
    d.table_stride = b->table_stride;
    d.n_seq = b->n_seq;
    d.n_tok = b->n_tok;
    d.max_q = b->max_q < b->n_tok ? b->max_q : (b->n_tok > 0 ? b->n_tok : 1); // no sequence has more rows than there are
    return B200Q_OK;
}

static int check_rope(const char * who, const b200q_rope * r) {
    if (!r || r->n_rot < 2 || (r->n_rot & 1) || r->n_rot > 128) {
        set_error("%s: n_rot must be even, 2 to 128 (got %d)", who, r ? r->n_rot : 0);
        return B200Q_EINVAL;
    }
    return B200Q_OK;
}

// rows of `n` values, `stride` apart, as a byte range
static bool rows_overlap(const float * a, int a_stride, int a_n, const float * b, int b_stride, int b_n, int rows) {
    const uintptr_t a0 = (uintptr_t)a, a1 = (uintptr_t)(a + (size_t)(rows - 1) * a_stride + a_n);
    const uintptr_t b0 = (uintptr_t)b, b1 = (uintptr_t)(b + (size_t)(rows - 1) * b_stride + b_n);
    if (a1 <= b0 || b1 <= a0) {
        return false;
    }
    if (a_stride == b_stride && a0 % 4 == b0 % 4) { // columns of one buffer
        const long long s = a_stride, d = ((long long)(b0 - a0) / 4) % s, at = d < 0 ? d + s : d;
        return at < a_n || at + b_n > s;
    }
    return true;
}

constexpr size_t kCounterBytes = kAttnCounters * sizeof(uint32_t);

} // namespace b200q

using namespace b200q;

extern "C" {

int b200q_rope_table(void * stream, const b200q_rope * rope, double * table) {
    const int rc = check_rope("b200q_rope_table", rope);
    if (rc != B200Q_OK) {
        return rc;
    }
    if (!table || !aligned(table, 8) || !aligned(rope->freq_factors, 4)) {
        set_error("b200q_rope_table: table must be non-null and 8-byte aligned, freq_factors 4-byte aligned");
        return B200Q_EINVAL;
    }
    if (!(rope->base > 1.0f) || std::isinf(rope->base) || !(rope->freq_scale > 0.0f) || !(rope->freq_scale <= 1.0f) ||
        !(rope->ext_factor >= 0.0f) || !(rope->ext_factor <= 1.0f) || !(rope->attn_factor > 0.0f) || std::isinf(rope->attn_factor)) {
        set_error("b200q_rope_table: base must be above 1, freq_scale in (0, 1], ext_factor in [0, 1], attn_factor positive");
        return B200Q_EINVAL;
    }
    if (rope->ext_factor > 0.0f && (rope->n_ctx_orig < 1 || !(rope->beta_fast > 0.0f) || !(rope->beta_slow > 0.0f) ||
                                    std::isinf(rope->beta_fast) || std::isinf(rope->beta_slow))) {
        set_error("b200q_rope_table: YaRN needs n_ctx_orig, beta_fast and beta_slow above 0");
        return B200Q_EINVAL;
    }
    B200Q_CUDA_OK(launch_rope_table((cudaStream_t)stream, *rope, table));
    return B200Q_OK;
}

int b200q_rope_append(void * stream, const double * table, const b200q_rope * rope, const float * q, int q_stride, int n_head,
                      const float * k, int k_stride, const float * v, int v_stride, float * q_out, int q_out_stride,
                      const b200q_kv_cache * cache, const b200q_kv_batch * batch) {
    const char * who = "b200q_rope_append";
    KvDev kv;
    BatchDev b;
    int rc = check_cache(who, cache, kv);
    rc = rc == B200Q_OK ? check_batch(who, batch, b) : rc;
    rc = rc == B200Q_OK && table ? check_rope(who, rope) : rc;
    if (rc != B200Q_OK) {
        return rc;
    }
    if (table && (!aligned(table, 8) || rope->n_rot > kv.head_dim)) {
        set_error("%s: n_rot must not exceed head_dim, the table must be 8-byte aligned (n_rot=%d)", who, rope->n_rot);
        return B200Q_EINVAL;
    }
    if ((!q && !k) || (!k) != (!v) || (q && !q_out) || !aligned(q, 4) || !aligned(k, 4) || !aligned(v, 4) || (q && !aligned(q_out, 4))) {
        set_error("%s: q with q_out, or k with v, or both must be non-null, and 4-byte aligned", who);
        return B200Q_EINVAL;
    }
    const int kd = kv.n_kv * kv.head_dim;
    if (q && (n_head < 1 || n_head > 65536 / 8 || q_stride < n_head * kv.head_dim || q_out_stride < n_head * kv.head_dim)) {
        set_error("%s: n_head must be 1..8192 and the strides of q and q_out at least n_head * head_dim", who);
        return B200Q_EINVAL;
    }
    if (k && (k_stride < kd || v_stride < kd)) {
        set_error("%s: the strides of k and v must be at least n_kv * head_dim", who);
        return B200Q_EINVAL;
    }
    if (b.n_tok == 0) {
        return B200Q_OK;
    }
    if (q && !(q == q_out && q_stride == q_out_stride) &&
        rows_overlap(q, q_stride, n_head * kv.head_dim, q_out, q_out_stride, n_head * kv.head_dim, b.n_tok)) {
        set_error("%s: q_out must be q or not overlap it", who);
        return B200Q_EINVAL;
    }
    if (q && k && (rows_overlap(k, k_stride, kd, q_out, q_out_stride, n_head * kv.head_dim, b.n_tok) ||
                   rows_overlap(v, v_stride, kd, q_out, q_out_stride, n_head * kv.head_dim, b.n_tok))) {
        set_error("%s: q_out must not overlap k or v", who);
        return B200Q_EINVAL;
    }
    B200Q_CUDA_OK(launch_rope_append((cudaStream_t)stream, table, table ? rope->n_rot : 0, table ? rope->interleaved != 0 : 0, q,
                                     q_stride, n_head, k, k_stride, v, v_stride, q_out, q_out_stride, kv, b));
    return B200Q_OK;
}

size_t b200q_attn_scratch_bytes(int n_head, int n_kv, int head_dim, int n_seq, int n_tok, int max_q) {
    if (n_head < 1 || n_kv < 1 || n_head % n_kv || n_seq < 1 || n_tok < 0 || max_q < 1 || (head_dim != 64 && head_dim != 128)) {
        return 0;
    }
    const int mq = max_q < n_tok ? max_q : (n_tok > 0 ? n_tok : 1);
    const size_t parts = (long long)mq * (n_head / n_kv) <= kDecodeRows ? attn_decode_part_bytes(n_head, n_kv, head_dim, n_seq, mq)
                                                                        : attn_prompt_part_bytes(head_dim);
    return kCounterBytes + parts;
}

int b200q_attn(void * stream, const float * q, int q_stride, int n_head, const b200q_kv_cache * cache,
               const b200q_kv_batch * batch, const b200q_attn_opts * opts, float * out, int out_stride, void * scratch,
               size_t scratch_bytes) {
    const char * who = "b200q_attn";
    AttnDev a = {};
    int rc = check_cache(who, cache, a.kv);
    rc = rc == B200Q_OK ? check_batch(who, batch, a.b) : rc;
    if (rc != B200Q_OK) {
        return rc;
    }
    const int D = a.kv.head_dim;
    if (!q || !out || !aligned(q, 4) || !aligned(out, 4)) {
        set_error("%s: q and out must be non-null and 4-byte aligned", who);
        return B200Q_EINVAL;
    }
    if (n_head < 1 || n_head > 8192 || n_head % a.kv.n_kv || q_stride < n_head * D || out_stride < n_head * D) {
        set_error("%s: n_head must be a multiple of n_kv (up to 8192), the strides at least n_head * head_dim (n_head=%d n_kv=%d)",
                  who, n_head, a.kv.n_kv);
        return B200Q_EINVAL;
    }
    if ((long long)a.b.max_q * (n_head / a.kv.n_kv) > (1 << 30)) {
        set_error("%s: max_q * n_head / n_kv must not exceed 2^30", who);
        return B200Q_EUNSUPPORTED;
    }
    if (a.b.n_tok == 0) {
        return B200Q_OK;
    }
    if (rows_overlap(q, q_stride, n_head * D, out, out_stride, n_head * D, a.b.n_tok)) {
        set_error("%s: out must not overlap q", who);
        return B200Q_EINVAL;
    }
    float scale = 0.0f;
    if (opts) {
        if (!(opts->scale >= 0.0f) || std::isinf(opts->scale) || opts->window < 0 || opts->n_sink < 0) {
            set_error("%s: scale, window and n_sink must not be negative (scale finite)", who);
            return B200Q_EINVAL;
        }
        scale = opts->scale;
        constexpr int far = 1 << 30; // no key is further; keeps the kernels' differences in 32 bits
        a.window = opts->window < far ? opts->window : far;
        a.n_sink = opts->window ? (opts->n_sink < far ? opts->n_sink : far) : 0;
    }
    const size_t need = b200q_attn_scratch_bytes(n_head, a.kv.n_kv, D, a.b.n_seq, a.b.n_tok, a.b.max_q);
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < need) {
        set_error("%s: scratch must be 16-byte aligned and hold %zu bytes (got %zu)", who, need, scratch_bytes);
        return B200Q_EINVAL;
    }
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n_head = n_head;
    a.group = n_head / a.kv.n_kv;
    if (scale == 0.0f) {
        scale = 1.0f / std::sqrt((float)D);
    }
    a.scale_log2 = (float)((double)scale * 1.4426950408889634 * (double)a.kv.k_scale);
    a.v_scale = a.kv.v_scale;
    a.counters = static_cast<uint32_t *>(scratch);
    a.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + kCounterBytes);
    if ((long long)a.b.max_q * a.group <= kDecodeRows) {
        B200Q_CUDA_OK(launch_attn_decode((cudaStream_t)stream, a));
    } else {
        B200Q_CUDA_OK(launch_attn_prompt((cudaStream_t)stream, a));
    }
    return B200Q_OK;
}

int b200q_kv_copy_pages(void * stream, const b200q_kv_cache * layers, int n_layers, const int32_t * src, const int32_t * dst,
                        int n) {
    const char * who = "b200q_kv_copy_pages";
    if (!layers || n_layers < 1 || n < 0 || (n > 0 && (!src || !dst || !aligned(src, 4) || !aligned(dst, 4)))) {
        set_error("%s: layers, src and dst must be non-null (src and dst 4-byte aligned), n_layers >= 1, n >= 0", who);
        return B200Q_EINVAL;
    }
    KvDev first, d;
    for (int l = 0; l < n_layers; l++) { // all of them before the first launch
        const int rc = check_cache(who, layers + l, l ? d : first);
        if (rc != B200Q_OK) {
            return rc;
        }
        if (l && (d.type != first.type || d.page_bytes != first.page_bytes || d.n_pages != first.n_pages ||
                  d.page_shift != first.page_shift || d.n_kv != first.n_kv || d.head_dim != first.head_dim)) {
            set_error("%s: layer %d differs from the first in more than k and v", who, l);
            return B200Q_EINVAL;
        }
    }
    if (n == 0) {
        return B200Q_OK;
    }
    if (n >= first.n_pages) { // one source may have many copies, but the copies are distinct and none is a source
        set_error("%s: %d copies do not fit a pool of %d pages", who, n, first.n_pages);
        return B200Q_EINVAL;
    }
    if ((long long)n * kv_copy_chunks(first) > INT32_MAX) {
        set_error("%s: too many pages for one call (%d)", who, n);
        return B200Q_EINVAL;
    }
    for (int l0 = 0; l0 < n_layers; l0 += kCopyLayers) {
        const int m = n_layers - l0 < kCopyLayers ? n_layers - l0 : kCopyLayers;
        void * pools[2 * kCopyLayers];
        for (int l = 0; l < m; l++) {
            pools[2 * l] = layers[l0 + l].k;
            pools[2 * l + 1] = layers[l0 + l].v;
        }
        B200Q_CUDA_OK(launch_kv_copy_pages((cudaStream_t)stream, first, pools, 2 * m, src, dst, n));
    }
    return B200Q_OK;
}

int b200q_kv_remap(void * stream, const int32_t * table, int table_stride, int n_seq, int width, const int32_t * map, int n_pages,
                   int32_t * out, int out_stride) {
    const char * who = "b200q_kv_remap";
    if (!table || !map || !out || !aligned(table, 4) || !aligned(map, 4) || !aligned(out, 4) || n_seq < 1 || width < 1 || n_pages < 1 ||
        table_stride < width || out_stride < width) {
        set_error("%s: table, map and out must be non-null and 4-byte aligned, n_seq, width and n_pages >= 1, strides >= width", who);
        return B200Q_EINVAL;
    }
    if (!(table == out && table_stride == out_stride) &&
        rows_overlap(reinterpret_cast<const float *>(table), table_stride, width, reinterpret_cast<const float *>(out), out_stride,
                     width, n_seq)) {
        set_error("%s: out must be table or not overlap it", who);
        return B200Q_EINVAL;
    }
    B200Q_CUDA_OK(launch_kv_remap((cudaStream_t)stream, table, table_stride, n_seq, width, map, n_pages, out, out_stride));
    return B200Q_OK;
}

} // extern "C"
