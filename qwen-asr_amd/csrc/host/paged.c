/*
 * paged.c - op-level ABI of the paged KV cache: appending rows, attention of
 * single tokens and of packed prompts, over all positions, over a window, of
 * drafted trees.  No counterpart in the reference, which keeps one contiguous
 * cache for one stream (qwen_asr_decoder.c:122-160).
 *
 * Host checks cover everything the host can see (types, shapes, alignment,
 * the workspace's size).  Lengths, row starts and page ids are device data:
 * the kernels clamp them.  Nothing here allocates or synchronises.
 */
#include "host_internal.h"

#include <float.h>
#include <limits.h>
#include <math.h>

#define MAX_CAPACITY (1L << 30)   /* positions of one sequence */

static int is_dtype(int t) { return t == QWEN_HIP_ST_F32 || t == QWEN_HIP_ST_BF16; }

/* the cache and the batch, checked, in the kernels' form */
int qk_paged_view(const char *op, const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *b, int heads, int dtype,
                  qk_paged *p) {
    if (!kv || !b) QK_REFUSE("%s: no cache or no batch", op);
    if (!is_dtype(kv->dtype) || !is_dtype(dtype))
        QK_REFUSE("%s: types are QWEN_HIP_ST_F32 or QWEN_HIP_ST_BF16 (rows %d, cache %d)", op, dtype, kv->dtype);
    if (kv->head_dim != QWEN_HIP_HEAD_DIM) QK_REFUSE("%s: head_dim %d (only %d)", op, kv->head_dim, QWEN_HIP_HEAD_DIM);
    if (kv->page_size <= 0 || kv->page_size > (1 << 24) || (kv->page_size & (kv->page_size - 1)))
        QK_REFUSE("%s: page_size %d is no power of two up to 2^24", op, kv->page_size);
    if (kv->n_pages <= 0 || kv->kv_heads <= 0 || kv->n_seqs < 0 || kv->table_stride <= 0)
        QK_REFUSE("%s: n_pages %d, kv_heads %d, n_seqs %d, table_stride %d", op, kv->n_pages, kv->kv_heads, kv->n_seqs,
               kv->table_stride);
    /* 2^31 rows of 128 values are more than any memory holds */
    if ((double)kv->n_pages * kv->kv_heads * kv->page_size > (double)INT_MAX)
        QK_REFUSE("%s: %d pages of %d positions and %d kv heads", op, kv->n_pages, kv->page_size, kv->kv_heads);
    if (heads <= 0 || heads % kv->kv_heads) QK_REFUSE("%s: %d heads over %d kv heads", op, heads, kv->kv_heads);
    if (b->rows < 0 || b->max_len < 0) QK_REFUSE("%s: rows %d, max_len %d", op, b->rows, b->max_len);
    if ((long)b->rows * heads > INT_MAX / QWEN_HIP_HEAD_DIM) QK_REFUSE("%s: %d rows of %d heads", op, b->rows, heads);
    if ((long)kv->n_seqs * kv->kv_heads > INT_MAX / 2) QK_REFUSE("%s: %d sequences of %d kv heads", op, kv->n_seqs, kv->kv_heads);
    if (!b->row_start && b->rows != kv->n_seqs)
        QK_REFUSE("%s: without row_start a sequence has one row (%d rows, %d sequences)", op, b->rows, kv->n_seqs);
    int shift = 0;
    while ((1 << shift) < kv->page_size) shift++;
    const long cap = (long)kv->table_stride << shift;
    *p = (qk_paged){.k = kv->k, .v = kv->v, .table = kv->table, .row_start = b->row_start, .kv_len = b->kv_len,
                    .cache_bf16 = kv->dtype == QWEN_HIP_ST_BF16, .n_pages = kv->n_pages, .page_shift = shift,
                    .kv_heads = kv->kv_heads, .n_seqs = kv->n_seqs, .table_stride = kv->table_stride,
                    .rows = b->rows, .capacity = (int)(cap < MAX_CAPACITY ? cap : MAX_CAPACITY)};
    return 0;
}

/* no row is a sequence's: nothing to launch, nothing to plan (a plan divides by the blocks of its sequences) */
static int no_call(const qk_paged *p) { return p->rows == 0 || p->n_seqs == 0; }

/* ... and the pointers that a call with rows reads */
static int paged_pointers(const char *op, const qk_paged *p) {
    if (!p->k || !p->v || !p->table || !p->kv_len) QK_REFUSE("%s: a pointer of the cache or the batch is NULL", op);
    if (!qk_aligned16(p->k) || !qk_aligned16(p->v)) QK_REFUSE("%s: the pages are not 16-byte aligned", op);
    return 0;
}

static int append(const char *op, const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, const int *rope_pos,
                  void *q_out, const void *q, const void *k, const void *v, int dtype, long q_stride, long kv_stride,
                  int heads, const float *q_norm, const float *k_norm, float eps, const float *cos_vals,
                  const float *sin_vals, int n_pos, hipStream_t s) {
    qk_paged_append_args a = {0};
    const int rc = qk_paged_view(op, kv, batch, heads, dtype, &a.pg);
    if (rc) return rc;
    const int unit = dtype == QWEN_HIP_ST_F32 ? 4 : 8;
    if (q_stride < (long)heads * QWEN_HIP_HEAD_DIM || kv_stride < (long)kv->kv_heads * QWEN_HIP_HEAD_DIM ||
        q_stride % unit || kv_stride % unit)
        QK_REFUSE("%s: row strides %ld, %ld (at least a row, multiples of 16 bytes)", op, q_stride, kv_stride);
    if (!q_norm != !k_norm || !cos_vals != !sin_vals) QK_REFUSE("%s: one norm or one rotation table of two", op);
    if (q_norm && !(eps >= 0.0f && eps <= FLT_MAX)) QK_REFUSE("%s: eps %g", op, (double)eps);
    if (n_pos < 0) QK_REFUSE("%s: n_pos %d", op, n_pos);
    if (no_call(&a.pg)) return 0;
    if (paged_pointers(op, &a.pg)) return QWEN_HIP_EINVAL;
    if (!q_out || !q || !k || !v) QK_REFUSE("%s: a pointer of the rows is NULL", op);
    if (!qk_aligned16(q_out) || !qk_aligned16(q) || !qk_aligned16(k) || !qk_aligned16(v) || !qk_aligned16(q_norm) ||
        !qk_aligned16(k_norm) || !qk_aligned16(cos_vals) || !qk_aligned16(sin_vals))
        QK_REFUSE("%s: a pointer is not 16-byte aligned", op);
    if (q_out == q && q_stride != (long)heads * QWEN_HIP_HEAD_DIM)
        QK_REFUSE("%s: in place the queries' rows are %d values apart", op, heads * QWEN_HIP_HEAD_DIM);
    a.q_out = q_out;
    a.q = q;
    a.k = k;
    a.v = v;
    a.act_bf16 = dtype == QWEN_HIP_ST_BF16;
    a.heads = heads;
    /* without a table no position is out of it */
    a.n_pos = cos_vals ? n_pos : INT_MAX;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.cos_v = cos_vals;
    a.sin_v = sin_vals;
    a.eps = eps;
    a.rope_pos = cos_vals ? rope_pos : NULL;
    QK_TRY(qk_paged_append_launch(&a, s));
    return 0;
}

int qwen_hip_paged_append(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, void *q_out, const void *q,
                          const void *k, const void *v, int dtype, long q_stride, long kv_stride, int heads,
                          const float *q_norm, const float *k_norm, float eps, const float *cos_vals,
                          const float *sin_vals, int n_pos, hipStream_t s) {
    return append("paged_append", kv, batch, NULL, q_out, q, k, v, dtype, q_stride, kv_stride, heads, q_norm, k_norm, eps,
                  cos_vals, sin_vals, n_pos, s);
}

int qwen_hip_paged_append_at(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, const int *rope_pos,
                             void *q_out, const void *q, const void *k, const void *v, int dtype, long q_stride,
                             long kv_stride, int heads, const float *q_norm, const float *k_norm, float eps,
                             const float *cos_vals, const float *sin_vals, int n_pos, hipStream_t s) {
    static const char op[] = "paged_append_at";
    if (kv && batch && kv->n_seqs > 0 && batch->rows > 0 && (!rope_pos || !cos_vals))
        QK_REFUSE("%s: no rotation positions or no rotation tables", op);
    return append(op, kv, batch, rope_pos, q_out, q, k, v, dtype, q_stride, kv_stride, heads, q_norm, k_norm, eps,
                  cos_vals, sin_vals, n_pos, s);
}

/*
 * Whether single tokens run on the matrix cores, as prompts of one row do: where many heads share
 * a bf16 cache's rows, the vector units are what bounds the other kernel.  Microseconds, vector
 * kernel against matrix kernel, 8 kv heads, 24 sequences of 500 to 6001 positions:
 *   bf16 rows, 2 heads a kv head: 49, 66; 4: 59, 66; 8: 98, 66; 16: 141, 67
 *   fp32 rows (split into three terms), 4: 59, 89; 8: 98, 89; 16: 141, 90
 * and of 131 to 530: bf16 rows, 2: 13, 16; 4: 16, 16; 5: 23, 16; fp32 rows, 4: 15, 19; 8: 23, 20.
 * fp32 pages take the matrix kernel longer throughout (8 heads: 108, 234).
 */
static int tokens_by_matrix(int cache_bf16, int group) { return cache_bf16 && group > 4; }

enum { ALL, WINDOW, TREE };
typedef struct {
    int kind, window, sinks;
} seen_keys;

/*
 * splits of an attention call and the workspace it needs.  The plans split into at most
 * ceil(T / blocks) for a number T of blocks that they aim at, and not at all from T blocks on.  A
 * block has up to R rows of heads, so rows x heads x splits is at most R blocks (T + blocks - 1) / blocks
 * < 2 R T: for prompts 2 x 128 x 384, for single tokens 2 x 8 x 2048 (fewer heads a block: as many).
 * Of masks the splits are at most T / blocks: 128 x 512, and 64 x 768 with blocks of 64 rows.
 * Times 520 bytes, that is below QWEN_HIP_PAGED_ATTENTION_WS_MAX for any batch.
 */
static size_t attention_plan(const qk_paged *p, seen_keys seen, int matrix, int heads, int max_len, int *rows2, int *nsplit,
                             int *chunk) {
    if (max_len == 0 || max_len > p->capacity) max_len = p->capacity;
    const int all = max_len;
    if (seen.kind == WINDOW) {
        /* what a block walks at most, about: the window and the first positions, and of packed rows as many
         * positions more as a block has rows, and tiles that are seen in part */
        const long most = (long)seen.window + seen.sinks + (matrix ? 128 * p->kv_heads / heads + 62 : 0);
        if (most < max_len) max_len = (int)most;
    }
    *rows2 = 0;
    if (!matrix) qk_paged_decode_plan(p->n_seqs, heads, p->kv_heads, p->cache_bf16, max_len, nsplit, chunk);
    else if (seen.kind == ALL) *rows2 = qk_paged_prefill_plan(p, heads, max_len, nsplit, chunk);
    /* a window is filled early in sequences of more than 1.5 times what is walked (4 x 100 to 700 rows, fp32, up to 1200
     * positions, 642 walked: even 66 us, else 90; 24 x 4 to 8 rows, up to 6000, 4126 walked: 71, 69) */
    else *rows2 = qk_paged_masked_plan(p, seen.kind == TREE, seen.kind == WINDOW && all > 1.5 * max_len, heads, max_len, nsplit, chunk);
    if (*nsplit == 1) return 0;
    return (size_t)p->rows * heads * *nsplit * (QWEN_HIP_HEAD_DIM + 2) * sizeof(float);
}

static int by_matrix(const qk_paged *p, seen_keys seen, int heads) {
    return seen.kind == TREE || p->row_start || tokens_by_matrix(p->cache_bf16, heads / p->kv_heads);
}

size_t qwen_hip_paged_attention_ws_bytes(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, int heads) {
    qk_paged p;
    int rows2, nsplit, chunk;
    if (qk_paged_view("paged_attention_ws_bytes", kv, batch, heads, QWEN_HIP_ST_F32, &p) || no_call(&p)) return 0;
    const seen_keys all = {ALL, 0, 0};
    return attention_plan(&p, all, by_matrix(&p, all, heads), heads, batch->max_len, &rows2, &nsplit, &chunk);
}

/* rows: single tokens, packed ones, or either */
enum { TOKENS, PACKED, EITHER };

static int attention(const char *op, int kind, seen_keys seen, const uint64_t *tree, int words, const qwen_hip_paged_kv *kv,
                     const qwen_hip_paged_batch *batch, void *out, const void *q, int dtype, int heads, float scale,
                     void *ws, size_t ws_bytes, hipStream_t s) {
    qk_paged_attn_args a = {0};
    const int rc = qk_paged_view(op, kv, batch, heads, dtype, &a.pg);
    if (rc) return rc;
    if (kind == PACKED && !batch->row_start) QK_REFUSE("%s: no row_start", op);
    if (kind == TOKENS && batch->row_start) QK_REFUSE("%s: one row per sequence: row_start has to be NULL", op);
    if (!(scale >= 1e-30f && scale <= 1e30f)) QK_REFUSE("%s: scale %g", op, (double)scale);
    if (no_call(&a.pg)) return 0;
    if (paged_pointers(op, &a.pg)) return QWEN_HIP_EINVAL;
    if (!out || !q) QK_REFUSE("%s: a pointer of the rows is NULL", op);
    if (!qk_aligned16(out) || !qk_aligned16(q)) QK_REFUSE("%s: the rows are not 16-byte aligned", op);
    if (out == q) QK_REFUSE("%s: out cannot be q", op);
    if (seen.kind == TREE && !tree) QK_REFUSE("%s: no tree", op);
    const int matrix = by_matrix(&a.pg, seen, heads);
    const size_t need = attention_plan(&a.pg, seen, matrix, heads, batch->max_len, &a.rows2, &a.nsplit, &a.chunk);
    if (need > 0 && (!ws || ws_bytes < need || !qk_aligned16(ws)))
        QK_REFUSE("%s: workspace of %zu bytes at %p (needs %zu, 16-byte aligned)", op, ws_bytes, ws, need);
    a.out = out;
    a.q = q;
    a.act_bf16 = dtype == QWEN_HIP_ST_BF16;
    a.heads = heads;
    a.scale = scale;
    a.window = seen.window;
    a.sinks = seen.sinks;
    /* little-endian: bit i of a row is bit i % 32 of its 32-bit word i / 32 */
    a.tree = (const uint32_t *)tree;
    a.tree_words = 2 * words;
    a.part_o = (float *)ws;
    a.part_ml = need ? a.part_o + (size_t)a.pg.rows * heads * a.nsplit * QWEN_HIP_HEAD_DIM : NULL;
    if (matrix) QK_TRY(qk_paged_prefill_launch(&a, s));
    else QK_TRY(qk_paged_decode_launch(&a, s));
    if (need) QK_TRY(qk_paged_merge_launch(&a, s));
    return 0;
}

int qwen_hip_paged_attention_decode(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, void *out,
                                    const void *q, int dtype, int heads, float scale, void *ws, size_t ws_bytes,
                                    hipStream_t s) {
    const seen_keys all = {ALL, 0, 0};
    return attention("paged_attention_decode", TOKENS, all, NULL, 0, kv, batch, out, q, dtype, heads, scale, ws, ws_bytes, s);
}

int qwen_hip_paged_attention_prefill(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, void *out,
                                     const void *q, int dtype, int heads, float scale, void *ws, size_t ws_bytes,
                                     hipStream_t s) {
    const seen_keys all = {ALL, 0, 0};
    return attention("paged_attention_prefill", PACKED, all, NULL, 0, kv, batch, out, q, dtype, heads, scale, ws, ws_bytes, s);
}

/* a window of more positions than a length can name, and more first positions than a table holds, are as good as those */
static int first_positions(int sinks) { return sinks < MAX_CAPACITY ? sinks : (int)MAX_CAPACITY; }

size_t qwen_hip_paged_attention_window_ws_bytes(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, int heads,
                                                int window, int sinks) {
    qk_paged p;
    int rows2, nsplit, chunk;
    if (window <= 0 || sinks < 0 ||
        qk_paged_view("paged_attention_window_ws_bytes", kv, batch, heads, QWEN_HIP_ST_F32, &p) || no_call(&p))
        return 0;
    const seen_keys seen = {WINDOW, window, first_positions(sinks)};
    return attention_plan(&p, seen, by_matrix(&p, seen, heads), heads, batch->max_len, &rows2, &nsplit, &chunk);
}

int qwen_hip_paged_attention_window(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, void *out,
                                    const void *q, int dtype, int heads, float scale, int window, int sinks, void *ws,
                                    size_t ws_bytes, hipStream_t s) {
    static const char op[] = "paged_attention_window";
    if (window <= 0 || sinks < 0) QK_REFUSE("%s: a window of %d positions, %d first ones", op, window, sinks);
    const seen_keys seen = {WINDOW, window, first_positions(sinks)};
    return attention(op, EITHER, seen, NULL, 0, kv, batch, out, q, dtype, heads, scale, ws, ws_bytes, s);
}

size_t qwen_hip_paged_attention_tree_ws_bytes(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, int heads) {
    qk_paged p;
    int rows2, nsplit, chunk;
    if (qk_paged_view("paged_attention_tree_ws_bytes", kv, batch, heads, QWEN_HIP_ST_F32, &p) || no_call(&p)) return 0;
    const seen_keys seen = {TREE, 0, 0};
    return attention_plan(&p, seen, 1, heads, batch->max_len, &rows2, &nsplit, &chunk);
}

int qwen_hip_paged_attention_tree(const qwen_hip_paged_kv *kv, const qwen_hip_paged_batch *batch, void *out, const void *q,
                                  int dtype, int heads, float scale, const uint64_t *tree, int words, void *ws,
                                  size_t ws_bytes, hipStream_t s) {
    static const char op[] = "paged_attention_tree";
    if (words <= 0 || words > QK_TREE_WORDS / 2) QK_REFUSE("%s: %d words of bits a row (1 .. %d)", op, words, QK_TREE_WORDS / 2);
    if ((uintptr_t)tree % 8) QK_REFUSE("%s: the tree is not 8-byte aligned", op);
    const seen_keys seen = {TREE, 0, 0};
    return attention(op, EITHER, seen, tree, words, kv, batch, out, q, dtype, heads, scale, ws, ws_bytes, s);
}
