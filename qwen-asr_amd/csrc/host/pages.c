/*
 * pages.c - op-level ABI: page tables of sequences that continue others, copies of
 * pages in all layers, accepted drafts that move up, and the choice of the best
 * continuations of a sequence's beams.  No counterpart in the reference (one
 * stream, greedy decoding, one contiguous cache).  Nothing here allocates or
 * synchronises.
 */
#include "host_internal.h"

#include <limits.h>

#define BEAM_MAX_VOCAB (1 << 20)
#define BEAM_MAX_ROWS (1 << 16)

/* n bytes at a and m at b */
static int overlap_bytes(const void *a, size_t n, const void *b, size_t m) {
    return a && b && (uintptr_t)a < (uintptr_t)b + m && (uintptr_t)b < (uintptr_t)a + n;
}

/* n values at a and m at b, 4 bytes each */
static int overlap(const void *a, size_t n, const void *b, size_t m) { return overlap_bytes(a, 4 * n, b, 4 * m); }

/* the cache's shape, checked; its sequences as ones of a row each */
static int shape(const char *op, const qwen_hip_paged_kv *kv, qk_paged *p) {
    const qwen_hip_paged_batch none = {0};
    if (!kv) QK_REFUSE("%s: no cache", op);
    qwen_hip_paged_kv one = *kv;
    one.n_seqs = 0;
    const int rc = qk_paged_view(op, &one, &none, kv->kv_heads, kv->dtype, p);
    if (rc) return rc;
    if (kv->n_seqs < 0) QK_REFUSE("%s: n_seqs %d", op, kv->n_seqs);
    p->n_seqs = kv->n_seqs;
    return 0;
}

/* layers of one shape, checked, in the kernels' form */
static int layers_view(const char *op, const qwen_hip_paged_kv *layers, int n, qk_paged_layers *L) {
    if (!layers || n <= 0 || n > QK_PAGED_MAX_LAYERS) QK_REFUSE("%s: %d layers at %p (1 .. %d)", op, n, (const void *)layers, QK_PAGED_MAX_LAYERS);
    qk_paged p;
    const int rc = shape(op, layers, &p);
    if (rc) return rc;
    for (int i = 0; i < n; i++) {
        const qwen_hip_paged_kv *a = layers + i;
        if (a->dtype != layers->dtype || a->n_pages != layers->n_pages || a->page_size != layers->page_size ||
            a->kv_heads != layers->kv_heads || a->head_dim != layers->head_dim)
            QK_REFUSE("%s: layer %d has another shape than the first", op, i);
        if (!a->k || !a->v || !qk_aligned16(a->k) || !qk_aligned16(a->v))
            QK_REFUSE("%s: the pages of layer %d are NULL or not 16-byte aligned", op, i);
        L->k[i] = a->k;
        L->v[i] = a->v;
    }
    L->n_layers = n;
    L->n_pages = p.n_pages;
    L->page_shift = p.page_shift;
    L->kv_heads = p.kv_heads;
    L->row_bytes = QWEN_HIP_HEAD_DIM * (p.cache_bf16 ? 2 : 4);
    return 0;
}

size_t qwen_hip_paged_fork_ws_bytes(const qwen_hip_paged_kv *kv, int n_out) {
    qk_paged p;
    if (n_out <= 0 || n_out > QK_PAGED_FORK_ROWS || shape("paged_fork_ws_bytes", kv, &p)) return 0;
    return qk_paged_fork_ws_bytes(p.n_pages);
}

int qwen_hip_paged_fork(const qwen_hip_paged_kv *kv, const int *kv_len, const int *parent, const int *new_rows,
                        const unsigned char *outside, int n_out, int *table_out, int *len_out, int *copies, int *missing,
                        void *ws, size_t ws_bytes, hipStream_t s) {
    static const char op[] = "paged_fork";
    qk_paged p;
    const int rc = shape(op, kv, &p);
    if (rc) return rc;
    if (n_out < 0 || n_out > QK_PAGED_FORK_ROWS) QK_REFUSE("%s: %d rows (at most %d)", op, n_out, QK_PAGED_FORK_ROWS);
    if (!parent && n_out != p.n_seqs) QK_REFUSE("%s: without parents row s continues row s (%d rows of %d)", op, n_out, p.n_seqs);
    if (n_out == 0) return 0;
    if (p.n_seqs > 0 && (!p.table || !kv_len)) QK_REFUSE("%s: no table or no lengths", op);
    if (!table_out || !len_out || !copies || !missing) QK_REFUSE("%s: an output is NULL", op);
    if (!qk_aligned16(copies)) QK_REFUSE("%s: copies is not 16-byte aligned", op);
    const size_t in = (size_t)p.n_seqs * p.table_stride, out = (size_t)n_out * p.table_stride;
    if (out > INT_MAX) QK_REFUSE("%s: %d rows of %d page ids", op, n_out, p.table_stride);
    if (overlap(table_out, out, p.table, in) || overlap(len_out, n_out, kv_len, p.n_seqs))
        QK_REFUSE("%s: the new table or lengths overlap the old ones", op);
    const size_t need = qk_paged_fork_ws_bytes(p.n_pages);
    if (need > 0 && (!ws || ws_bytes < need || !qk_aligned16(ws)))
        QK_REFUSE("%s: workspace of %zu bytes at %p (needs %zu, 16-byte aligned)", op, ws_bytes, ws, need);
    /* what one thread writes another may read later; of lengths in the place of parents or new rows it is the same one */
    const struct {
        const void *at;
        size_t n;
    } outs[] = {{table_out, out}, {len_out, n_out}, {copies, 4 * (size_t)n_out}, {missing, 1}};
    for (int i = 0; i < 4; i++) {
        const int own = i == 1;
        if (overlap_bytes(outs[i].at, 4 * outs[i].n, outside, p.n_pages) || overlap(outs[i].at, outs[i].n, p.table, in) ||
            overlap(outs[i].at, outs[i].n, kv_len, p.n_seqs) ||
            (!(own && outs[i].at == parent) && overlap(outs[i].at, outs[i].n, parent, n_out)) ||
            (!(own && outs[i].at == new_rows) && overlap(outs[i].at, outs[i].n, new_rows, n_out)))
            QK_REFUSE("%s: an output overlaps an input", op);
    }
    const qk_paged_fork_args a = {.table = p.table, .kv_len = kv_len, .parent = parent, .new_rows = new_rows,
                                  .outside = outside, .table_out = table_out, .len_out = len_out, .copies = copies,
                                  .missing = missing, .n_in = p.n_seqs, .n_out = n_out, .stride = p.table_stride,
                                  .page_shift = p.page_shift, .n_pages = p.n_pages, .ws = (unsigned *)ws};
    QK_TRY(qk_paged_fork_launch(&a, s));
    return 0;
}

int qwen_hip_paged_copy(const qwen_hip_paged_kv *layers, int n_layers, const int *copies, int n_copies, hipStream_t s) {
    static const char op[] = "paged_copy";
    qk_paged_layers L;
    const int rc = layers_view(op, layers, n_layers, &L);
    if (rc) return rc;
    if (n_copies < 0) QK_REFUSE("%s: %d copies", op, n_copies);
    if (n_copies == 0) return 0;
    if (!copies || !qk_aligned16(copies)) QK_REFUSE("%s: copies is NULL or not 16-byte aligned", op);
    QK_TRY(qk_paged_copy_launch(&L, copies, n_copies, s));
    return 0;
}

int qwen_hip_paged_compact(const qwen_hip_paged_kv *layers, int n_layers, const qwen_hip_paged_batch *batch, int *len_out,
                           const int *path, long path_stride, const int *n_path, hipStream_t s) {
    static const char op[] = "paged_compact";
    qk_paged_layers L;
    qk_paged p;
    int rc = layers_view(op, layers, n_layers, &L);
    if (rc) return rc;
    if ((rc = qk_paged_view(op, layers, batch, layers->kv_heads, layers->dtype, &p))) return rc;
    for (int i = 1; i < n_layers; i++)
        if (layers[i].table != layers->table || layers[i].n_seqs != layers->n_seqs || layers[i].table_stride != layers->table_stride)
            QK_REFUSE("%s: layer %d has another table than the first", op, i);
    if (path_stride <= 0) QK_REFUSE("%s: path_stride %ld", op, path_stride);
    if (p.n_seqs == 0) return 0;
    if (!p.table || !p.kv_len || !len_out || !path || !n_path) QK_REFUSE("%s: a pointer is NULL", op);
    if (overlap(len_out, p.n_seqs, p.kv_len, p.n_seqs)) QK_REFUSE("%s: the new lengths overlap the old ones", op);
    /* every layer's blocks read what the first one's would write over */
    if (overlap(len_out, p.n_seqs, n_path, p.n_seqs) || overlap(len_out, p.n_seqs, p.row_start, (size_t)p.n_seqs + 1) ||
        overlap(len_out, p.n_seqs, p.table, (size_t)p.n_seqs * p.table_stride) ||
        overlap(len_out, p.n_seqs, path, (size_t)(p.n_seqs - 1) * path_stride + (path_stride < p.rows ? path_stride : p.rows)))
        QK_REFUSE("%s: the new lengths overlap an input", op);
    QK_TRY(qk_paged_compact_launch(&L, &p, len_out, path, path_stride, n_path, s));
    return 0;
}

static int beam_shape(int seqs, int beams, int vocab, int n_out) {
    return seqs >= 0 && beams > 0 && beams <= QK_BEAM_MAX && (long)seqs * beams <= BEAM_MAX_ROWS && vocab > 0 &&
           vocab <= BEAM_MAX_VOCAB && n_out > 0 && n_out <= QK_BEAM_MAX;
}

size_t qwen_hip_beam_select_ws_bytes(int seqs, int beams, int vocab, int n_out) {
    return beam_shape(seqs, beams, vocab, n_out) && seqs > 0 ? qk_beam_ws_bytes(seqs, beams, vocab, n_out) : 0;
}

int qwen_hip_beam_select(int *parent, int *token, float *score_out, const void *logits, int dtype, long row_stride,
                         int seqs, int beams, int vocab, const float *score, const int *ended, int n_out, void *ws,
                         size_t ws_bytes, hipStream_t s) {
    static const char op[] = "beam_select";
    if (!beam_shape(seqs, beams, vocab, n_out))
        QK_REFUSE("%s: %d sequences of %d beams, %d entries, %d places (beams and places at most %d, rows %d, entries %d)", op,
                  seqs, beams, vocab, n_out, QK_BEAM_MAX, BEAM_MAX_ROWS, BEAM_MAX_VOCAB);
    if (dtype != QWEN_HIP_ST_F32 && dtype != QWEN_HIP_ST_BF16) QK_REFUSE("%s: logits of type %d", op, dtype);
    if (row_stride < vocab) QK_REFUSE("%s: rows of %d entries %ld apart", op, vocab, row_stride);
    if (seqs == 0) return 0;
    if (!parent || !token || !score_out || !logits || !score) QK_REFUSE("%s: a pointer is NULL", op);
    if ((uintptr_t)logits % (dtype == QWEN_HIP_ST_F32 ? 4 : 2)) QK_REFUSE("%s: the logits are not aligned to their type", op);
    const size_t rows = (size_t)seqs * beams, places = (size_t)seqs * n_out;
    if (overlap(parent, places, score, rows) || overlap(parent, places, ended, rows) || overlap(token, places, score, rows) ||
        overlap(token, places, ended, rows) || overlap(score_out, places, score, rows) || overlap(score_out, places, ended, rows))
        QK_REFUSE("%s: an output overlaps score or ended", op);
    const size_t need = qk_beam_ws_bytes(seqs, beams, vocab, n_out);
    if (!ws || ws_bytes < need || !qk_aligned16(ws))
        QK_REFUSE("%s: workspace of %zu bytes at %p (needs %zu, 16-byte aligned)", op, ws_bytes, ws, need);
    const qk_beam_args a = {.parent = parent, .token = token, .score_out = score_out, .logits = logits,
                            .bf16 = dtype == QWEN_HIP_ST_BF16, .row_stride = row_stride, .seqs = seqs, .beams = beams,
                            .vocab = vocab, .n_out = n_out, .score = score, .ended = ended, .ws = ws};
    QK_TRY(qk_beam_launch(&a, s));
    return 0;
}
