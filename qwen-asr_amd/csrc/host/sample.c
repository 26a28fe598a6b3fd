/*
 * sample.c - op-level ABI: drawing tokens from logits.  The reference decodes
 * greedily only (qwen_argmax_matvec_bf16, qwen_asr_kernels.h:156).  Neither
 * allocates nor synchronises.
 */
#include "host_internal.h"

#define SAMPLE_MAX_VOCAB (1 << 20)
#define SAMPLE_MAX_ROWS (1 << 16)

size_t qwen_hip_sample_ws_bytes(int rows, int vocab) {
    if (rows <= 0 || rows > SAMPLE_MAX_ROWS || vocab <= 0 || vocab > SAMPLE_MAX_VOCAB) return 0;
    return qk_sample_ws_bytes(rows, vocab);
}

int qwen_hip_sample(int *tokens, const float *logits, long row_stride, int rows, int vocab, const float *temperature,
                    const int *top_k, const float *top_p, const float *min_p, const float *u, void *ws,
                    size_t ws_bytes, hipStream_t s) {
    static const char op[] = "sample";
    if (rows < 0 || rows > SAMPLE_MAX_ROWS || vocab <= 0 || vocab > SAMPLE_MAX_VOCAB)
        QK_REFUSE("%s: %d rows of %d entries (at most %d, %d)", op, rows, vocab, SAMPLE_MAX_ROWS, SAMPLE_MAX_VOCAB);
    if (row_stride < vocab) QK_REFUSE("%s: rows of %d entries %ld apart", op, vocab, row_stride);
    if (rows == 0) return 0;
    if (!tokens || !logits || !u) QK_REFUSE("%s: tokens, logits and u are needed", op);
    const size_t need = qk_sample_ws_bytes(rows, vocab);
    if (!ws || ws_bytes < need || !qk_aligned16(ws))
        QK_REFUSE("%s: workspace of %zu bytes at %p (needs %zu, 16-byte aligned)", op, ws_bytes, ws, need);
    const qk_sample_args a = {.tokens = tokens, .logits = logits, .row_stride = row_stride, .rows = rows,
                              .vocab = vocab, .temperature = temperature, .top_p = top_p, .min_p = min_p, .u = u,
                              .top_k = top_k, .ws = ws};
    QK_TRY(qk_sample_launch(&a, s));
    return 0;
}
