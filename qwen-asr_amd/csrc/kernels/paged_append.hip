// paged_append.hip - new rows enter a paged KV cache: per-head RMS norm of
// queries and keys, rotation by their positions, keys and values stored into
// the sequences' pages, in one pass over the rows.
//
//   x^ = x / sqrt(mean(x^2) + eps) * w         (where w is given)
//   (x^[d], x^[d + 64]) -> (x^[d] c - x^[d + 64] s, x^[d + 64] c + x^[d] s),
//   c, s = cos, sin[position][d], d = 0..63
//
// or, where the rows say by which position they turn (drafts of one depth alike, wherever they sit), of that one.
// Everything in fp32, rounded once to the type it is stored in.  Bound by the
// bytes it moves (rows in, queries and pages out) for many rows, by the chain
// row -> sequence -> length -> page id -> store for one.
//
// Sixteen lanes own one head of one row (4 + 4 dims a lane, whole rotation
// pairs), 16 heads a block.  The row's values do not depend on where it goes:
// their loads are issued before the search for its sequence.
//
// Measured: 8 prompts of 101 to 1515 rows, bf16, 16 heads over 8: 16 us for 76 MB, the
// rate of a device copy (4.8 TB/s); one row: 2.3 us.
#include "paged.h"

template <typename T>
struct PgAppend {
    qk_paged pg;
    T *q_out;
    const T *q, *k, *v;
    long q_stride, kv_stride;
    int heads;
    const float *q_norm, *k_norm, *cos_v, *sin_v;
    float eps;
    int n_pos;
    const int *rope_pos;
};

template <typename T, typename C>
__global__ __launch_bounds__(256) void paged_append(PgAppend<T> a) {
    const qk_paged &pg = a.pg;
    const int c = threadIdx.x & 15, nh = a.heads + pg.kv_heads;
    const long units = (long)nh * pg.rows;
    const long u = 16L * blockIdx.x + (threadIdx.x >> 4);
    // groups past the end stay for the search's ballots
    const bool on = u < units;
    const int row = on ? (int)(u / nh) : 0, head = on ? (int)(u % nh) : 0;
    const bool is_q = head < a.heads;
    const int kvh = head - a.heads;
    const T *src = is_q ? a.q + (size_t)row * a.q_stride + head * PG_HD
                        : a.k + (size_t)row * a.kv_stride + kvh * PG_HD;
    float4 lo = pg_load4(src + 4 * c), hi = pg_load4(src + 64 + 4 * c), vl = {}, vh = {};
    if (!is_q) {
        const T *vs = a.v + (size_t)row * a.kv_stride + kvh * PG_HD;
        vl = pg_load4(vs + 4 * c);
        vh = pg_load4(vs + 64 + 4 * c);
    }
    const float *nw = is_q ? a.q_norm : a.k_norm;
    float4 wl, wh;
    if (nw) {
        wl = pg_load4(nw + 4 * c);
        wh = pg_load4(nw + 64 + 4 * c);
    }
    // drafts of one depth turn alike, wherever they sit
    const int turn = a.rope_pos ? a.rope_pos[row] : 0;
    int s = row, start = row, stop = row + 1;
    if (pg.row_start) {
        s = pg_search<16>(pg.n_seqs, row, [&](int i) { return (long)pg.row_start[i]; });
        if (s >= 0) {
            start = pg.row_start[s];
            stop = pg.row_start[s + 1];
        }
    }
    // rows before the first or behind the last sequence are left as they are
    if (!on || s < 0 || s >= pg.n_seqs || row >= stop) return;
    const long p = (long)pg_len(pg, s) - ((long)stop - row);
    const long by = a.rope_pos ? (long)turn : p;
    if (p < 0 || p >= pg.capacity || by < 0 || by >= a.n_pos) return;
    const int pos = (int)p;
    const int pid = is_q ? 0 : pg_page(pg, s, pos);
    float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.cos_v) {
        c4 = pg_load4(a.cos_v + (size_t)by * PG_HD + 4 * c);
        s4 = pg_load4(a.sin_v + (size_t)by * PG_HD + 4 * c);
    }
    if (nw) {
        norm_rope_row16(lo, hi, wl, wh, c4, s4, a.eps);
    } else if (a.cos_v) {
        const float4 x = lo, y = hi;
        lo = make_float4(fmaf(x.x, c4.x, -(y.x * s4.x)), fmaf(x.y, c4.y, -(y.y * s4.y)),
                         fmaf(x.z, c4.z, -(y.z * s4.z)), fmaf(x.w, c4.w, -(y.w * s4.w)));
        hi = make_float4(fmaf(y.x, c4.x, x.x * s4.x), fmaf(y.y, c4.y, x.y * s4.y), fmaf(y.z, c4.z, x.z * s4.z),
                         fmaf(y.w, c4.w, x.w * s4.w));
    }
    if (is_q) {
        T *dst = a.q_out + ((size_t)row * a.heads + head) * PG_HD;
        pg_store4(dst + 4 * c, lo);
        pg_store4(dst + 64 + 4 * c, hi);
    } else if (pid >= 0) {
        const size_t o = pg_offset(pg, pid, kvh, pos);
        C *kd = (C *)pg.k + o, *vd = (C *)pg.v + o;
        pg_store4(kd + 4 * c, lo);
        pg_store4(kd + 64 + 4 * c, hi);
        pg_store4(vd + 4 * c, vl);
        pg_store4(vd + 64 + 4 * c, vh);
    }
}

template <typename T>
static int append_launch(const qk_paged_append_args *x, hipStream_t s) {
    const PgAppend<T> a = {x->pg, (T *)x->q_out, (const T *)x->q, (const T *)x->k, (const T *)x->v, x->q_stride,
                           x->kv_stride, x->heads, x->q_norm, x->k_norm, x->cos_v, x->sin_v, x->eps, x->n_pos,
                           x->rope_pos};
    const long blocks = ((long)(x->heads + x->pg.kv_heads) * x->pg.rows + 15) / 16;
    if (blocks > 0x7fffffffL) return QWEN_HIP_EINVAL;
    if (x->pg.cache_bf16) paged_append<T, uint16_t><<<(unsigned)blocks, 256, 0, s>>>(a);
    else paged_append<T, float><<<(unsigned)blocks, 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}

extern "C" int qk_paged_append_launch(const qk_paged_append_args *a, hipStream_t s) {
    return a->act_bf16 ? append_launch<uint16_t>(a, s) : append_launch<float>(a, s);
}
