// paged_prefill.hip - causal attention of packed prompts over a paged KV cache:
// row i of a sequence with n new rows and len cached positions (its new rows
// included) sits at position p = len - n + i and sees the positions j <= p:
//
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m = max_j s_j
//
// on v_mfma_f32_32x32x16_bf16, with fp32 statistics and sums.
//
// Operands.  bf16 values go to the matrix cores as they are.  An fp32 value is
// the sum of three bf16 terms, x = h + m + l: h the upper 16 bits, m those of
// x - h, l those of x - h - m; 8 + 8 + 8 significant bits hold all 24, so the split
// is exact.  Products of two such values keep the term pairs (i, j) with i + j <= 2
// (h is term 0): the dropped ones are below 2^-24 of the product.  With fp32
// queries the probabilities are split as well, so such a call is as exact as fp32
// products (3 matrix products a pair on a bf16 cache, 6 on an fp32 one, against
// 16 times the time of one on the fp32 matrix cores).  With bf16 queries the
// probabilities are rounded to bf16 (half a step is 2^-9 of each, as for the
// result itself).
//
// Layout.  Lane l (hl = l >> 5) of the MFMA supplies A[l & 31][8 hl + i] and
// B[8 hl + i][l & 31], i = 0..7, and holds D[8 (r / 4) + 4 hl + r % 4][l & 31],
// r = 0..15.  The rows of a kv head's query heads are flattened, row f = query
// f / G, head f % G, so a few queries of many heads fill a tile as well; a wave
// owns 32 of them, a block 128 of one sequence.  Per tile of 32 keys:
//   S^T = K Q^T      A = K rows from LDS, B = the wave's queries, in registers;
//   softmax          a row lives in the two lanes l, l ^ 32;
//   O^T += V^T P^T   B = the probabilities where S^T left them: k slot 8 hl + i
//                    of step j is key 16 j + 8 (i / 4) + 4 hl + i % 4; A = V^T read
//                    from the row-major V tile by transposing LDS reads (16
//                    lanes take 4 keys x 16 dims and get 4 keys of one dim each).
// LDS rows are 256 bytes, 16-byte chunk c of row r in slot c ^ 2 (r & 7): eight
// rows of a fragment read, and the four rows of a transposing read, meet
// different banks.
//
// bf16 pages go straight to LDS (two buffers); fp32 pages pass through
// registers, split on the way (one buffer a block, two blocks a CU).
//
// Blocks go out longest first; few rows split the keys over blocks, whose
// partials paged_merge joins.
//
// Masked keys: a masked score is -inf before the maximum, but 0 times what the
// cache holds is no number where that is infinite or none.  Rows past the split's
// keys or without a page are read as zeros.  A V row that some rows of a tile see
// and others do not shows in the sums, which stay no number once they are: a
// block that ends with one runs again with every V element looked at, the ones
// that are not finite counted per row that sees them (nothing for the others).
#include "paged.h"

typedef float pp_f32x16 __attribute__((ext_vector_type(16)));
typedef short pp_i16x4 __attribute__((ext_vector_type(4)));

#define PP_ROWS 128               // flattened rows per block
#define PP_KT 32                  // keys per tile
#define PP_PLANE (PP_KT * 256)    // bytes of one term of a K or V tile

__device__ __forceinline__ pp_f32x16 pp_mfma(bf16x8 a, bf16x8 b, pp_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// what a masked or missing key's row is read from
__device__ __attribute__((aligned(256))) unsigned pp_zero_row[PG_HD];

__device__ __forceinline__ void pp_lds_load16(const unsigned char *g, unsigned char *l0) {
    __builtin_amdgcn_global_load_lds(g, l0, 16, 0, 0);
}

// the three terms of two values, each pair in one word (a low)
__device__ __forceinline__ void pp_split2(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
    for (int t = 0; t < 3; t++) {
        const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
        w[t] = __builtin_amdgcn_perm(ub, ua, 0x07060302);          // upper halves
        a -= __uint_as_float(ua & 0xffff0000u);
        b -= __uint_as_float(ub & 0xffff0000u);
    }
}

// NT terms (1: rounded to nearest even) of 8 values as MFMA operands
template <int NT>
__device__ __forceinline__ void pp_terms8(const float *x, bf16x8 (&t)[NT]) {
    if constexpr (NT == 1) {
        t[0] = __builtin_bit_cast(bf16x8, make_uint4(bf16_pack2(x[0], x[1]), bf16_pack2(x[2], x[3]),
                                                     bf16_pack2(x[4], x[5]), bf16_pack2(x[6], x[7])));
    } else {
        uint32_t w[4][3];
#pragma unroll
        for (int i = 0; i < 4; i++) pp_split2(x[2 * i], x[2 * i + 1], w[i]);
#pragma unroll
        for (int k = 0; k < 3; k++) t[k] = __builtin_bit_cast(bf16x8, make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]));
    }
}

// c += sum of the term pairs (i, j), i + j <= 2, small ones first
template <int NA, int NB>
__device__ __forceinline__ pp_f32x16 pp_products(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], pp_f32x16 c) {
#pragma unroll
    for (int sum = (NA == 3 || NB == 3) ? 2 : 0; sum >= 0; sum--)
#pragma unroll
        for (int i = NA - 1; i >= 0; i--)
#pragma unroll
            for (int j = NB - 1; j >= 0; j--)
                if (i + j == sum) c = pp_mfma(a[i], b[j], c);
    return c;
}

// 8 elements of V^T (dims by lane, the lane's 8 keys of step j): two transposing reads
__device__ __forceinline__ bf16x8 pp_vfrag(const unsigned char *p) {
    typedef __attribute__((address_space(3))) pp_i16x4 *lds_p;
    const pp_i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p);
    const pp_i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p + 8 * 256));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The lanes' words with every element that is infinite or no number replaced by
// 0; cls gets 1, 64 or 4096 in the places of +inf, -inf and no number.
__device__ __forceinline__ bf16x8 pp_finite(bf16x8 v, bf16x8 &cls) {
    uint4 w = __builtin_bit_cast(uint4, v), k = make_uint4(0u, 0u, 0u, 0u);
    uint32_t *pw = &w.x, *pk = &k.x;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t e = pw[i] >> (16 * h) & 0xffffu;
            if ((e & 0x7f80u) == 0x7f80u) {
                pk[i] |= (e & 0x7fu ? 0x4580u : e & 0x8000u ? 0x4280u : 0x3f80u) << (16 * h);
                pw[i] &= ~(0xffffu << (16 * h));
            }
        }
    cls = __builtin_bit_cast(bf16x8, k);
    return __builtin_bit_cast(bf16x8, w);
}

template <typename T>
struct PpTerms {
    static constexpr int N = sizeof(T) == 4 ? 3 : 1;
};

template <typename T, typename C>
__global__ __launch_bounds__(256, PpTerms<T>::N == 3 ? 1 : 2) void paged_prefill(qk_paged_attn_args a) {
    constexpr int NQ = PpTerms<T>::N, NK = PpTerms<C>::N;
    constexpr bool DIRECT = NK == 1;
    constexpr int NBUF = DIRECT ? 2 : 1;
    __shared__ __attribute__((aligned(16))) unsigned char lds[NBUF][2][NK][PP_PLANE];
    __shared__ __attribute__((aligned(4))) unsigned char seen_lds[NBUF][4];   // keys of a tile that are there, a bit each

    const qk_paged &pg = a.pg;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, hl = lane >> 5;
    const int G = a.heads / pg.kv_heads;
    const int slots = pg.rows * G / PP_ROWS + pg.n_seqs;      // rows * heads fits an int
    const int slot = slots - 1 - (int)(blockIdx.x / pg.kv_heads), kvh = blockIdx.x % pg.kv_heads;
    // Tiles of sequence s take the slots from start_s G / 128 + s on: ceil(n G / 128)
    // never passes the next sequence's first.
    auto begin = [&](int s) { return min(max(pg.row_start[s], 0), pg.rows); };
    auto first_slot = [&](int s) { return begin(s) * G / PP_ROWS + s; };
    const int s = __builtin_amdgcn_readfirstlane(pg_search<64>(pg.n_seqs, slot, first_slot));
    if (s < 0) return;
    const int r0 = begin(s), n = max(begin(s + 1) - r0, 0);
    const int f0 = (slot - first_slot(s)) * PP_ROWS, frows = n * G;
    if (f0 >= frows) return;                              // block-uniform, as all above
    const int len = pg_len(pg, s);
    const int off0 = len - n;                      // position of the sequence's first new row (< 0: sees nothing)
    const int lastf = min(f0 + PP_ROWS, frows) - 1;
    const int kend = min(max(off0 + lastf / G + 1, 0), pg.capacity);
    const int need = (int)(((long)kend + a.nsplit - 1) / a.nsplit);
    const int chunk = max(a.chunk, (need + PP_KT - 1) / PP_KT * PP_KT), split = blockIdx.y;
    const int k0s = (int)min((long)split * chunk, (long)kend), k1 = (int)min((long)k0s + chunk, (long)kend);

    // this lane's row
    const int f = f0 + 32 * wave + ql;
    const bool on = f < frows;
    const int qi = on ? f / G : 0, head = kvh * G + (on ? f % G : 0);
    const size_t orow = (size_t)(r0 + qi) * a.heads + head;
    const int pos = on ? off0 + qi : -1;
    if (k0s >= k1 && a.nsplit > 1) {
        if (on && hl == 0) {
            float *ml = a.part_ml + 2 * (orow * a.nsplit + split);
            ml[0] = -INFINITY;
            ml[1] = 0.0f;
        }
        return;
    }
    // the wave's first and last positions (rows do not fall with f)
    const int fw = f0 + 32 * wave;
    const bool wave_on = fw < frows;
    const int pos_lo = off0 + fw / G, pos_hi = off0 + min(fw + 31, frows - 1) / G;

    // queries: dims 16 t + 8 hl .. + 7; fp32 ones take the scale along
    bf16x8 q[8][NQ];
#pragma unroll
    for (int t = 0; t < 8; t++) {
        const T *qp = (const T *)a.q + orow * PG_HD + 16 * t + 8 * hl;
        if constexpr (NQ == 1) {
            q[t][0] = *reinterpret_cast<const bf16x8 *>(qp);
        } else {
            const float4 x0 = pg_load4(qp), x1 = pg_load4(qp + 4);
            const float fs = a.scale * PG_LOG2E;
            const float x[8] = {x0.x * fs, x0.y * fs, x0.z * fs, x0.w * fs, x1.x * fs, x1.y * fs, x1.z * fs, x1.w * fs};
            pp_terms8<NQ>(x, q[t]);
        }
    }
    const float sc = NQ == 1 ? a.scale * PG_LOG2E : 1.0f;

    pp_f32x16 o[4];
    float m, l;

    // ---- staging: the wave's 8 rows of a tile; a lane's rows RPL of them -------------
    constexpr int RPL = DIRECT ? 2 : 4;
    const int srow0 = DIRECT ? lane >> 4 : lane >> 5;     // row 8 wave + RSTEP i + srow0
    constexpr int RSTEP = DIRECT ? 4 : 2;
    int pid[RPL];
    auto ids = [&](int k0) {
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const int key = k0 + 8 * wave + RSTEP * i + srow0;
            pid[i] = key < k1 ? pg_page(pg, s, key) : -1;
        }
    };
    auto seen_byte = [&]() {
        unsigned b = 0;
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const unsigned long long v = __ballot(pid[i] >= 0);
#pragma unroll
            for (int j = 0; j < RSTEP; j++) b |= (unsigned)(v >> (64 / RSTEP * j) & 1) << (RSTEP * i + j);
        }
        return b;
    };
    float4 stk[DIRECT ? 1 : 4], stv[DIRECT ? 1 : 4];
    unsigned st_seen = 0;
    // bf16: K and V rows to buffer buf; fp32: to registers
    auto fetch = [&](int k0, int buf) {
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const int r = 8 * wave + RSTEP * i + srow0;
            const size_t off = pid[i] >= 0 ? pg_offset(pg, pid[i], kvh, k0 + r) : 0;
            if constexpr (DIRECT) {
                const int byte = 16 * ((lane & 15) ^ (2 * (r & 7)));
                const unsigned char *z = (const unsigned char *)pp_zero_row;
                const unsigned char *kr = pid[i] >= 0 ? (const unsigned char *)((const C *)pg.k + off) : z;
                const unsigned char *vr = pid[i] >= 0 ? (const unsigned char *)((const C *)pg.v + off) : z;
                pp_lds_load16(kr + byte, &lds[buf][0][0][256 * (8 * wave + RSTEP * i)]);
                pp_lds_load16(vr + byte, &lds[buf][1][0][256 * (8 * wave + RSTEP * i)]);
            } else {
                const float *kr = pid[i] >= 0 ? (const float *)pg.k + off : (const float *)pp_zero_row;
                const float *vr = pid[i] >= 0 ? (const float *)pg.v + off : (const float *)pp_zero_row;
                stk[i] = pg_load4(kr + 4 * ql);
                stv[i] = pg_load4(vr + 4 * ql);
            }
        }
        const unsigned b = seen_byte();
        if constexpr (DIRECT) {
            if (lane == 0) seen_lds[buf][wave] = (unsigned char)b;
        } else {
            st_seen = b;
        }
    };
    // fp32: the terms of the staged rows to LDS
    auto put = [&]() {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < RPL; i++) {
                const int r = 8 * wave + RSTEP * i + srow0;
                const int at = 256 * r + 16 * ((ql >> 1) ^ (2 * (r & 7))) + 8 * (ql & 1);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float4 v = x ? stv[i] : stk[i];
                    uint32_t w0[3], w1[3];
                    pp_split2(v.x, v.y, w0);
                    pp_split2(v.z, v.w, w1);
                    // the terms below an infinite one (or none) are 0, not inf - inf
                    const float z = fmaf(v.x, 0.0f, fmaf(v.y, 0.0f, fmaf(v.z, 0.0f, v.w * 0.0f)));
                    if (z != 0.0f) {
                        auto fix = [](uint32_t hw, uint32_t w) {
                            const uint32_t lo = (hw & 0x7f80u) == 0x7f80u ? 0u : 0xffffu;
                            const uint32_t hi = (hw & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
                            return w & (lo | hi);
                        };
#pragma unroll
                        for (int t = 1; t < 3; t++) {
                            w0[t] = fix(w0[0], w0[t]);
                            w1[t] = fix(w1[0], w1[t]);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < 3; t++)
                        *reinterpret_cast<uint2 *>(&lds[0][x][t][at]) = make_uint2(w0[t], w1[t]);
                }
            }
            if (lane == 0) seen_lds[0][wave] = (unsigned char)st_seen;
        }
    };

    // ---- fragment addresses ----------------------------------------------------------
    const int ksw = 2 * (ql & 7);                         // K row ql: chunk 2 t + hl in slot (2 t + hl) ^ ksw
    const int vrow = 4 * hl + ((lane & 15) >> 2);         // V row of this lane's transposing reads (mod 8)
    const int vchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vbyte = 256 * vrow + 8 * (lane & 1);
    auto vaddr = [&](int buf, int t, int d, int j) {
        return &lds[buf][1][t][vbyte + 16 * ((4 * d + vchunk) ^ (2 * (vrow & 7))) + 16 * 256 * j];
    };

    bool guarded = false;
    for (;;) {
#pragma unroll
    for (int d = 0; d < 4; d++) o[d] = (pp_f32x16){};
    m = -INFINITY;
    l = 0.0f;
    ids(k0s);
    fetch(k0s, 0);
    ids(k0s + PP_KT);
    int buf = 0;
    for (int k0 = k0s; k0 < k1; k0 += PP_KT) {
        if constexpr (DIRECT) {
            __builtin_amdgcn_s_waitcnt(0x0f70);           // this wave's rows are in LDS
            __syncthreads();                              // everyone's are, and the other buffer is read
            if (k0 + PP_KT < k1) {
                fetch(k0 + PP_KT, buf ^ 1);
                ids(k0 + 2 * PP_KT);
            }
        } else {
            __syncthreads();                              // the last tile is read
            put();
            __syncthreads();
            if (k0 + PP_KT < k1) {
                fetch(k0 + PP_KT, 0);
                ids(k0 + 2 * PP_KT);
            }
        }
        if (wave_on && k0 <= pos_hi) {
            pp_f32x16 st = {};
#pragma unroll
            for (int t = 0; t < 8; t++) {
                bf16x8 kf[NK];
#pragma unroll
                for (int x = 0; x < NK; x++)
                    kf[x] = *reinterpret_cast<const bf16x8 *>(&lds[buf][0][x][256 * ql + 16 * ((2 * t + hl) ^ ksw)]);
                st = pp_products<NK, NQ>(kf, q[t], st);
            }
            const unsigned seen = *reinterpret_cast<const unsigned *>(seen_lds[buf]);
            const bool open = seen == 0xffffffffu && k0 + PP_KT - 1 <= pos_lo;    // wave-uniform
            if (!open) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = 8 * (r / 4) + 4 * hl + r % 4;
                    if (!((seen >> key) & 1) || k0 + key > pos) st[r] = -INFINITY;
                }
            }
            float mx = st[0];
#pragma unroll
            for (int r = 1; r < 16; r++) mx = fmaxf(mx, st[r]);
            float other = mx;
            swap32(mx, other);
            const float mn = fmaxf(m, fmaxf(mx, other) * sc), ref = pg_ref(mn);
            const float corr = __builtin_amdgcn_exp2f(m - ref);
            m = mn;
            float p[16], sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(st[r], sc, -ref));
                sum += p[r];
            }
            l = fmaf(l, corr, sum);
            if (!__all(corr == 1.0f)) {
#pragma unroll
                for (int d = 0; d < 4; d++) o[d] *= corr;
            }
            bf16x8 pt[2][NQ];
            pp_terms8<NQ>(p, pt[0]);
            pp_terms8<NQ>(p + 8, pt[1]);
            if (!guarded) {
#pragma unroll
                for (int d = 0; d < 4; d++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        bf16x8 vf[NK];
#pragma unroll
                        for (int x = 0; x < NK; x++) vf[x] = pp_vfrag(vaddr(buf, x, d, j));
                        o[d] = pp_products<NK, NQ>(vf, pt[j], o[d]);
                    }
            } else {
                // finite values as ever, and how many infinite ones (and ones that are no
                // number) each row sees, counted on the matrix cores: + 1, 64 or 4096
                // each, at most 32 of them
                bf16x8 one[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = p[8 * j + i] > 0.0f ? 1.0f : 0.0f;
                    bf16x8 t[1];
                    pp_terms8<1>(x, t);
                    one[j] = t[0];
                }
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    pp_f32x16 cnt = {};
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        bf16x8 vf[NK], cls;
#pragma unroll
                        for (int x = NK - 1; x >= 0; x--) vf[x] = pp_finite(pp_vfrag(vaddr(buf, x, d, j)), cls);
                        o[d] = pp_products<NK, NQ>(vf, pt[j], o[d]);
                        cnt = pp_mfma(cls, one[j], cnt);
                        __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int k = (int)cnt[r], pi = k & 63, ni = k >> 6 & 63;
                        if (k >= 4096 || (pi && ni)) o[d][r] = NAN;
                        else if (k) o[d][r] += pi ? INFINITY : -INFINITY;
                    }
                }
            }
        }
        if constexpr (DIRECT) buf ^= 1;
    }
    if (guarded) break;
    float z = 0.0f;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) z = fmaf(o[d][r], 0.0f, z);
    if (!__syncthreads_or(z != 0.0f)) break;              // 0 times what is infinite or no number is none
    guarded = true;
    }
    if (!wave_on) return;

    float lo_ = l, hi_ = l;
    swap32(lo_, hi_);
    const float L = lo_ + hi_;
    if (!on) return;
    if (a.nsplit == 1) {
        // 0 only where no key was seen: the largest p is 1
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        T *dst = (T *)a.out + orow * PG_HD + 4 * hl;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                pg_store4(dst + 32 * d + 2 * r, make_float4(o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv));
    } else {
        const size_t at = orow * a.nsplit + split;
        float *dst = a.part_o + at * PG_HD + 4 * hl;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4 *>(dst + 32 * d + 2 * r) = make_float4(o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
        if (hl == 0) {
            a.part_ml[2 * at] = m;
            a.part_ml[2 * at + 1] = L;
        }
    }
}

extern "C" void qk_paged_prefill_plan(int rows, int n_seqs, int heads, int kv_heads, int max_len, int *nsplit,
                                      int *chunk) {
    const long tiles = (long)rows * (heads / kv_heads) / PP_ROWS + n_seqs;
    const long blocks = tiles * kv_heads;
    long n = (512 + blocks - 1) / blocks;
    if (n > QK_PAGED_MAX_SPLIT) n = QK_PAGED_MAX_SPLIT;
    long c = (max_len + n - 1) / n;
    c = (c + 63) / 64 * 64;
    if (c < 64) c = 64;
    n = (max_len + c - 1) / c;
    *nsplit = n < 1 ? 1 : (int)n;
    *chunk = (int)c;
}

extern "C" int qk_paged_prefill_launch(const qk_paged_attn_args *a, hipStream_t s) {
    const long slots = (long)a->pg.rows * (a->heads / a->pg.kv_heads) / PP_ROWS + a->pg.n_seqs;
    if (slots * a->pg.kv_heads > 0x7fffffffL) return QWEN_HIP_EINVAL;
    const dim3 grid((unsigned)(slots * a->pg.kv_heads), (unsigned)a->nsplit);
    if (a->act_bf16) {
        if (a->pg.cache_bf16) paged_prefill<uint16_t, uint16_t><<<grid, 256, 0, s>>>(*a);
        else paged_prefill<uint16_t, float><<<grid, 256, 0, s>>>(*a);
    } else {
        if (a->pg.cache_bf16) paged_prefill<float, uint16_t><<<grid, 256, 0, s>>>(*a);
        else paged_prefill<float, float><<<grid, 256, 0, s>>>(*a);
    }
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
