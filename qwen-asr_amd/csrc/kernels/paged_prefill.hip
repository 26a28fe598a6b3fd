// paged_prefill.hip - causal attention of packed prompts over a paged KV cache:
// row i of a sequence with n new rows and len cached positions (its new rows
// included) sits at position p = len - n + i and sees the positions j <= p:
//
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m = max_j s_j
//
// on v_mfma_f32_32x32x16_bf16, with fp32 statistics and sums.
//
// Operands.  bf16 values go to the matrix cores as they are.  An fp32 value is
// the sum of three bf16 terms, x = h + m + l: h is x rounded to nearest, m what is left
// of x rounded so, l what is left then, which has no more than 8 bits: the split
// is exact.  Products of two such values keep the term pairs (i, j) with i + j <= 2
// (h is term 0): m is at most 2^-8 and l 2^-17 of the value's power of two, so the
// dropped ones are below 2^-24 of the product, of either sign (terms that are cut off
// instead of rounded drop up to 2^-21, always towards 0).  With fp32
// queries the probabilities are split as well, so such a call is as exact as fp32
// products (3 matrix products a pair on a bf16 cache, 6 on an fp32 one, against
// 16 times the time of one on the fp32 matrix cores).  With bf16 queries the
// probabilities are held in two terms (2^-17 of them), and
// so are fp32 values (the upper two of their three): one term alone is off by as much as
// the result's own rounding, 1.3 to 1.4 times the error of an fp32 softmax rounded once
// (8191 rows: 0.0021 and 0.0016 of the result's norm; 306 us with one, 392 with two).
//
// Layout.  Lane l (hl = l >> 5) of the MFMA supplies A[l & 31][8 hl + i] and
// B[8 hl + i][l & 31], i = 0..7, and holds D[8 (r / 4) + 4 hl + r % 4][l & 31],
// r = 0..15.  The rows of a kv head's query heads are flattened, row f = query
// f / G, head f % G, so a few queries of many heads fill a tile as well; a wave
// owns 32 of them, a block 64 or 128 of one sequence.  Per tile of 32 keys:
//   S^T = K Q^T      A = K rows from LDS, B = the wave's queries, in registers;
//   softmax          a row lives in the two lanes l, l ^ 32;
//   O^T += V^T P^T   B = the probabilities where S^T left them: k slot 8 hl + i
//                    of step j is key 16 j + 8 (i / 4) + 4 hl + i % 4; A = V^T read
//                    from the row-major V tile by transposing LDS reads (16
//                    lanes take 4 keys x 16 dims and get 4 keys of one dim each).
// LDS rows are 256 bytes, their 16-byte chunks in an order by row (swz) that
// keeps both kinds of reads free of bank conflicts.
//
// A block is two groups of waves, every other tile of keys each, joined in LDS at the
// end: groups of four (128 rows), or of two (64 rows) where that is the faster (see the
// plan).  The second group runs half a turn behind the first, so that with four waves
// each SIMD has one wave's products beside another's softmax; of 64-row blocks a CU
// runs two.  bf16 pages go straight to LDS (two buffers a group); fp32 pages pass
// through registers, split on the way.
//
// Blocks go out longest first; few rows split the keys over blocks, whose
// partials paged_merge joins.
//
// Measured (8 kv heads, 2 heads each; the card's large bf16 product: 1290 TFLOP/s):
//   one prompt of 8191 rows, bf16: 392 us, the causal half's products (three for two, by the
//     probabilities' second term) at 1050 TFLOP/s; bound by them and the softmax beside them
//     (with one term, in 306 us, tiles staged through registers took 1.24 times the time; 64
//     rows a wave, one wave a SIMD: 2.1; three buffers, loads among the products: 1.20)
//   8 prompts of 101 to 1515 rows, fp32 rows on a bf16 cache (three products for one): 71 to 81 us;
//     bound by the products, and by what a block does before and behind them
//     (about 11 us of its 31: tile search, first tiles, join)
//   the same on fp32 pages (six products for one; more than 64 rows a sequence: about 50 registers
//     spill): 159 us; bf16 rows on fp32 pages (three for one): 82 us
//   31 new rows behind 993, all fp32: 19.6 to 20.7 us, a chain of first loads and the join's launch
//
// Masked keys: a masked score is -inf before the maximum, but 0 times what the
// cache holds is no number where that is infinite or none.  Such a V
// element shows in the sums, which stay no number once they are: a block that
// ends with one runs again with every V element looked at, the ones that are not
// finite counted per row that sees them (nothing for the others).
#include "paged.h"
#include "ring.h"

#include <limits.h>

typedef float pp_f32x16 __attribute__((ext_vector_type(16)));
typedef short pp_i16x4 __attribute__((ext_vector_type(4)));

#define PP_KT 32                  // keys per tile
#define PP_PLANE (PP_KT * 256)    // bytes of one term of a K or V tile

__device__ __forceinline__ pp_f32x16 pp_mfma(bf16x8 a, bf16x8 b, pp_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 16 bytes a lane from global memory straight into LDS (lane l at byte 16 l of the
// 1 KB at l0): base + off, base the same for the wave.  Written out because the
// compiler lets every transposing LDS read wait for all such loads on their way,
// also those to the other buffer; the walk's barriers wait for them instead.
// They write no register but m0, which the compiler sets anew before each use, and
// its own counts of loads only become stricter by ones that it does not see.
__device__ __forceinline__ void pp_lds_load16(const unsigned char *base, unsigned off, unsigned char *l0) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)l0;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(off), "s"(base), "s"(at) : "memory");
}
// ... from an address of each lane's own
__device__ __forceinline__ void pp_lds_load16(const unsigned char *p, unsigned char *l0) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)l0;
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(p), "s"(at) : "memory");
}

// the three terms of two values, each pair in one word (a low).  ANY: the largest values would round to an
// infinite h, so it ends at the largest bf16; then m says what the value is, infinite or no number as that
#define PP_BF16_MAX 0x1.fep127f
template <bool ANY>
__device__ __forceinline__ void pp_split2(float a, float b, uint32_t (&w)[3]) {
    if constexpr (ANY) w[0] = bf16_pack2(__builtin_amdgcn_fmed3f(a, -PP_BF16_MAX, PP_BF16_MAX),
                                         __builtin_amdgcn_fmed3f(b, -PP_BF16_MAX, PP_BF16_MAX));
    else w[0] = bf16_pack2(a, b);
    a -= bf16_lo(w[0]);
    b -= bf16_hi(w[0]);
    w[1] = bf16_pack2(a, b);
    a -= bf16_lo(w[1]);
    b -= bf16_hi(w[1]);
    w[2] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);      // upper halves: all that is left
}

// NT terms of 8 values as MFMA operands: 1, rounded to nearest even; 2, each rounded so, x to 2^-17; 3, x itself
template <int NT, bool ANY = false>
__device__ __forceinline__ void pp_terms8(const float *x, bf16x8 (&t)[NT]) {
    if constexpr (NT == 1) {
        t[0] = __builtin_bit_cast(bf16x8, make_uint4(bf16_pack2(x[0], x[1]), bf16_pack2(x[2], x[3]),
                                                     bf16_pack2(x[4], x[5]), bf16_pack2(x[6], x[7])));
    } else if constexpr (NT == 2) {
        uint4 hi, lo;
        bf16_split2(x[0], x[1], hi.x, lo.x);
        bf16_split2(x[2], x[3], hi.y, lo.y);
        bf16_split2(x[4], x[5], hi.z, lo.z);
        bf16_split2(x[6], x[7], hi.w, lo.w);
        t[0] = __builtin_bit_cast(bf16x8, hi);
        t[1] = __builtin_bit_cast(bf16x8, lo);
    } else {
        uint32_t w[4][3];
#pragma unroll
        for (int i = 0; i < 4; i++) pp_split2<ANY>(x[2 * i], x[2 * i + 1], w[i]);
#pragma unroll
        for (int k = 0; k < 3; k++) t[k] = __builtin_bit_cast(bf16x8, make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]));
    }
}

// The term pairs (i, j) of a product of NA by NB terms, small ones first: i + j <= 2, or <= 1 where B is
// held in two terms
template <int NA, int NB>
struct PpPairs {
    static constexpr int MOST = NB == 2 ? 1 : 2;
    static constexpr int count() {
        int n = 0;
        for (int i = 0; i < NA; i++)
            for (int j = 0; j < NB; j++) n += i + j <= MOST;
        return n;
    }
    static constexpr int N = count();
    struct List {
        int a[N], b[N];
    };
    static constexpr List make() {
        List l = {};
        int n = 0;
        for (int sum = MOST; sum >= 0; sum--)
            for (int i = NA - 1; i >= 0; i--)
                for (int j = NB - 1; j >= 0; j--)
                    if (i + j == sum) {
                        l.a[n] = i;
                        l.b[n++] = j;
                    }
        return l;
    }
};

template <int NA, int NB>
__device__ __forceinline__ pp_f32x16 pp_products(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], pp_f32x16 c) {
    constexpr auto L = PpPairs<NA, NB>::make();
#pragma unroll
    for (int n = 0; n < PpPairs<NA, NB>::N; n++) c = pp_mfma(a[L.a[n]], b[L.b[n]], c);
    return c;
}

// 8 elements of V^T (dims by lane, the lane's 8 keys of step j): two transposing reads
__device__ __forceinline__ bf16x8 pp_vfrag(const unsigned char *p, const unsigned char *p8) {
    typedef __attribute__((address_space(3))) pp_i16x4 *lds_p;
    const pp_i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p);
    const pp_i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p8);
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

// v with 0 in the places that cls says something of
__device__ __forceinline__ bf16x8 pp_cleared(bf16x8 v, bf16x8 cls) {
    uint4 w = __builtin_bit_cast(uint4, v), k = __builtin_bit_cast(uint4, cls);
    uint32_t *pw = &w.x, *pk = &k.x;
#pragma unroll
    for (int i = 0; i < 4; i++) pw[i] &= (pk[i] & 0xffffu ? 0u : 0xffffu) | (pk[i] >> 16 ? 0u : 0xffff0000u);
    return __builtin_bit_cast(bf16x8, w);
}

template <bool B>
struct PpBool {
    static constexpr bool value = B;
};

template <typename T>
struct PpTerms {
    static constexpr int N = sizeof(T) == 4 ? 3 : 1;
};

// A block: WR waves over the rows, 32 each, and KG groups of such waves over the keys (tiles in turn,
// joined in LDS).
#define PP_KG 2
#define PP_ROWS(WR) (32 * (WR))
#define PP_THREADS(WR) (64 * (WR) * PP_KG)

// First row of sequence i (i = n_seqs: the end of the last); without row_start each has one
__device__ __forceinline__ int pp_begin(const qk_paged &pg, int i) {
    return pg.row_start ? min(max(pg.row_start[i], 0), pg.rows) : i;
}

// The tile of block `b`: its sequence s with rows r0 .. r0 + n - 1 and len cached positions, and
// its first flattened row f0 (a whole wave asks).  Longest first over up to 64 sequences: a tile's
// level is its last position in steps of 128 keys, and tiles go out by falling level, so the ones
// that take longest start first.  For more sequences, by sequence from the last: tiles of
// sequence s take the slots from start_s G / ROWS + s on (ceil(n G / ROWS) of them never pass the
// next sequence's first).
struct PpTile {
    int s, f0, r0, n, len;
};
template <int ROWS>
__device__ __forceinline__ bool pp_tile(const qk_paged &pg, int G, int b, int slots, PpTile &o) {
    const int lane = threadIdx.x & 63;
    auto begin = [&](int i) { return pp_begin(pg, i); };
    auto take = [&](int s) {
        o.s = s;
        o.r0 = begin(s);
        o.n = max(begin(s + 1) - o.r0, 0);
        o.len = pg_len(pg, s);
    };
    if (pg.n_seqs > 64) {
        const int slot = slots - 1 - b;
        auto first_slot = [&](int i) { return begin(i) * G / ROWS + i; };
        const int s = __builtin_amdgcn_readfirstlane(pg_search<64>(pg.n_seqs, slot, first_slot));
        if (s < 0) return false;
        take(s);
        o.f0 = (slot - (o.r0 * G / ROWS + s)) * ROWS;
        return o.f0 >= 0;
    }
    if (pg.n_seqs == 1) {
        take(0);
        o.f0 = ((o.n * G + ROWS - 1) / ROWS - 1 - b) * ROWS;
        return o.f0 >= 0;
    }
    const int i = min(lane, pg.n_seqs - 1), r0 = begin(i), end = begin(i + 1), len = pg_len(pg, i);
    const bool on = lane < pg.n_seqs;
    const int n = on ? max(end - r0, 0) : 0;
    const int tiles = (n * G + ROWS - 1) / ROWS, off = on ? min(max(len - n, 0), pg.capacity) : 0;
    // tiles of this lane's sequence at level t or above; counts fit a float exactly
    auto first_at = [&](int t) {
        const long want = ((long)t * 128 - off) * G;
        return (int)min(max((want + ROWS - 1) / ROWS - 1, 0L), (long)tiles);
    };
    auto sum_at = [&](int t) { return (int)wave_sum((float)(tiles - first_at(t))); };
    if (b >= sum_at(0)) return false;
    int lo = 0, hi = (int)wave_max(on && n > 0 ? (float)((off + n + ROWS) / 128 + 2) : 0.0f);
    while (hi - lo > 1) {                        // sum_at(lo) > b >= sum_at(hi)
        const int mid = (lo + hi) >> 1;
        if (sum_at(mid) > b) lo = mid;
        else hi = mid;
    }
    const int left = b - sum_at(lo + 1), from = first_at(lo), mine = first_at(lo + 1) - from;
    int upto = mine;                             // inclusive sum over the lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(upto, d, 64);
        if (lane >= d) upto += v;
    }
    const unsigned long long past = __ballot(upto > left);
    o.s = __builtin_amdgcn_readfirstlane(past ? __builtin_ctzll(past) : 0);
    o.f0 = __builtin_amdgcn_readlane(from + left - (upto - mine), o.s) * ROWS;
    o.r0 = __builtin_amdgcn_readlane(r0, o.s);
    o.n = __builtin_amdgcn_readlane(n, o.s);
    o.len = __builtin_amdgcn_readlane(len, o.s);
    return past != 0 && o.f0 >= 0;
}

// SMALL: pages that do not hold a wave's rows of a tile (fewer than 8 positions).  Two waves a SIMD, but for
// 64-row blocks on fp32 pages, which LDS lets only one of onto a CU.
template <typename T, typename C, bool SMALL, int WR>
__global__ __launch_bounds__(PP_THREADS(WR), sizeof(C) == 4 && WR == 2 ? 1 : 2) void paged_prefill(qk_paged_attn_args a, int slots) {
    // terms of the queries, the keys, the probabilities, the values
    constexpr int NQ = PpTerms<T>::N, NK = PpTerms<C>::N, NP = NQ == 1 ? 2 : NQ, NV = NQ == 1 && NK == 3 ? 2 : NK;
    constexpr int KG = PP_KG, ROWS = PP_ROWS(WR);
    constexpr bool DIRECT = NK == 1;
    constexpr int NBUF = DIRECT ? 2 : 1;
    constexpr int STAGE = 2 * NK * PP_PLANE;              // bytes of one K and V tile
    constexpr int JOIN = (KG - 1) * WR * (16384 + 512);
    constexpr int BYTES = KG * NBUF * STAGE > JOIN ? KG * NBUF * STAGE : JOIN;
    __shared__ __attribute__((aligned(1024))) unsigned char lds_all[BYTES];

    const qk_paged &pg = a.pg;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = wid % WR, kg = wid / WR;
    const int ql = lane & 31, hl = lane >> 5;
    const int G = a.heads / pg.kv_heads, kvh = blockIdx.x % pg.kv_heads;
    PpTile tile;
    if (!pp_tile<ROWS>(pg, G, (int)(blockIdx.x / pg.kv_heads), slots, tile)) return;      // block-uniform, as the next
    const int s = __builtin_amdgcn_readfirstlane(tile.s), f0 = __builtin_amdgcn_readfirstlane(tile.f0),
              r0 = __builtin_amdgcn_readfirstlane(tile.r0), n = __builtin_amdgcn_readfirstlane(tile.n),
              len = __builtin_amdgcn_readfirstlane(tile.len);
    const int frows = n * G;
    if (f0 >= frows) return;
    const int off0 = len - n;                             // position of the sequence's first new row (< 0: sees nothing)
    const int lastf = min(f0 + ROWS, frows) - 1;
    const int kend = min(max(off0 + lastf / G + 1, 0), pg.capacity);
    const int need = (int)(((long)kend + a.nsplit - 1) / a.nsplit);
    const int chunk = max(a.chunk, (need + PP_KT - 1) / PP_KT * PP_KT), split = blockIdx.y;
    const int k0s = (int)min((long)split * chunk, (long)kend), k1 = (int)min((long)k0s + chunk, (long)kend);

    // this lane's row
    const int fw = f0 + 32 * wave, f = fw + ql;
    const bool on = f < frows, wave_on = fw < frows;
    const int qi = on ? f / G : 0, pos = on ? off0 + qi : -1;
    const size_t orow = (size_t)(r0 + qi) * a.heads + kvh * G + (on ? f % G : 0);
    if (k0s >= k1 && a.nsplit > 1) {
        if (on && hl == 0 && kg == 0) {
            float *ml = a.part_ml + 2 * (orow * a.nsplit + split);
            ml[0] = -INFINITY;
            ml[1] = 0.0f;
        }
        return;
    }
    const int pos_lo = off0 + fw / G;                     // the wave's first position (rows do not fall with f)

    bf16x8 q[8][NQ];
    const float sc = NQ == 1 ? a.scale * PG_LOG2E : 1.0f;
    pp_f32x16 o[4];
    float m, l;

    // ---- staging: the group's waves take SROWS rows of its tile each; a lane's rows RPL of them ----
    constexpr int SROWS = PP_KT / WR, RSTEP = DIRECT ? 4 : 2, RPL = SROWS / RSTEP;
    constexpr int ROWB = PG_HD * sizeof(C);
    const int srow0 = DIRECT ? lane >> 4 : lane >> 5;     // row SROWS wave + RSTEP i + srow0
    unsigned char *const lds = lds_all + kg * NBUF * STAGE;
    auto plane = [&](int buf, int v, int t) { return lds + buf * STAGE + (v * NK + t) * PP_PLANE; };
    // The slot of row r's chunk 0: 16 rows of a K fragment read meet the 16 16-byte slots of
    // the banks' 256 bytes, and so do the 64-byte pieces of four rows of a transposing read.
    auto swz = [](int r) { return 4 * (r & 3) + ((r >> 2) & 3); };
    const int smask = (1 << pg.page_shift) - 1;
    const int *const table = pg.table + (size_t)s * pg.table_stride;
    auto tile_k0 = [&](int t) { return k0s + PP_KT * (KG * t + kg); };
    // Where the wave's rows of tile t lie, and which of its keys are there.  Pages of at least
    // SROWS positions hold the wave's rows in one page (the tiles start at multiples of 32): one
    // offset from the pages' start, without vector arithmetic.  Rows past the split's end are
    // read at its last key (any row does: their scores are masked), rows without a page from the
    // first page's start.  The page ids come 64 tiles at a time, a lane each: ones that were loaded
    // every turn would be waited for behind the tiles' loads.  Smaller pages: a lane a key, and
    // that wait.
    const size_t pstride = ((size_t)pg.kv_heads << pg.page_shift) * ROWB;
    const unsigned char *const pages[2] = {(const unsigned char *)pg.k + ((size_t)kvh << pg.page_shift) * ROWB,
                                           (const unsigned char *)pg.v + ((size_t)kvh << pg.page_shift) * ROWB};
    constexpr int PIECES = PP_KT / SROWS;                 // parts of a tile that are in one page each
    int own_ids = 0, keys_there = 0, ids_at = INT_MIN / 2; // of tiles ids_at + lane: the wave's rows' page, Where.seen
    auto refill = [&](int t) {
        ids_at = t;
        const long kt = min(k0s + (long)PP_KT * (KG * (t + lane) + kg), (long)k1);
        const int left = k1 - (int)kt;
        int id[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; i++) id[i] = table[min((int)kt + SROWS * i, k1 - 1) >> pg.page_shift];
        unsigned there = 0;
        own_ids = 0;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const bool page = (unsigned)id[i] < (unsigned)pg.n_pages;
            there |= page ? ((1u << SROWS) - 1) << (SROWS * i) : 0u;
            if (i == wave && page) own_ids = id[i];
        }
        keys_there = (int)(there & (left >= PP_KT ? ~0u : (1u << left) - 1));
    };
    struct Where {
        size_t off;
        int id;                                           // SMALL: of key lane % 32
        unsigned seen;                                    // keys that are there, a bit each
    };
    auto where = [&](int t) {
        Where w = {};
        if constexpr (SMALL) {
            const int left = k1 - tile_k0(t);
            w.id = table[min(tile_k0(t) + ql, k1 - 1) >> pg.page_shift];
            w.seen = left >= PP_KT ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
            w.seen &= (unsigned)__ballot((unsigned)w.id < (unsigned)pg.n_pages);
        } else {
            if (t - ids_at >= 64) refill(t);
            const int at = min(tile_k0(t) + SROWS * wave, k1 - 1) & smask;
            w.off = __builtin_amdgcn_readlane(own_ids, t - ids_at) * pstride + (size_t)at * ROWB;
            w.seen = (unsigned)__builtin_amdgcn_readlane(keys_there, t - ids_at);
        }
        return w;
    };
    // this lane's row i of tile t at its wave's offset: of_wave(base, bytes); or at its own
    auto row_of = [&](int t, const Where &w, int v, int i, auto of_wave, auto of_lane) {
        const int key0 = tile_k0(t) + SROWS * wave, r = RSTEP * i + srow0;
        if constexpr (!SMALL) {
            of_wave(pages[v] + w.off, (unsigned)min(r, max(k1 - 1 - key0, 0)) * ROWB);
        } else {
            const int at = min(key0 + r, k1 - 1), i1 = __shfl(w.id, SROWS * wave + r, 64);
            of_lane(pages[v] + ((unsigned)i1 < (unsigned)pg.n_pages ? i1 : 0) * pstride + (unsigned)(at & smask) * ROWB);
        }
    };
    // bf16: straight to the K (v 0) or V (v 1) rows of buffer buf
    auto fetch_row = [&](int t, const Where &w, int v, int buf, int i) {
        const unsigned chunk = 16u * ((lane & 15) ^ swz(SROWS * wave + RSTEP * i + srow0));
        unsigned char *const to = plane(buf, v, 0) + 256 * (SROWS * wave + RSTEP * i);
        row_of(t, w, v, i, [&](const unsigned char *p, unsigned at) { pp_lds_load16(p, at + chunk, to); },
               [&](const unsigned char *row) { pp_lds_load16(row + chunk, to); });
    };
    auto fetch = [&](int t, const Where &w, int v, int buf) {
#pragma unroll
        for (int i = 0; i < RPL; i++) fetch_row(t, w, v, buf, i);
    };
    // fp32: to registers, and from there split into terms
    auto load = [&](int t, const Where &w, int v, float4 (&st)[RPL]) {
#pragma unroll
        for (int i = 0; i < RPL; i++)
            row_of(t, w, v, i,
                   [&](const unsigned char *p, unsigned at) { st[i] = pg_load4((const float *)(p + (at + 16 * ql))); },
                   [&](const unsigned char *row) { st[i] = pg_load4((const float *)(row + 16 * ql)); });
    };
    auto put = [&](int v, const float4 (&st)[RPL]) {
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const int r = SROWS * wave + RSTEP * i + srow0;
            const int at = 256 * r + 16 * ((ql >> 1) ^ swz(r)) + 8 * (ql & 1);
            uint32_t w0[3], w1[3];
            pp_split2<true>(st[i].x, st[i].y, w0);
            pp_split2<true>(st[i].z, st[i].w, w1);
#pragma unroll
            for (int t = 0; t < (v ? NV : NK); t++) *reinterpret_cast<uint2 *>(plane(0, v, t) + at) = make_uint2(w0[t], w1[t]);
        }
    };

    // ---- fragment addresses: what depends on the lane once, the rest as bits over it ----
    const unsigned klane = 256 * ql + 16 * (hl ^ swz(ql));            // K row ql, chunk 2 t + hl: ^ 32 t
    // V^T rows 32 d + 16 (lane / 16 % 2) + lane % 16, keys 16 j + 4 hl .. + 3 and + 8: the rows that
    // this lane addresses, chunk 4 d + ..: ^ 64 d
    const int vrow = 4 * hl + ((lane & 15) >> 2), vchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const unsigned vlane = 256 * vrow + 8 * (lane & 1) + 16 * (vchunk ^ swz(vrow)),
                   vlane8 = 256 * (vrow + 8) + 8 * (lane & 1) + 16 * (vchunk ^ swz(vrow + 8));
    auto kfrag = [&](int buf, int y, int t) {
        return *reinterpret_cast<const bf16x8 *>(plane(buf, 0, y) + (klane ^ (32 * t)));
    };
    auto vfrag = [&](int buf, int y, int d, int j) {
        const unsigned char *p = plane(buf, 1, y) + 16 * 256 * j;
        return pp_vfrag(p + (vlane ^ (64 * d)), p + (vlane8 ^ (64 * d)));
    };

    // Barriers by hand: behind __syncthreads() the compiler has every LDS read wait for loads
    // that are still on their way to LDS.
    auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const int nt = (k1 - k0s + KG * PP_KT - 1) / (KG * PP_KT);       // tiles of a group
    pp_f32x16 st;
    bf16x8 pt[2][NP];
    [[maybe_unused]] bf16x8 one[2];

    // S^T of the tile in K buffer buf
    auto scores = [&](int buf) {
        st = (pp_f32x16){};
#pragma unroll
        for (int t = 0; t < 8; t++) {
            bf16x8 kf[NK];
#pragma unroll
            for (int y = 0; y < NK; y++) kf[y] = kfrag(buf, y, t);
            st = pp_products<NK, NQ>(kf, q[t], st);
        }
    };
    // The matrix part of a turn: V of one tile and K of the next, fragments read AHEAD steps before
    // their products.  The scores are one chain of sums: products in turn where a step has
    // few.  Six pairs have K's first, and V's fragments read only a step's length before.
    auto matrix = [&](int vbuf, int kbuf) {
        // products a step: of K, of V
        constexpr int KP = PpPairs<NK, NQ>::N, VP = PpPairs<NV, NP>::N, AHEAD = KP == 1 ? 3 : 1, RING = AHEAD + 1;
        constexpr bool TURNS = KP < 6;
        constexpr int VAHEAD = TURNS ? AHEAD : 0, VRING = VAHEAD + 1;
        constexpr auto LK = PpPairs<NK, NQ>::make();
        constexpr auto LV = PpPairs<NV, NP>::make();
        bf16x8 kf[RING][NK], vf[VRING][NV];
        auto read_k = [&](int u) {
#pragma unroll
            for (int y = 0; y < NK; y++) kf[u % RING][y] = kfrag(kbuf, y, u);
        };
        auto read_v = [&](int u) {
#pragma unroll
            for (int y = 0; y < NV; y++) vf[u % VRING][y] = vfrag(vbuf, y, u & 3, u >> 2);
        };
        st = (pp_f32x16){};
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            read_k(u);
            if (VAHEAD) read_v(u);
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (u + AHEAD < 8) read_k(u + AHEAD);
            if (u + VAHEAD < 8) read_v(u + VAHEAD);
#pragma unroll
            for (int n = 0; n < (KP > VP ? KP : VP); n++) {
                if (n < KP) st = pp_mfma(kf[u % RING][LK.a[n]], q[u][LK.b[n]], st);
                if (TURNS && n < VP) o[u & 3] = pp_mfma(vf[u % VRING][LV.a[n]], pt[u >> 2][LV.b[n]], o[u & 3]);
            }
            if (!TURNS) {
#pragma unroll
                for (int n = 0; n < VP; n++)
                    o[u & 3] = pp_mfma(vf[u % VRING][LV.a[n]], pt[u >> 2][LV.b[n]], o[u & 3]);
            }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, (NK + (TURNS ? 2 * NV : 0)) * AHEAD, 0);
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (u + AHEAD < 8) __builtin_amdgcn_sched_group_barrier(0x100, NK + 2 * NV, 0);
            else if (!TURNS) __builtin_amdgcn_sched_group_barrier(0x100, 2 * NV, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, KP + VP, 0);
        }
    };
    // The probabilities of the tile at k0.  The maximum that they are taken against follows the
    // running one only once a row has passed it by 2^8: p stays below that, no sum is the worse
    // for it, and most tiles leave the accumulators alone.
    auto softmax = [&](int k0, unsigned seen, auto guarded) {
        if (seen != 0xffffffffu || k0 + PP_KT - 1 > pos_lo) {                  // wave-uniform
            const int last = pos - k0;
            const unsigned bits = (last >= 31 ? seen : last < 0 ? 0u : seen & ((2u << last) - 1)) >> (4 * hl);
#pragma unroll
            for (int r = 0; r < 16; r++)
                if ((int)(bits << (31 - 8 * (r / 4) - r % 4)) >= 0) st[r] = -INFINITY;
        }
        float mx = st[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, st[r]);
        float other = mx;
        swap32(mx, other);
        mx = fmaxf(mx, other) * sc;
        if (__any(mx > m + 8.0f)) {
            const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - pg_ref(mn));
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < 4; d++) o[d] *= corr;
        }
        const float ref = pg_ref(m);
        float p[16], sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            p[r] = __builtin_amdgcn_exp2f(fmaf(st[r], sc, -ref));
            sum += p[r];
        }
        l += sum;
        pp_terms8<NP>(p, pt[0]);
        pp_terms8<NP>(p + 8, pt[1]);
        if constexpr (decltype(guarded)::value) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = p[8 * j + i] > 0.0f ? 1.0f : 0.0f;
                bf16x8 t[1];
                pp_terms8<1>(v, t);
                one[j] = t[0];
            }
        }
    };
    // O^T += V^T P^T with V buffer buf, where values may be infinite or none: finite ones as ever,
    // and how many others each row sees, counted on the matrix cores: + 1, 64 or 4096 each, at
    // most 32 of them
    auto values_guarded = [&](int buf) {
#pragma unroll
        for (int d = 0; d < 4; d++) {
            pp_f32x16 cnt = {};
#pragma unroll
            for (int j = 0; j < 2; j++) {
                bf16x8 vf[NV], cls;
                if constexpr (NK == 1) {
                    vf[0] = pp_finite(vfrag(buf, 0, d, j), cls);
                } else {                                  // see pp_split2
                    vf[1] = pp_finite(vfrag(buf, 1, d, j), cls);
#pragma unroll
                    for (int y = 0; y < NV; y += 2) vf[y] = pp_cleared(vfrag(buf, y, d, j), cls);
                }
                o[d] = pp_products<NV, NP>(vf, pt[j], o[d]);
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
    };

    // What a walk begins with: its first tiles on their way.
    Where next_v = {}, next_k = {};                       // of the tile whose V is fetched next, whose K was last
    unsigned seen1 = 0, seen2 = 0;                        // of the next softmax's tile, and of the one behind it
    float4 kr[DIRECT ? 2 : RPL], vr[DIRECT ? 2 : RPL];
    auto prime = [&]() {
        ids_at = INT_MIN / 2;
        next_v = where(0);
        next_k = where(1);
        seen1 = next_v.seen;
        seen2 = next_k.seen;
        if constexpr (DIRECT) {
            fetch(0, next_v, 0, 0);
            if (nt > 1) fetch(1, next_k, 0, 1);
            fetch(0, next_v, 1, 0);
        } else {
            load(0, next_v, 0, kr);
        }
    };
    // The group's tiles.  Turn i is a matrix part (V of tile i, K of tile i + 1) and a vector part
    // (softmax of tile i + 1, staging), a barrier behind each; the second group is a barrier
    // behind the first, so that on every SIMD one wave's matrix part meets another's vector
    // part.  Waves in step would leave the matrix cores idle in their vector parts.
    auto walk = [&](auto guarded) {
#pragma unroll
        for (int d = 0; d < 4; d++) o[d] = (pp_f32x16){};
        m = -INFINITY;
        l = 0.0f;
        if (nt == 0) return;                              // block-uniform
        if constexpr (DIRECT) __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        else put(0, kr);
        barrier();
        if (kg == 1) barrier();
        for (int i = -1; i < nt; i++) {
            if (wave_on) {
                // past the last tile the scores are of what the buffer held, and not used
                const int vbuf = i & (NBUF - 1), kbuf = (i + 1) & (NBUF - 1);
                if constexpr (decltype(guarded)::value) {
                    if (i >= 0) values_guarded(vbuf);
                    scores(kbuf);
                } else {
                    if (i >= 0) matrix(vbuf, kbuf);
                    else scores(kbuf);
                }
            }
            barrier();
            const unsigned seen = seen1;
            seen1 = seen2;
            if constexpr (DIRECT) {
                // over K of tile i + 1 and V of tile i, which are read
                next_v = next_k;
                if (i + 3 < nt) {
                    next_k = where(i + 3);
                    seen2 = next_k.seen;
                    fetch(i + 3, next_k, 0, (i + 1) & 1);
                }
                if (i + 2 < nt) fetch(i + 2, next_v, 1, i & 1);
                if (wave_on && i + 1 < nt) softmax(tile_k0(i + 1), seen, guarded);
                // the last turn's loads are there
                if (i + 3 < nt) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * RPL));
                else if (i + 2 < nt) __builtin_amdgcn_s_waitcnt(vmcnt_imm(RPL));
                else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            } else if (i + 1 < nt) {
                if (i >= 0) {
                    next_v = next_k;
                    next_k = where(i + 2);
                    seen1 = next_k.seen;
                }
                load(i + 2, next_k, 0, kr);
                load(i + 1, next_v, 1, vr);
                if (wave_on) softmax(tile_k0(i + 1), seen, guarded);
                put(0, kr);
                put(1, vr);
            }
            barrier();
        }
        if (kg == 0) barrier();
    };
    // Queries: dims 16 t + 8 hl .. + 7.  bf16 ones are on their way before the page ids are waited
    // for (16 prompts of 300 to 1000 rows: 154 us behind them, 151 before); fp32 ones, which are
    // split and take the scale along, would cost registers there (8 prompts on a bf16 cache: 72, 77).
    const T *const qp = (const T *)a.q + orow * PG_HD + 8 * hl;
    if constexpr (NQ == 1) {
#pragma unroll
        for (int t = 0; t < 8; t++) q[t][0] = *reinterpret_cast<const bf16x8 *>(qp + 16 * t);
    }
    if (nt > 0) prime();                                  // block-uniform
    if constexpr (NQ > 1) {
        const float fs = a.scale * PG_LOG2E;
#pragma unroll
        for (int t = 0; t < 8; t++) {
            const float4 x0 = pg_load4(qp + 16 * t), x1 = pg_load4(qp + 16 * t + 4);
            const float v[8] = {x0.x * fs, x0.y * fs, x0.z * fs, x0.w * fs, x1.x * fs, x1.y * fs, x1.z * fs, x1.w * fs};
            pp_terms8<NQ, true>(v, q[t]);
        }
    }
    walk(PpBool<false>());
    float z = 0.0f;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) z = fmaf(o[d][r], 0.0f, z);
    // 0 times what is infinite or no number is none
    if (__syncthreads_or(z != 0.0f)) {
        if (nt > 0) prime();
        walk(PpBool<true>());
        __syncthreads();
    }

    float L = l, other = l;
    swap32(L, other);
    L += other;
    // the second group's sums over the buffers that were last read before the barrier
    float4 *const po = reinterpret_cast<float4 *>(lds_all + wave * 16384) + lane;
    float2 *const pm = reinterpret_cast<float2 *>(lds_all + WR * 16384 + wave * 512) + lane;
    if (kg == 1) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int d = i / 4, r = 4 * (i % 4);
            po[64 * i] = make_float4(o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
        }
        *pm = make_float2(m, L);
    }
    __syncthreads();
    if (kg == 1) return;
    const float2 ml = *pm;
    const float mn = fmaxf(m, ml.x), ref = pg_ref(mn);
    const float c0 = __builtin_amdgcn_exp2f(m - ref), c1 = __builtin_amdgcn_exp2f(ml.x - ref);
    m = mn;
    L = fmaf(L, c0, ml.y * c1);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int d = i / 4, r = 4 * (i % 4);
        const float4 v = po[64 * i];
        o[d][r] = fmaf(v.x, c1, o[d][r] * c0);
        o[d][r + 1] = fmaf(v.y, c1, o[d][r + 1] * c0);
        o[d][r + 2] = fmaf(v.z, c1, o[d][r + 2] * c0);
        o[d][r + 3] = fmaf(v.w, c1, o[d][r + 3] * c0);
    }
    if (!on) return;
    if (a.nsplit == 1) {
        // 0 only where no key was seen: the largest p is at least 2^-8
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        T *dst = (T *)a.out + orow * PG_HD + 4 * hl;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                pg_store4(dst + 32 * d + 2 * r,
                          make_float4(o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv));
    } else {
        const size_t at = orow * a.nsplit + split;
        float *dst = a.part_o + at * PG_HD + 4 * hl;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4 *>(dst + 32 * d + 2 * r) =
                    make_float4(o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
        if (hl == 0) {
            a.part_ml[2 * at] = m;
            a.part_ml[2 * at + 1] = L;
        }
    }
}

extern "C" int qk_paged_prefill_plan(const qk_paged *p, int heads, int max_len, int *nsplit, int *chunk) {
    const long f = (long)p->rows * (heads / p->kv_heads);
    // Blocks of 64 rows run two to a CU, one's begin and end beside the other's products, but read every key twice as
    // often.  bf16, 128 and 64 rows: 16 prompts of 300 to 1000, 4 heads a kv head, 163 and
    // 151 us; 8 of 60 to 400, 2 heads, 32 and 16; 24 single tokens of 131 to 530, 8 heads, 22 and 16; but 4 prompts
    // of 1000 to 4000, 362 and 370, one of 8191, 392 and 426.  Where the keys are split, up to 768: 4 chunks of 30 rows
    // on fp32 rows, 500 positions, 17.3 and 16.6; 1000, 19.3 and 20.7.  On fp32 pages their tiles do not fit LDS twice,
    // but sequences of no more rows leave half of a larger block's waves idle, and one wave a SIMD has the registers
    // for six products with hardly a spill (fp32 rows, 31 behind 993: 22.6 and 20.6 us; 16 of 16 to 32 behind up to 600,
    // 46.6 and 38.0).  The host knows the mean of the sequences' rows alone, and goes by that: a long prompt among many
    // short ones gets blocks of 64 rows too (512 rows beside 31 tokens of 1000 positions, fp32: 164 and 114 us; of 4000:
    // 430 and 299; 4 of 500 beside 60 of 1000, whose mean is above: 250).
    const int fits = (f / PP_ROWS(2) + p->n_seqs) * p->kv_heads >= 320 ? 2048 : 768;
    const int rows2 = p->page_shift >= 4 && (p->cache_bf16 ? max_len <= fits : f <= PP_ROWS(2) * (long)p->n_seqs);
    const long blocks = (f / PP_ROWS(rows2 ? 2 : 4) + p->n_seqs) * p->kv_heads;
    // 1.5 blocks of 128 rows for each CU (24 single tokens of 500 to 6001 positions, 8 heads a kv head, bf16: 66 us, as
    // with 256 blocks; 512: 79; 4 chunks of 30 rows behind 970, fp32: 28.4, 31.5, 25.5), 1.25 of 64 (4 chunks of 30
    // rows behind 470, bf16: 14.2 us, as with 256 blocks; 512: 15.9)
    long n = ((rows2 ? 320 : 384) + blocks - 1) / blocks;
    if (n > QK_PAGED_MAX_SPLIT) n = QK_PAGED_MAX_SPLIT;
    long c = (max_len + n - 1) / n;
    c = (c + 63) / 64 * 64;
    if (c < 64) c = 64;
    // one block where that saves the join's launch (30 rows, 100 positions: bf16 10.2 us against 13.5, fp32 rows 11.7
    // against 14.3, but on an fp32 cache 18.8 against 18.6, and of 130 positions 22.7 against 18.5)
    if (p->cache_bf16 && max_len <= 128) c = 128;
    n = (max_len + c - 1) / c;
    *nsplit = n < 1 ? 1 : (int)n;
    *chunk = (int)c;
    return rows2;
}

template <typename T, typename C, int WR>
static int prefill_launch(const qk_paged_attn_args *a, hipStream_t s) {
    const qk_paged &pg = a->pg;
    const long slots = (long)pg.rows * (a->heads / pg.kv_heads) / PP_ROWS(WR) + pg.n_seqs;
    // a launch has fewer than 2^32 threads along an axis
    if (slots * pg.kv_heads > 0xffffffffL / PP_THREADS(WR)) return QWEN_HIP_EINVAL;
    const dim3 grid((unsigned)(slots * pg.kv_heads), (unsigned)a->nsplit);
    // the plan takes 64 rows for pages of 16 positions and more
    constexpr bool SOME_SMALL = WR == 4;
    if (SOME_SMALL && (1 << pg.page_shift) < PP_KT / WR)
        paged_prefill<T, C, SOME_SMALL, WR><<<grid, PP_THREADS(WR), 0, s>>>(*a, (int)slots);
    else paged_prefill<T, C, false, WR><<<grid, PP_THREADS(WR), 0, s>>>(*a, (int)slots);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}

extern "C" int qk_paged_prefill_launch(const qk_paged_attn_args *a, hipStream_t s) {
    if (!a->pg.cache_bf16) {
        if (a->act_bf16) return prefill_launch<uint16_t, float, 4>(a, s);        // 31 rows behind 600: 64 rows a block 17.6 us, 16.4; 16 of 16 to 32: 33.0, 27.8
        return a->rows2 ? prefill_launch<float, float, 2>(a, s) : prefill_launch<float, float, 4>(a, s);
    }
    if (a->rows2) return a->act_bf16 ? prefill_launch<uint16_t, uint16_t, 2>(a, s) : prefill_launch<float, uint16_t, 2>(a, s);
    return a->act_bf16 ? prefill_launch<uint16_t, uint16_t, 4>(a, s) : prefill_launch<float, uint16_t, 4>(a, s);
}
