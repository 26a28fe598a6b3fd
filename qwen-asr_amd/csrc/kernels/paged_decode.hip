// paged_decode.hip - attention of one new row per sequence over its paged KV
// cache, split over the cache's length and joined, and the join itself.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j,
//   m = max_j s_j over the positions j < kv_len whose page id is valid
//
// in one pass over the keys with a running m; a sequence without any gets 0.
// Bound by the bytes of K and V: every K and V row is read once for all query
// heads that share it (up to 8 in one block; more take another block's pass).  Many
// heads on a bf16 cache run on the matrix cores instead (csrc/host/paged.c).
//
// Block (sequence x kv head x up to 8 heads, split): four waves take the split's
// keys in turns.  L lanes own one key (128 / L dims a lane, in 16-byte chunks L
// apart, so that a load of the wave reads whole lines: with 32 bytes a lane, fp32
// pages took 114 us instead of 84), each such group with statistics of its own, joined
// at the end: over the wave by halving exchanges, over the waves in LDS.  Fewer lanes
// a key mean fewer steps of the sum over them and fewer lanes that compute the same
// exponential, but more registers for queries and outputs.  Loads of a turn (U keys'
// K and V a group) are all in flight before the first product, the page ids of the
// next turn before those.  L, U by heads and page type, 24 sequences of 500 to 6001:
//   1 and 2 heads, bf16: 8, 2 (2 heads: 47 us; 8, 4: 50; 16, 4: 48; 4, 4: 68); fp32: 16, 4
//     (84 us; 8, 4: 86; 16, 2: 85)
//   4 heads, bf16: 16, 4 (58 us; 16, 2: 60); fp32 likewise (88; 32, 4: 92)
//   8 heads: 16, 4 (fp32: 114 us; 16, 2: 118; 32, 4: 136)
//
// Measured, kernel and join, 8 kv heads (a device copy moves 4.8 TB/s):
//   64 sequences of 31 to 4097 positions, bf16, 2 heads each: 46.5 us, 4.8 TB/s
//   3 sequences of 20011 to 32769, fp32 rows on bf16 pages, 4 heads each: 66 us, 4.9 TB/s
//   24 sequences of 500 to 6001, all fp32, 1 head each: 81 us, 5.3 TB/s; 8 heads: 108 us,
//     bound by the vector units
// One short sequence is the time of two launches (11 us).
//
// Windows (WIN): the same over the positions that the row sees, the first ones and the window's, as if they were next
// to each other (PgSeen).  64 sequences of 31 to 32769 positions, bf16, 2048 positions and 16 first ones: 52.5 us, 5.5 TB/s.
#include "paged.h"

// 16 bytes of a cached row as they lie in memory, widened at their use.  NT: rows that are
// read once pass by the caches (64 sequences, 222 MB of pages: 54 us without, 48 with; fp32
// pages, 24 sequences: 93 and 83).
typedef uint32_t pd_u32x4 __attribute__((ext_vector_type(4)));
template <typename C>
struct PdRaw {
    static constexpr int N = 16 / sizeof(C);
    pd_u32x4 w;
    template <bool NT>
    __device__ __forceinline__ void load(const C *p) {
        if constexpr (NT) w = __builtin_nontemporal_load((const pd_u32x4 *)p);
        else w = *(const pd_u32x4 *)p;
    }
    __device__ __forceinline__ void zero() { w = (pd_u32x4){0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (N == 4) return __uint_as_float(w[i]);
        else return i % 2 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
    }
};

// Sums over the lanes that differ in the bits 32, 16, .., L of v[N], halving the values that
// a lane carries at each step: the lane ends with N L / 64 of them, from `base` on.
template <int N, int M, int L, int FULL>
__device__ __forceinline__ void pd_gather(float (&v)[FULL], int lane, int &base) {
    if constexpr (M >= L) {
        transpose_step<FULL, M>(v, N, lane);
        if (lane & M) base += N / 2;
        pd_gather<N / 2, M / 2, L, FULL>(v, lane, base);
    }
}

__device__ __forceinline__ int pd_chunk(int len, int chunk, int nsplit) {
    const int need = (int)(((long)len + nsplit - 1) / nsplit);
    return max(chunk, (need + 63) & ~63);
}

// WIN: of a window and the first positions.
template <typename T, typename C, int GT, int L, int U, bool NT, bool WIN>
__global__ __launch_bounds__(256) void paged_decode(qk_paged_attn_args a, int gchunks) {
    // dims a lane, in NC chunks of 16 bytes (CD dims); keys a wave at once
    constexpr int D = PG_HD / L, CD = PdRaw<C>::N, NC = D / CD, KEYS = 64 / L;
    static_assert(NC * CD * L == PG_HD, "lanes a key");
    const qk_paged &pg = a.pg;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % L, grp = lane / L;
    const int G = a.heads / pg.kv_heads;
    const int kvh = blockIdx.x / gchunks % pg.kv_heads, s = blockIdx.x / gchunks / pg.kv_heads;
    const int g0 = blockIdx.x % gchunks * GT, gn = min(GT, G - g0);
    const int h0 = kvh * G + g0, split = blockIdx.y;
    const size_t qrow = (size_t)s * a.heads + h0;
    int len = min(pg_len(pg, s), pg.capacity);
    PgSeen seen = {};
    if constexpr (WIN) {
        seen = pg_seen<1>(a, (long)pg_len(pg, s) - 1, len);
        len = seen.end;
    }
    // position of the key `i` that the row sees
    auto place = [&](int i) {
        if constexpr (WIN) return seen.at(i);
        else return i;
    };
    const int chunk = pd_chunk(len, a.chunk, a.nsplit);
    const long first = (long)split * chunk;
    if (first >= len && split > 0) {
        // no keys here: the join skips what has the sum 0
        if ((int)threadIdx.x < gn) {
            float *ml = a.part_ml + 2 * ((qrow + threadIdx.x) * a.nsplit + split);
            ml[0] = -INFINITY;
            ml[1] = 0.0f;
        }
        return;
    }
    const int k0 = (int)first, k1 = (int)min((long)len, first + chunk);

    // rows of a kv head: page id * rstride + slot (the host has seen that they fit an int)
    const int *const table = pg.table + (size_t)s * pg.table_stride;
    const int rstride = pg.kv_heads << pg.page_shift, smask = (1 << pg.page_shift) - 1;
    const C *kp = (const C *)pg.k + ((size_t)kvh << pg.page_shift) * PG_HD + CD * c;
    const C *vp = (const C *)pg.v + ((size_t)kvh << pg.page_shift) * PG_HD + CD * c;
    constexpr int TURN = KEYS * U;                    // keys of one wave's turn
    int pid[U];
    auto ids = [&](int kb) {
#pragma unroll
        for (int u = 0; u < U; u++) pid[u] = k1 > k0 ? table[place(min(kb + KEYS * u + grp, k1 - 1)) >> pg.page_shift] : -1;
    };
    ids(k0 + wave * TURN);

    // this lane's dims of each head's query, times scale * log2(e)
    float q[GT][D];
#pragma unroll
    for (int g = 0; g < GT; g++) {
        const T *qp = (const T *)a.q + (qrow + min(g, gn - 1)) * PG_HD + CD * c;
        const float f = a.scale * PG_LOG2E;
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int e = 0; e < CD; e += 4) {
                const float4 x = pg_load4(qp + CD * L * i + e);
                float *o = &q[g][CD * i + e];
                o[0] = x.x * f; o[1] = x.y * f; o[2] = x.z * f; o[3] = x.w * f;
            }
    }
    float m[GT], l[GT], o[GT * D];
#pragma unroll
    for (int g = 0; g < GT; g++) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < GT * D; i++) o[i] = 0.0f;

    for (int kb = k0 + wave * TURN; kb < k1; kb += 4 * TURN) {
        PdRaw<C> kr[U][NC], vr[U][NC];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            // a key past the end, or without a page, is read where it does no harm and weighs nothing
            const int key = kb + KEYS * u + grp;
            const bool page = (unsigned)pid[u] < (unsigned)pg.n_pages;
            on[u] = page && key < k1;
            const size_t row = (unsigned)((page ? pid[u] : 0) * rstride + (place(min(key, k1 - 1)) & smask));
#pragma unroll
            for (int i = 0; i < NC; i++) {
                kr[u][i].template load<NT>(kp + row * PG_HD + CD * L * i);
                vr[u][i].template load<NT>(vp + row * PG_HD + CD * L * i);
            }
        }
        if (kb + 4 * TURN < k1) ids(kb + 4 * TURN);   // the next turn's pages
        float sc[U][GT];
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int g = 0; g < GT; g++) sc[u][g] = 0.0f;
#pragma unroll
            for (int i = 0; i < NC; i++)
#pragma unroll
                for (int g = 0; g < GT; g++)
#pragma unroll
                    for (int e = 0; e < CD; e++) sc[u][g] = fmaf(q[g][CD * i + e], kr[u][i][e], sc[u][g]);
#pragma unroll
            for (int g = 0; g < GT; g++) {
                const float d = group_sum<L>(sc[u][g]);
                sc[u][g] = on[u] ? d : -INFINITY;
            }
        }
        // the maximum, followed once a key has passed it by 2^8: weights stay below that, no sum is the
        // worse for it, and most turns leave the outputs alone
        bool passed = false;
        float mx[GT];
#pragma unroll
        for (int g = 0; g < GT; g++) {
            mx[g] = sc[0][g];
#pragma unroll
            for (int u = 1; u < U; u++) mx[g] = fmaxf(mx[g], sc[u][g]);
            passed = passed || mx[g] > m[g] + 8.0f;
        }
        if (__any(passed)) {
#pragma unroll
            for (int g = 0; g < GT; g++) {
                const float mn = fmaxf(m[g], mx[g]), corr = __builtin_amdgcn_exp2f(m[g] - pg_ref(mn));
                m[g] = mn;
                l[g] *= corr;
#pragma unroll
                for (int i = 0; i < D; i++) o[g * D + i] *= corr;
            }
        }
#pragma unroll
        for (int g = 0; g < GT; g++) {
            const float ref = pg_ref(m[g]);
#pragma unroll
            for (int u = 0; u < U; u++) {
                sc[u][g] = __builtin_amdgcn_exp2f(sc[u][g] - ref);
                l[g] += sc[u][g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (!__all(on[u])) {                      // the last turn: nothing may come of 0 times what is there
#pragma unroll
                for (int i = 0; i < NC; i++)
                    if (!on[u]) vr[u][i].zero();
            }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < NC; i++)
#pragma unroll
                for (int g = 0; g < GT; g++)
#pragma unroll
                    for (int e = 0; e < CD; e++)
                        o[g * D + CD * i + e] = fmaf(sc[u][g], vr[u][i][e], o[g * D + CD * i + e]);
    }

    // the wave's groups, then the four waves
    __shared__ __attribute__((aligned(16))) float so[4][GT][PG_HD];
    __shared__ float sm[4][GT], sl[4][GT];
#pragma unroll
    for (int g = 0; g < GT; g++) {
        const float M = wave_max(m[g]), f = __builtin_amdgcn_exp2f(m[g] - pg_ref(M));
        const float S = wave_sum(l[g] * f) * (1.0f / L);          // L lanes hold the same
#pragma unroll
        for (int i = 0; i < D; i++) o[g * D + i] *= f;
        if (lane == 0) {
            sm[wave][g] = M;
            sl[wave][g] = S;
        }
    }
    int base = 0;
    pd_gather<GT * D, 32, L>(o, lane, base);
#pragma unroll
    for (int i = 0; i < GT * D * L / 64; i++) {
        const int n = base + i, g = n / D, e = n % D;             // dim: chunk e / CD of this lane's
        so[wave][g][CD * c + CD * L * (e / CD) + e % CD] = o[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gn * (PG_HD / 4); i += 256) {
        const int g = i / (PG_HD / 4), d = 4 * (i % (PG_HD / 4));
        const float M = fmaxf(fmaxf(sm[0][g], sm[1][g]), fmaxf(sm[2][g], sm[3][g])), ref = pg_ref(M);
        float sum = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(sm[w][g] - ref);
            const float4 x = *reinterpret_cast<const float4 *>(&so[w][g][d]);
            sum = fmaf(sl[w][g], f, sum);
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
        }
        if (a.nsplit == 1) {
            // 0 only where no key was seen (the largest p is at least 2^-8); a sum that is no number stays one
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            pg_store4((T *)a.out + (qrow + g) * PG_HD + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        } else {
            const size_t at = (qrow + g) * a.nsplit + split;
            *reinterpret_cast<float4 *>(a.part_o + at * PG_HD + d) = v;
            if (d == 0) {
                a.part_ml[2 * at] = M;
                a.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The join: W waves per (row, head), two dims a lane.  Lane i holds split i's
// maximum and sum, so one load and one wave maximum give every weight; splits
// with the sum 0 have no partial output and are skipped.  A wave takes every W-th
// split, 16 loads in flight.  Rows before the first or behind the last sequence have
// no partials and are left as they are.
// ---------------------------------------------------------------------------
template <typename T, int W>
__global__ __launch_bounds__(256) void paged_merge(qk_paged_attn_args a) {
    const qk_paged &pg = a.pg;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long u = W == 1 ? 4L * blockIdx.x + wave : (long)blockIdx.x;
    if (u >= (long)pg.rows * a.heads) return;
    if (pg.row_start) {
        const int row = (int)(u / a.heads);
        if (row < pg.row_start[0] || row >= pg.row_start[pg.n_seqs]) return;
    }
    const int n = a.nsplit;
    const size_t at = (size_t)u * n;
    float m = -INFINITY, l = 0.0f;
    if (lane < n) {
        const float2 x = *reinterpret_cast<const float2 *>(a.part_ml + 2 * (at + lane));
        l = x.y;
        m = l == 0.0f ? -INFINITY : x.x;
    }
    if (__builtin_amdgcn_readfirstlane(__float_as_int(l)) == __float_as_int(QK_PAGED_DONE)) return;      // the wave's, and all waves of the row
    const float M = wave_max(m);
    // a maximum that is no number passes fmaxf by: its sum is none either
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - pg_ref(M));
    const float L = wave_sum(l * f);
    const unsigned long long some = __ballot(l != 0.0f);
    float x = 0.0f, y = 0.0f;
    const int last = 63 - __clzll((long long)some | 1), first = W == 1 ? 0 : wave;
    // a split without keys reads the last one that has some, with no weight
    constexpr int F = W == 1 ? 8 : 16;
    for (int i0 = first; some && i0 <= last; i0 += F * W) {
        float2 v[F];
#pragma unroll
        for (int j = 0; j < F; j++) {
            const int i = i0 + W * j <= last && (some >> (i0 + W * j)) & 1 ? i0 + W * j : last;
            v[j] = *reinterpret_cast<const float2 *>(a.part_o + (at + i) * PG_HD + 2 * lane);
        }
#pragma unroll
        for (int j = 0; j < F; j++) {
            if (i0 + W * j > last || !((some >> (i0 + W * j)) & 1)) continue;
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), i0 + W * j));
            x = fmaf(v[j].x, w, x);
            y = fmaf(v[j].y, w, y);
        }
    }
    if constexpr (W > 1) {
        __shared__ float2 part[W][64];
        part[wave][lane] = make_float2(x, y);
        __syncthreads();
        if (wave > 0) return;
        x = y = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) {
            x += part[i][lane].x;
            y += part[i][lane].y;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T *out = (T *)a.out + (size_t)u * PG_HD + 2 * lane;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(out) = make_float2(x * inv, y * inv);
    else *reinterpret_cast<uint32_t *>(out) = bf16_pack2(x * inv, y * inv);
}

extern "C" int qk_paged_merge_launch(const qk_paged_attn_args *a, hipStream_t s) {
    const long units = (long)a->pg.rows * a->heads;
    // few rows with many splits: a block each
    const bool wide = a->nsplit > 16 && units <= 4096;
    const unsigned blocks = (unsigned)(wide ? units : (units + 3) / 4);
    if (a->act_bf16) {
        if (wide) paged_merge<uint16_t, 4><<<blocks, 256, 0, s>>>(*a);
        else paged_merge<uint16_t, 1><<<blocks, 256, 0, s>>>(*a);
    } else {
        if (wide) paged_merge<float, 4><<<blocks, 256, 0, s>>>(*a);
        else paged_merge<float, 1><<<blocks, 256, 0, s>>>(*a);
    }
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}

static int decode_gt(int G) { return G >= 8 ? 8 : G > 2 ? (G > 4 ? 8 : 4) : G; }

extern "C" void qk_paged_decode_plan(int n_seqs, int heads, int kv_heads, int cache_bf16, int max_len, int *nsplit,
                                     int *chunk) {
    const int G = heads / kv_heads, gt = decode_gt(G);
    const long blocks = (long)n_seqs * kv_heads * ((G + gt - 1) / gt);
    // Blocks, where there are keys for them: 8192 of one or two heads (64 sequences of up to 4097, bf16: 46.7 us; 4096:
    // 48.5, 2048: 58.2), fewer of more, whose joins weigh more (24 of up to 6001, 4 heads, bf16: 58.4 us with 4096,
    // 60.7 with 8192; 8 heads, fp32: 108 us with 2048, 114 and 125).  Of 128 keys at least (16 sequences of 1000, bf16:
    // 14.2 us; 64 keys: 17.0), and one where that saves the join's launch (1 sequence of 300, bf16: 8.7 us against
    // 10.7; fp32: 11.1, 10.7; of 200: 8.5, 11.2).
    const long target = gt == 8 ? 2048 : gt == 4 ? 4096 : 8192;
    long n = (target + blocks - 1) / blocks;
    n = n > QK_PAGED_MAX_SPLIT ? QK_PAGED_MAX_SPLIT : n;
    long c = (max_len + n - 1) / n;
    c = (c + 63) / 64 * 64;
    if (c < 128) c = 128;
    if (max_len <= (cache_bf16 ? 512 : 256)) c = 512;
    n = (max_len + c - 1) / c;
    *nsplit = n < 1 ? 1 : (int)n;
    *chunk = (int)c;
}

template <typename T, typename C, bool WIN>
static void decode_dispatch(const qk_paged_attn_args *a, hipStream_t s) {
    const int G = a->heads / a->pg.kv_heads, gt = decode_gt(G), gc = (G + gt - 1) / gt;
    const dim3 grid((unsigned)(a->pg.rows * a->pg.kv_heads * gc), (unsigned)a->nsplit);
    constexpr int L = sizeof(C) == 4 ? 16 : 8, U = sizeof(C) == 4 ? 4 : 2;
    if (gt == 1) paged_decode<T, C, 1, L, U, true, WIN><<<grid, 256, 0, s>>>(*a, gc);
    else if (gt == 2) paged_decode<T, C, 2, L, U, true, WIN><<<grid, 256, 0, s>>>(*a, gc);
    else if (gt == 4) paged_decode<T, C, 4, 16, 4, true, WIN><<<grid, 256, 0, s>>>(*a, gc);
    else if constexpr (sizeof(C) == 4) {              // more than four heads on bf16 pages do not come here
        if (gc == 1) paged_decode<T, C, 8, 16, 4, true, WIN><<<grid, 256, 0, s>>>(*a, gc);
        // every block of heads reads the rows: 16 heads, 24 sequences of 500 to 6001: 153 us, 166 past the caches
        else paged_decode<T, C, 8, 16, 4, false, WIN><<<grid, 256, 0, s>>>(*a, gc);
    }
}

template <bool WIN>
static void decode_types(const qk_paged_attn_args *a, hipStream_t s) {
    if (a->act_bf16) {
        if (a->pg.cache_bf16) decode_dispatch<uint16_t, uint16_t, WIN>(a, s);
        else decode_dispatch<uint16_t, float, WIN>(a, s);
    } else {
        if (a->pg.cache_bf16) decode_dispatch<float, uint16_t, WIN>(a, s);
        else decode_dispatch<float, float, WIN>(a, s);
    }
}

extern "C" int qk_paged_decode_launch(const qk_paged_attn_args *a, hipStream_t s) {
    const int G = a->heads / a->pg.kv_heads, gt = decode_gt(G);
    if ((long)a->pg.rows * a->pg.kv_heads * ((G + gt - 1) / gt) > 0x7fffffffL) return QWEN_HIP_EINVAL;
    if (a->pg.cache_bf16 && gt == 8) return QWEN_HIP_EINVAL;
    if (a->window) decode_types<true>(a, s);
    else decode_types<false>(a, s);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
