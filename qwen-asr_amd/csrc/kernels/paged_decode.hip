// paged_decode.hip - attention of one new row per sequence over its paged KV
// cache, split over the cache's length and joined, and the join itself.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j,
//   m = max_j s_j over the positions j < kv_len whose page id is valid
//
// in one pass over the keys with a running m; a sequence without any gets 0.
// Bound by the bytes of K and V: every K and V row is read once for all query
// heads that share it (up to 8 in one block; more take another block's pass).
//
// Block (sequence x kv head x up to 8 heads, split): four waves take the
// split's keys in turns of 4 U.  Sixteen lanes own one key (8 dims a lane: 16 or
// 32 bytes, whole rows contiguous within a page), with statistics of their own,
// joined at the end: over the wave's four groups by row swaps, over the waves in
// LDS.  Loads of a turn (U keys' K and V a lane) are all in flight before the
// first product.
#include "paged.h"

struct PdRow8 {
    float x[8];
};
__device__ __forceinline__ PdRow8 pd_widen(uint4 w) {
    return {{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y), bf16_lo(w.z), bf16_hi(w.z), bf16_lo(w.w),
             bf16_hi(w.w)}};
}

// 8 values of a cached row as they lie in memory, widened at their use
template <typename C>
struct PdRaw;
template <>
struct PdRaw<uint16_t> {
    uint4 w;
    __device__ __forceinline__ void load(const uint16_t *p) { w = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ PdRow8 get() const { return pd_widen(w); }
};
template <>
struct PdRaw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = *reinterpret_cast<const float4 *>(p);
        b = *reinterpret_cast<const float4 *>(p + 4);
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ PdRow8 get() const { return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}}; }
};

__device__ __forceinline__ int pd_chunk(int len, int chunk, int nsplit) {
    const int need = (int)(((long)len + nsplit - 1) / nsplit);
    return max(chunk, (need + 63) & ~63);
}

template <typename T, typename C, int GT, int U>
__global__ __launch_bounds__(256) void paged_decode(qk_paged_attn_args a, int gchunks) {
    const qk_paged &pg = a.pg;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, grp = lane >> 4;
    const int G = a.heads / pg.kv_heads;
    const int kvh = blockIdx.x / gchunks % pg.kv_heads, s = blockIdx.x / gchunks / pg.kv_heads;
    const int g0 = blockIdx.x % gchunks * GT, gn = min(GT, G - g0);
    const int h0 = kvh * G + g0, split = blockIdx.y;
    const size_t qrow = (size_t)s * a.heads + h0;

    // this lane's 8 dims of each head's query, times scale * log2(e)
    float q[GT][8];
#pragma unroll
    for (int g = 0; g < GT; g++) {
        const T *qp = (const T *)a.q + (qrow + min(g, gn - 1)) * PG_HD + 8 * c;
        const float4 x = pg_load4(qp), y = pg_load4(qp + 4);
        const float f = a.scale * PG_LOG2E;
        q[g][0] = x.x * f; q[g][1] = x.y * f; q[g][2] = x.z * f; q[g][3] = x.w * f;
        q[g][4] = y.x * f; q[g][5] = y.y * f; q[g][6] = y.z * f; q[g][7] = y.w * f;
    }
    const int len = min(pg_len(pg, s), pg.capacity);
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

    float m[GT], l[GT], o[GT][8];
#pragma unroll
    for (int g = 0; g < GT; g++) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) o[g][i] = 0.0f;
    }
    const C *kp = (const C *)pg.k, *vp = (const C *)pg.v;
    constexpr int TURN = 4 * U;                       // keys of one wave's turn
    int pid[U];
    auto ids = [&](int kb) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int key = kb + 4 * u + grp;
            pid[u] = key < k1 ? pg_page(pg, s, key) : -1;
        }
    };
    ids(k0 + wave * TURN);
    for (int kb = k0 + wave * TURN; kb < k1; kb += 4 * TURN) {
        PdRaw<C> kr[U], vr[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            on[u] = pid[u] >= 0;
            if (on[u]) {
                const size_t off = pg_offset(pg, pid[u], kvh, kb + 4 * u + grp) + 8 * c;
                kr[u].load(kp + off);
                vr[u].load(vp + off);
            } else {
                kr[u].zero();
                vr[u].zero();
            }
        }
        ids(kb + 4 * TURN);                           // the next turn's pages
        float sc[U][GT];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const PdRow8 k8 = kr[u].get();
#pragma unroll
            for (int g = 0; g < GT; g++) {
                float d = q[g][0] * k8.x[0];
#pragma unroll
                for (int i = 1; i < 8; i++) d = fmaf(q[g][i], k8.x[i], d);
                d = group_sum<16>(d);
                sc[u][g] = on[u] ? d : -INFINITY;
            }
        }
#pragma unroll
        for (int g = 0; g < GT; g++) {
            float mn = m[g];
#pragma unroll
            for (int u = 0; u < U; u++) mn = fmaxf(mn, sc[u][g]);
            const float ref = pg_ref(mn), corr = __builtin_amdgcn_exp2f(m[g] - ref);
            m[g] = mn;
            l[g] *= corr;
#pragma unroll
            for (int i = 0; i < 8; i++) o[g][i] *= corr;
#pragma unroll
            for (int u = 0; u < U; u++) {
                sc[u][g] = __builtin_amdgcn_exp2f(sc[u][g] - ref);
                l[g] += sc[u][g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const PdRow8 v8 = vr[u].get();
#pragma unroll
            for (int g = 0; g < GT; g++)
#pragma unroll
                for (int i = 0; i < 8; i++) o[g][i] = fmaf(sc[u][g], v8.x[i], o[g][i]);
        }
    }

    // the wave's four groups, then the four waves
    __shared__ __attribute__((aligned(16))) float so[4][GT][PG_HD];
    __shared__ float sm[4][GT], sl[4][GT];
#pragma unroll
    for (int g = 0; g < GT; g++) {
        const float M = xor_max16_32(m[g]), f = __builtin_amdgcn_exp2f(m[g] - pg_ref(M));
        const float L = xor_sum16_32(l[g] * f);
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = xor_sum16_32(o[g][i] * f);
        if (grp == 0) {
            *reinterpret_cast<float4 *>(&so[wave][g][8 * c]) = make_float4(t[0], t[1], t[2], t[3]);
            *reinterpret_cast<float4 *>(&so[wave][g][8 * c + 4]) = make_float4(t[4], t[5], t[6], t[7]);
        }
        if (lane == 0) {
            sm[wave][g] = M;
            sl[wave][g] = L;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gn * (PG_HD / 4); i += 256) {
        const int g = i / (PG_HD / 4), d = 4 * (i % (PG_HD / 4));
        const float M = fmaxf(fmaxf(sm[0][g], sm[1][g]), fmaxf(sm[2][g], sm[3][g])), ref = pg_ref(M);
        float L = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(sm[w][g] - ref);
            const float4 x = *reinterpret_cast<const float4 *>(&so[w][g][d]);
            L = fmaf(sl[w][g], f, L);
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
        }
        if (a.nsplit == 1) {
            // L is 0 only where no key was seen (the largest p is 1); a sum that is no number stays one
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            pg_store4((T *)a.out + (qrow + g) * PG_HD + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        } else {
            const size_t at = (qrow + g) * a.nsplit + split;
            *reinterpret_cast<float4 *>(a.part_o + at * PG_HD + d) = v;
            if (d == 0) {
                a.part_ml[2 * at] = M;
                a.part_ml[2 * at + 1] = L;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The join: a wave per (row, head), two dims a lane.  Lane i holds split i's
// maximum and sum, so one load and one wave maximum give every weight; splits
// with the sum 0 have no partial output and are skipped.  Rows before the first
// or behind the last sequence have no partials and are left as they are.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void paged_merge(qk_paged_attn_args a) {
    const qk_paged &pg = a.pg;
    const int lane = threadIdx.x & 63;
    const long u = 4L * blockIdx.x + (threadIdx.x >> 6);
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
    const float M = wave_max(m);
    // a maximum that is no number passes fmaxf by: its sum is none either
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - pg_ref(M));
    const float L = wave_sum(l * f);
    const unsigned long long some = __ballot(l != 0.0f);
    float x = 0.0f, y = 0.0f;
    const int last = 63 - __clzll((long long)some | 1);
    // four loads in flight; a split without keys reads the last one that has some
    for (int i0 = 0; i0 <= last; i0 += 4) {
        float2 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = (some >> min(i0 + j, 63)) & 1 ? i0 + j : last;
            v[j] = some ? *reinterpret_cast<const float2 *>(a.part_o + (at + i) * PG_HD + 2 * lane) : make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (i0 + j > last || !((some >> (i0 + j)) & 1)) continue;
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), i0 + j));
            x = fmaf(v[j].x, w, x);
            y = fmaf(v[j].y, w, y);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T *out = (T *)a.out + (size_t)u * PG_HD + 2 * lane;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(out) = make_float2(x * inv, y * inv);
    else *reinterpret_cast<uint32_t *>(out) = bf16_pack2(x * inv, y * inv);
}

extern "C" int qk_paged_merge_launch(const qk_paged_attn_args *a, hipStream_t s) {
    const long blocks = ((long)a->pg.rows * a->heads + 3) / 4;
    if (blocks > 0x7fffffffL) return QWEN_HIP_EINVAL;
    if (a->act_bf16) paged_merge<uint16_t><<<(unsigned)blocks, 256, 0, s>>>(*a);
    else paged_merge<float><<<(unsigned)blocks, 256, 0, s>>>(*a);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}

static int decode_gt(int G) { return G >= 8 ? 8 : G > 2 ? (G > 4 ? 8 : 4) : G; }

extern "C" void qk_paged_decode_plan(int n_seqs, int heads, int kv_heads, int max_len, int *nsplit, int *chunk) {
    const int G = heads / kv_heads, gt = decode_gt(G);
    const long blocks = (long)n_seqs * kv_heads * ((G + gt - 1) / gt);
    long n = (4096 + blocks - 1) / blocks;
    n = n > QK_PAGED_MAX_SPLIT ? QK_PAGED_MAX_SPLIT : n;
    long c = (max_len + n - 1) / n;
    c = (c + 63) / 64 * 64;
    if (c < 64) c = 64;
    n = (max_len + c - 1) / c;
    *nsplit = n < 1 ? 1 : (int)n;
    *chunk = (int)c;
}

template <typename T, typename C>
static void decode_dispatch(const qk_paged_attn_args *a, hipStream_t s) {
    const int G = a->heads / a->pg.kv_heads, gt = decode_gt(G), gc = (G + gt - 1) / gt;
    const dim3 grid((unsigned)(a->pg.rows * a->pg.kv_heads * gc), (unsigned)a->nsplit);
    constexpr int U = 4;
    if (gt == 1) paged_decode<T, C, 1, U><<<grid, 256, 0, s>>>(*a, gc);
    else if (gt == 2) paged_decode<T, C, 2, U><<<grid, 256, 0, s>>>(*a, gc);
    else if (gt == 4) paged_decode<T, C, 4, U><<<grid, 256, 0, s>>>(*a, gc);
    else paged_decode<T, C, 8, U><<<grid, 256, 0, s>>>(*a, gc);
}

extern "C" int qk_paged_decode_launch(const qk_paged_attn_args *a, hipStream_t s) {
    const int G = a->heads / a->pg.kv_heads, gt = decode_gt(G);
    if ((long)a->pg.rows * a->pg.kv_heads * ((G + gt - 1) / gt) > 0x7fffffffL) return QWEN_HIP_EINVAL;
    if (a->act_bf16) {
        if (a->pg.cache_bf16) decode_dispatch<uint16_t, uint16_t>(a, s);
        else decode_dispatch<uint16_t, float>(a, s);
    } else {
        if (a->pg.cache_bf16) decode_dispatch<float, uint16_t>(a, s);
        else decode_dispatch<float, float>(a, s);
    }
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
