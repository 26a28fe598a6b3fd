// beam.hip - the best continuations of a sequence's beams: of the candidates (beam b, token i)
// the n with the largest
//
//   score_b + x_i - M_b - log(sum_i e^(x_i - M_b)),   M_b = max_i x_i
//
// by falling score, equal ones by (b, i).  One pass over the logits:
//
//   beam_rows    block (share of a row): its maximum and sum of exponentials, and its n largest entries
//                in order.  Only entries from a threshold on are looked at: the n-th largest of the 64 lanes'
//                maxima of a wave is no larger than the n-th largest entry, so it is a lower
//                bound; in each of the four waves at most n lanes reach the largest such
//                bound, so at most 4 n VPT entries do (as a rule about 2 n).
//   beam_select  block (sequence): each beam's logarithm from its shares, and the n best of all shares'
//                lists, by a threshold of the same kind.
//
// Exponentials: (x - M) log2(e) in 64 bits, its whole part into the exponent, v_exp_f32 (1 ulp) of the rest;
// sums, logarithms and scores in 64 bits, in an order that does not depend on the run.
// Entries are compared as whole numbers (the value's order in the upper half, the index below, the lower
// one first), so equal ones are in order and every choice is unique.
#include "common.h"
#include "qk_kernels.h"
#include "qwen_asr_hip.h"

#include <math.h>

#define BM_THREADS 256
#define BM_WAVES 4
#define BM_LIST 2048                  // entries from the threshold on: 4 n VPT at most
#define BM_LOG2E 1.4426950408889634

typedef unsigned long long bm_u64;

struct BmShare {                      // of a row: maximum (-inf: no entry), sum of e^(x - maximum)
    double sum;
    float max, pad;
};

// what is no number is no entry, +inf the largest number
__device__ __forceinline__ float bm_clean(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f) + 0.0f; }

// the order of entries: larger first, then the lower index; 0 is none
__device__ __forceinline__ bm_u64 bm_key(float x, unsigned i) {
    const unsigned u = __float_as_uint(x);
    return (bm_u64)(u ^ ((unsigned)((int)u >> 31) | 0x80000000u)) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float bm_value(bm_u64 key) {
    const unsigned u = (unsigned)(key >> 32);
    return __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ unsigned bm_index(bm_u64 key) { return 0xffffffffu - (unsigned)key; }

__device__ __forceinline__ bm_u64 bm_order(double x) {
    const bm_u64 u = (bm_u64)__double_as_longlong(x);
    return u ^ ((bm_u64)((long long)u >> 63) | 1ull << 63);
}
__device__ __forceinline__ double bm_double(bm_u64 u) {
    return __longlong_as_double((long long)(u >> 63 ? u ^ 1ull << 63 : ~u));
}

// 2^t, t <= 0 or so
__device__ __forceinline__ float bm_exp2(double t) {
    const double magic = 6755399441055744.0, z = t + magic;      // 1.5 2^52: t's whole part in the low word
    const float f = (float)(t - (z - magic));
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(f), (int)(unsigned)(bm_u64)__double_as_longlong(z));
}

__device__ __forceinline__ double bm_sum(double v) {             // of a wave, the same in every lane
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// A number that at least n of the wave's 64 keys reach, and not many more (0 where fewer are entries): the
// bits of the n-th largest from the top, until no more than n reach them.
template <typename K, int BITS>
__device__ __forceinline__ K bm_bound(K key, int n) {
    K t = 0;
    for (int b = BITS - 1; b >= 0; b--) {
        const K u = t | (K)1 << b;
        const int c = __popcll(__ballot(key >= u));
        if (c >= n) t = u;
        if (c == n) break;
    }
    return t;
}

struct BmRows {
    const void *logits;
    long stride;
    int vocab, n, shares;
    const float *score;
    const int *ended;
    BmShare *share;                   // [rows][shares]
    bm_u64 *list;                     // [rows][shares][n]
};

// a beam that takes no part with its logits: one at its end, one without a score
__device__ __forceinline__ bool bm_idle(const float *score, const int *ended, int row, int vocab) {
    const float s = score[row];
    return !(fabsf(s) <= 3.402823466e38f) || (ended && (unsigned)ended[row] < (unsigned)vocab);
}

template <typename T, int VPT>
__global__ __launch_bounds__(BM_THREADS) void beam_rows(BmRows a) {
    constexpr int V = 16 / sizeof(T), NV = VPT / V;              // entries of a load, loads
    __shared__ float wmax[BM_WAVES];
    __shared__ bm_u64 wbound[BM_WAVES], list[BM_LIST];
    __shared__ double wsum[BM_WAVES];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int share = blockIdx.y, row = blockIdx.x;
    const T *const x0 = (const T *)a.logits + (size_t)row * a.stride;
    if (bm_idle(a.score, a.ended, row, a.vocab)) return;
    if (tid == 0) count = 0;
    // Shares and threads by index, whatever the row's alignment: equal rows have equal sums.  (Loads of 16 bytes
    // need no more alignment than the type's.)
    auto index = [&](int j) { return share * BM_THREADS * VPT + (j * BM_THREADS + tid) * V; };
    float x[VPT];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = index(j);
        if (i + V <= a.vocab) {
            unsigned u[4];
            __builtin_memcpy(u, x0 + i, 16);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (V == 4) x[V * j + k] = __uint_as_float(u[k]);
                else x[V * j + k] = k % 2 ? bf16_hi(u[k / 2]) : bf16_lo(u[k / 2]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; k++) {
                float v = -INFINITY;
                if (i + k < a.vocab) {
                    if constexpr (V == 4) v = x0[i + k];
                    else v = bf16_to_f32(x0[i + k]);
                }
                x[V * j + k] = v;
            }
        }
    }
    // the thread's largest entry (indexes rise with j and k: the first of equal ones stays)
    float mx = -INFINITY;
    int mi = 0;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        x[j] = bm_clean(x[j]);
        if (x[j] > mx) {
            mx = x[j];
            mi = j;
        }
    }
    const bm_u64 top = mx > -INFINITY ? bm_key(mx, index(mi / V) + mi % V) : 0;
    const float wm = wave_max(mx);
    const bm_u64 bound = bm_bound<bm_u64, 64>(top, a.n);
    if (lane == 0) {
        wmax[wave] = wm;
        wbound[wave] = bound;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    bm_u64 T0 = wbound[0];
#pragma unroll
    for (int w = 1; w < BM_WAVES; w++) T0 = wbound[w] > T0 ? wbound[w] : T0;
    double sum = 0.0;
    if (M > -INFINITY) {
        // differences in 64 bits; of what is far below nothing is left
#pragma unroll
        for (int j = 0; j < VPT; j++) sum += (double)bm_exp2(fmax(((double)x[j] - (double)M) * BM_LOG2E, -300.0));
    }
    sum = bm_sum(sum);
    if (lane == 0) wsum[wave] = sum;
    if (top >= T0 && top > 0) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            const bm_u64 key = bm_key(x[j], index(j / V) + j % V);
            if (x[j] > -INFINITY && key >= T0) list[atomicAdd(&count, 1)] = key;
        }
    }
    __syncthreads();
    const size_t at = (size_t)row * a.shares + share;
    if (tid == 0) a.share[at] = {(wsum[0] + wsum[1]) + (wsum[2] + wsum[3]), M, 0.0f};
    // places by counting
    const int c = count;
    bm_u64 *const out = a.list + at * a.n;
    for (int i = tid; i < c; i += BM_THREADS) {
        const bm_u64 key = list[i];
        int rank = 0;
        for (int j = 0; j < c; j++) rank += list[j] > key;
        if (rank < a.n) out[rank] = key;
    }
    for (int i = c + tid; i < a.n; i += BM_THREADS) out[i] = 0;
}

// ---------------------------------------------------------------------------
// A candidate is ordered by its score (64 bits), then by its place among the sequence's candidates (beam * vocab +
// token, the lower first).
// ---------------------------------------------------------------------------
#define BS_THREADS 1024
#define BS_WAVES 16
#define BS_LIST 2048

struct BsKey {
    bm_u64 score;                     // 0: none
    unsigned at;                      // 2^32 - 1 - place
    __device__ __forceinline__ bool operator>(const BsKey &o) const { return score > o.score || (score == o.score && at > o.at); }
    __device__ __forceinline__ bool operator>=(const BsKey &o) const { return !(o > *this); }
};

__global__ __launch_bounds__(BS_THREADS) void beam_select(qk_beam_args a, int shares, const BmShare *share,
                                                          const bm_u64 *lists) {
    __shared__ double base[QK_BEAM_MAX];                         // score - log(sum); NaN: no candidates by logits
    __shared__ float most[QK_BEAM_MAX];                          // the largest logit
    __shared__ BsKey bounds[BS_WAVES], list[BS_LIST];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = blockIdx.x, n = a.n_out;
    const int row0 = q * a.beams;
    for (int b = wave; b < a.beams; b += BS_WAVES) {
        double v = NAN;
        if (!bm_idle(a.score, a.ended, row0 + b, a.vocab)) {
            const BmShare *const s = share + (size_t)(row0 + b) * shares;
            float M = -INFINITY;
            for (int i = lane; i < shares; i += 64) M = fmaxf(M, s[i].max);
            M = wave_max(M);
            double sum = 0.0;
            for (int i = lane; i < shares; i += 64)
                if (s[i].max > -INFINITY) sum += s[i].sum * exp((double)s[i].max - (double)M);
            sum = bm_sum(sum);
            if (M > -INFINITY) v = (double)a.score[row0 + b] - log(sum);
            if (lane == 0) most[b] = M;
        }
        if (lane == 0) base[b] = v;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    const int per = shares * n, all = per * a.beams;
    const bm_u64 *const mine = lists + (size_t)row0 * per;
    // candidate i: an entry of a list, or behind those a beam at its end
    auto candidate = [&](int i) {
        BsKey k = {0, 0};
        if (i < all) {
            const int b = i / per;
            const double s = base[b];
            if (s == s) {                                        // otherwise its lists hold nothing
                const bm_u64 e = mine[i];
                if (e) k = {bm_order(s + ((double)bm_value(e) - (double)most[b])), 0xffffffffu - ((unsigned)b * a.vocab + bm_index(e))};
            }
        } else if (i < all + a.beams && a.ended) {
            const int b = i - all;
            const float s = a.score[row0 + b];
            const int t = a.ended[row0 + b];
            if ((unsigned)t < (unsigned)a.vocab && fabsf(s) <= 3.402823466e38f)
                k = {bm_order((double)s), 0xffffffffu - ((unsigned)b * a.vocab + t)};
        }
        return k;
    };
    const int m = all + a.beams;
    BsKey top = {0, 0};
    for (int i = tid; i < m; i += BS_THREADS) {
        const BsKey k = candidate(i);
        if (k > top) top = k;
    }
    // a bound as in beam_rows, and by the places where scores are equal
    {
        BsKey b = {bm_bound<bm_u64, 64>(top.score, n), 0};
        const bool equal = top.score == b.score;
        const int above = __popcll(__ballot(top.score > b.score));
        if (b.score && above + __popcll(__ballot(equal)) > n) b.at = bm_bound<unsigned, 32>(equal ? top.at : 0u, n - above);
        if (lane == 0) bounds[wave] = b;
    }
    __syncthreads();
    BsKey T0 = bounds[0];
#pragma unroll
    for (int w = 1; w < BS_WAVES; w++)
        if (bounds[w] > T0) T0 = bounds[w];
    auto collect = [&]() {
        for (int i = tid; i < m; i += BS_THREADS) {
            const BsKey k = candidate(i);
            if (k.score && k >= T0) {
                const int at = atomicAdd(&count, 1);
                if (at < BS_LIST) list[at] = k;
            }
        }
        __syncthreads();
    };
    collect();
    if (count > BS_LIST) {
        // candidates beyond the list (many of one thread's are large): the bound's bits from the top, by
        // counting all of them, until they fit
        BsKey t = {0, 0};
        for (int b = 95; b >= 0; b--) {
            BsKey u = t;
            if (b >= 32) u.score |= 1ull << (b - 32);
            else u.at |= 1u << b;
            __syncthreads();
            if (tid == 0) count = 0;
            __syncthreads();
            int c = 0;
            for (int i = tid; i < m; i += BS_THREADS) {
                const BsKey k = candidate(i);
                c += k.score && k >= u;
            }
            c = (int)wave_sum((float)c);
            if (lane == 0) atomicAdd(&count, c);
            __syncthreads();
            const int got = count;
            if (got >= n) t = u;
            if (got >= n && got <= BS_LIST) break;
        }
        T0 = t;
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        collect();
    }
    const int c = count;
    const size_t o = (size_t)q * n;
    for (int i = tid; i < c; i += BS_THREADS) {
        const BsKey key = list[i];
        int rank = 0;
        for (int j = 0; j < c; j++) rank += list[j] > key;
        if (rank < n) {
            const unsigned place = 0xffffffffu - key.at;
            a.parent[o + rank] = row0 + (int)(place / a.vocab);
            a.token[o + rank] = (int)(place % a.vocab);
            a.score_out[o + rank] = (float)bm_double(key.score);
        }
    }
    for (int i = c + tid; i < n; i += BS_THREADS) {
        a.parent[o + i] = a.token[o + i] = -1;
        a.score_out[o + i] = -INFINITY;
    }
}

// Entries a thread: few for few rows, whose shares have to fill the card, and for many places (BM_LIST).
static int vpt(int rows, int vocab, int n) {
    if (n > 32) return 8;
    if (n > 16) return 16;
    return (long)rows * vocab < 4 << 20 ? 8 : 32;
}

static int row_shares(int vocab, int v) { return (vocab + BM_THREADS * v - 1) / (BM_THREADS * v); }

extern "C" size_t qk_beam_ws_bytes(int seqs, int beams, int vocab, int n_out) {
    const int rows = seqs * beams, shares = row_shares(vocab, vpt(rows, vocab, n_out));
    return (size_t)rows * shares * (sizeof(BmShare) + sizeof(bm_u64) * n_out);
}

template <typename T>
static void rows_launch(const BmRows &r, int rows, int v, hipStream_t s) {
    const dim3 grid((unsigned)rows, (unsigned)r.shares);
    if (v == 8) beam_rows<T, 8><<<grid, BM_THREADS, 0, s>>>(r);
    else if (v == 16) beam_rows<T, 16><<<grid, BM_THREADS, 0, s>>>(r);
    else beam_rows<T, 32><<<grid, BM_THREADS, 0, s>>>(r);
}

extern "C" int qk_beam_launch(const qk_beam_args *a, hipStream_t s) {
    const int rows = a->seqs * a->beams, v = vpt(rows, a->vocab, a->n_out), shares = row_shares(a->vocab, v);
    BmShare *const share = (BmShare *)a->ws;
    bm_u64 *const lists = (bm_u64 *)(share + (size_t)rows * shares);
    const BmRows r = {a->logits, a->row_stride, a->vocab, a->n_out, shares, a->score, a->ended, share, lists};
    if (a->bf16) rows_launch<uint16_t>(r, rows, v, s);
    else rows_launch<float>(r, rows, v, s);
    beam_select<<<(unsigned)a->seqs, BS_THREADS, 0, s>>>(*a, shares, share, lists);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
