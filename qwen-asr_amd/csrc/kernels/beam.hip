// beam.hip - the best continuations of a sequence's beams: of the candidates (beam b, token i)
// the n with the largest
//
//   score_b + x_i - M_b - log(sum_i e^(x_i - M_b)),   M_b = max_i x_i
//
// by falling score, equal ones by b, then by falling x, then by i.  One pass over the logits:
//
//   beam_rows    block (share of a row): its maximum and sum of exponentials, and its entries from a threshold
//                on that n of them reach: with the threads in n groups or more, the least of the
//                groups' maxima, which about 3 n do (of a share that leaves groups empty: the n-th
//                largest of a wave's threads').  Of more than a list holds, 32 to 128 by n, those from the step of their
//                range on that n reach; of equal ones (forbidden entries of the type's lowest value), and
//                where too many are in one step, the n-th largest value by its bits, and the lowest indexes of that.
//   beam_select  block (sequence): each beam's logarithm from its shares; a bound from the shares' largest
//                entries (the n-th of them by counting; of many the waves' n-th largest, or the steps of their
//                range), the entries of the shares that reach it, fewer of these by steps, and the n best.  What a step holds too many of is cut by the bits of
//                score and place.
//
// Measured: 16 x 8 beams of 151936 fp32 entries, 16 places, one beam in eight at its end: 31 us, rows 22 (78 MB, 14 without
// lists and exponentials: exponentials 2 to 3, entries to the lists 5), choice 10 (a chain of loads, logarithms
// and bounds in one block a sequence); 1 x 4 beams, 4 places: 4 and 8 us; 8 x 16 beams, 32 places: 37; 2 x 32 beams, 64 places:
// 37; 8 x 8 beams of equal logits, 16 places: 66; 1 x 64, 64 places: 257 (the bits of score, logit and place over all
// lists in one block; from the first bit on, not the first that differs, 956).
// Exponentials of 64-bit differences took 3 us more, a bound by the n-th largest thread and every list in order 8.  Lists brought
// in order by counting, and a block's bounds by bits alone: 8 x 16 beams 52, 7 x 14 beams of 38397, 28 places 53 (22),
// 2 x 32, 64 places 11.1 ms (a loose bound for the shares, thousands of candidates, 96 bits for all of them).
//
// Exponentials: log2(e) x in two fp32 terms, its whole part into the exponent, v_exp_f32 (1 ulp) of the rest, where the
// share's maximum lies within 30 of 0 (no x is subtracted from then, so nothing is rounded before); otherwise of
// x - M in 64 bits.  Pairs are added in fp32 (a sum is off by less than 2^-23 + ln 2 2^-25 + 2^-24 of itself; of rows of
// one to three entries 1.0 x 2^-23 at most was measured), everything else, shares joined, logarithms and scores, in 64 bits,
// in an order that does not depend on the run or on the rows' alignment: equal beams have equal scores.  Entries are
// compared as whole numbers (the value's order in the upper half, the index below, the lower one
// first), so equal ones are in order and every choice is unique.
#include "common.h"
#include "qk_kernels.h"
#include "qwen_asr_hip.h"

#include <limits.h>
#include <math.h>

#define BM_THREADS 256
#define BM_WAVES 4
#define BM_PART 512                   // entries from a threshold on of a wave
#define BM_LOG2E 1.4426950408889634

typedef unsigned long long bm_u64;

struct BmShare {                      // of a row
    double sum;                       // of e^(x - ref)
    float ref;
    int count;                        // entries listed
    bm_u64 best;                      // the largest entry; without an index (0 in its place) where it is not known; 0: none
};

// What is no number is no entry, +inf the largest number.  Asked for outright: of a maximum, a minimum or a middle with
// infinite constants the compiler leaves the minimum alone, which takes no number for the constant.  Largest by the bits:
// as whole numbers the positive ones are in order, and all negative ones below them.
__device__ __forceinline__ float bm_clean(float x) {
    return __int_as_float(min(__float_as_int(x == x ? x : -INFINITY), 0x7f7fffff));
}

// the order of values (-0 is 0), and of entries: larger first, then the lower index; 0 is none
__device__ __forceinline__ unsigned bm_rank(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ bm_u64 bm_key(float x, unsigned i) { return (bm_u64)bm_rank(x) << 32 | (0xffffffffu - i); }
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

// 2^t, -300 <= t < 127
__device__ __forceinline__ float bm_exp2(double t) {
    const double magic = 6755399441055744.0, z = t + magic;      // 1.5 2^52: t's whole part in the low word
    const float f = (float)(t - (z - magic));
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(f), (int)(unsigned)(bm_u64)__double_as_longlong(z));
}

// e^x for |x| of tens, e^-80 below (nothing beside a largest one of e^-30): x log2(e) less its whole part, that by adding
// 1.5 2^23, into the exponent's place.  Every product is part of an fma of its own: a product that is used twice may be
// taken unrounded in one of the places, and rounded in the other.  Off by v_exp_f32's 1 ulp, 2^-23, and what two fmas
// round of a number up to 1/2, ln 2 2^-25.
__device__ __forceinline__ float bm_exp(float x) {
    const float magic = 12582912.0f, L = 1.44269504e+00f, L2 = 1.92596299e-08f;
    x = fmaxf(x, -80.0f);
    const float z = fmaf(x, L, magic), f = fmaf(x, L2, fmaf(x, L, magic - z));
    return __uint_as_float(__float_as_uint(__builtin_amdgcn_exp2f(f)) + (__float_as_uint(z) << 23));
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
    int vocab, n, shares, width;   // entries of a share: a multiple of 8, BM_THREADS VPT at most
    const float *score;
    const int *ended;
    BmShare *share;                   // [rows][shares]
    bm_u64 *list;                     // [rows][shares][bm_slots(n)]
    bool late;                        // idle rows are found out behind the loads
};

// entries that a share lists at most: a power of two
__host__ __device__ __forceinline__ int bm_slots_log(int n) { return n <= 8 ? 5 : n <= 32 ? 6 : 7; }

// a beam that takes no part with its logits: one at its end, one without a score
__device__ __forceinline__ bool bm_idle(const float *score, const int *ended, int row, int vocab) {
    const float s = score[row];
    const int e = ended ? ended[row] : -1;
    return !(fabsf(s) <= 3.402823466e38f) || (unsigned)e < (unsigned)vocab;
}

template <typename T, int VPT>
__global__ __launch_bounds__(BM_THREADS) void beam_rows(BmRows a) {
    constexpr int V = 16 / sizeof(T), NV = VPT / V;              // entries of a load, loads
    __shared__ float wmax[BM_WAVES], wleast[BM_WAVES];
    __shared__ __attribute__((aligned(16))) bm_u64 list[BM_WAVES * BM_PART];
    __shared__ bm_u64 wkey[BM_WAVES];
    __shared__ double wsum[BM_WAVES];
    __shared__ int count[BM_WAVES], steps[BM_THREADS], above[BM_WAVES], cut, kept, place;
    __shared__ bm_u64 first;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int share = blockIdx.y, row = blockIdx.x;
    const T *const x0 = (const T *)a.logits + (size_t)row * a.stride;
    if (!a.late && bm_idle(a.score, a.ended, row, a.vocab)) return;
    // Shares and threads by index, whatever the row's alignment: equal rows have equal sums.  (Loads of 16 bytes
    // need no more alignment than the type's.)
    const int end = min((share + 1) * a.width, a.vocab);
    auto index = [&](int j) { return share * a.width + (j * BM_THREADS + tid) * V; };
    float x[VPT];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        // The planes before the share's end have no condition on a lane: behind one, loads would wait for each other.
        const int i = index(j), plane = share * a.width + j * BM_THREADS * V;
        if (plane + BM_THREADS * V <= end) {
            unsigned u[4];
            __builtin_memcpy(u, x0 + i, 16);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (V == 4) x[V * j + k] = __uint_as_float(u[k]);
                else x[V * j + k] = k % 2 ? bf16_hi(u[k / 2]) : bf16_lo(u[k / 2]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; k++) x[V * j + k] = -INFINITY;
            if (i + V <= end) {
                unsigned u[4];
                __builtin_memcpy(u, x0 + i, 16);
#pragma unroll
                for (int k = 0; k < V; k++) {
                    if constexpr (V == 4) x[V * j + k] = __uint_as_float(u[k]);
                    else x[V * j + k] = k % 2 ? bf16_hi(u[k / 2]) : bf16_lo(u[k / 2]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < V; k++)
                    if (i + k < end) {
                        if constexpr (V == 4) x[V * j + k] = x0[i + k];
                        else x[V * j + k] = bf16_to_f32(x0[i + k]);
                    }
            }
        }
    }
    if (a.late && bm_idle(a.score, a.ended, row, a.vocab)) return;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        x[j] = bm_clean(x[j]);
        mx = fmaxf(mx, x[j]);
    }
    // the least of the groups' maxima: 4, 8, 16, 32 or 64 groups of the block's threads
    float g = mx, all = mx;
    if (a.n > 4) {
        g = group_max<4>(g);
        if (a.n <= 32) g = group_max<8>(g);
        if (a.n <= 16) g = group_max<16>(g);
        if (a.n <= 8) g = group_max<32>(g);
        all = wave_max(g);
        g = -wave_max(-g);
    } else {
        g = all = wave_max(g);
    }
    if (lane == 0) {
        wmax[wave] = all;
        wleast[wave] = g;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    float T0 = fminf(fminf(wleast[0], wleast[1]), fminf(wleast[2], wleast[3]));
    if (T0 == -INFINITY) {
        // groups without entries (the row's last share): the n-th largest of a wave's threads instead
        const unsigned t = bm_bound<unsigned, 32>(mx > -INFINITY ? bm_rank(mx) : 0u, a.n);
        if (lane == 0) wkey[wave] = t;
        __syncthreads();
        const bm_u64 most = max(max(wkey[0], wkey[1]), max(wkey[2], wkey[3]));
        if (most) T0 = bm_value(most << 32);
    }
    T0 = fmaxf(T0, -3.402823466e38f);                 // what is -inf is no entry
    // the wave's entries from there on, into its part of the list
    bm_u64 *const part = list + BM_PART * wave;
    int n_part = 0;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        const bool in = x[j] >= T0;
        const bm_u64 m = __ballot(in);
        if (m) {
            const int to = n_part + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
            if (in && to < BM_PART) part[to] = bm_key(x[j], index(j / V) + j % V);
            n_part += __popcll(m);
        }
    }
    if (lane == 0) count[wave] = n_part;
    steps[tid] = 0;
    double sum = 0.0;
    const bool plain = fabsf(M) <= 30.0f;             // relative to 0, not to M
    if (plain) {
        float e[2];
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            e[j % 2] = bm_exp(x[j]);
            if (j % 2) sum += (double)(e[0] + e[1]);
        }
    } else if (M > -INFINITY) {
#pragma unroll
        for (int j = 0; j < VPT; j++) sum += (double)bm_exp2(fmax(((double)x[j] - (double)M) * BM_LOG2E, -300.0));
    }
    sum = bm_sum(sum);
    if (lane == 0) wsum[wave] = sum;
    __syncthreads();
    int before = 0, some = 0;
#pragma unroll
    for (int w = 0; w < BM_WAVES; w++) {
        before += w < wave ? count[w] : 0;
        some += count[w];
    }
    const size_t at = (size_t)row * a.shares + share;
    const int slots = bm_slots_log(a.n);
    bm_u64 *const out = a.list + (at << slots);
    BmShare result = {(wsum[0] + wsum[1]) + (wsum[2] + wsum[3]), plain ? 0.0f : M, some, M > -INFINITY ? bm_key(M, 0xffffffffu) : 0};
    bool like = max(max(count[0], count[1]), max(count[2], count[3])) > BM_PART;
    if (some <= 1 << slots) {
        for (int i = lane; i < n_part; i += 64) out[before + i] = part[i];
    } else if (!like) {
        // Fewer, by their values' places among BM_THREADS steps of one width from the threshold (no lower than 64 from
        // the largest) to the largest: those from the step on that n reach.
        const float from = fmaxf(T0, M - 64.0f), scale = M > from ? (BM_THREADS - 1) / (M - from) : 0.0f;
        auto step = [&](bm_u64 key) { return (int)fminf(fmaxf((bm_value(key) - from) * scale, 0.0f), BM_THREADS - 1.0f); };
        for (int i = lane; i < n_part; i += 64) atomicAdd(steps + step(part[i]), 1);
        if (tid == 0) place = 0;
        __syncthreads();
        const int here = steps[tid];
        int upto = here;                              // of this step and those above it
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_down(upto, d, 64);
            if (lane + d < 64) upto += v;
        }
        if (lane == 0) above[wave] = upto;
        __syncthreads();
#pragma unroll
        for (int w = 1; w < BM_WAVES; w++) upto += w > wave ? above[w] : 0;
        if (upto >= a.n && upto - here < a.n) {       // one thread's: more than n are listed
            cut = tid;
            kept = upto;
        }
        __syncthreads();
        if (kept <= 1 << slots) {
            result.count = kept;
            for (int i = lane; i < n_part; i += 64)
                if (step(part[i]) >= cut) out[atomicAdd(&place, 1)] = part[i];
        } else {
            like = true;
        }
    }
    if (like) {
        // Equal ones, or nearly: the n-th largest value v, its bits from the top; what is above it, and as many of v
        // as are missing, the lowest indexes first.
        unsigned r[VPT], v = 0;
#pragma unroll
        for (int j = 0; j < VPT; j++) r[j] = x[j] > -INFINITY ? bm_rank(x[j]) : 0u;
        __syncthreads();                              // every thread is behind the steps
        steps[tid] = 0;
        if (tid == 0) {
            place = 0;
            first = 0;
        }
        __syncthreads();
        for (int b = 31; b >= 0; b--) {
            const unsigned u = v | 1u << b;
            int c = 0;
#pragma unroll
            for (int j = 0; j < VPT; j++) c += __popcll(__ballot(r[j] >= u));
            if (lane == 0 && c) atomicAdd(steps + b, c);
            __syncthreads();
            if (steps[b] >= a.n) v = u;
        }
        int c = 0;
#pragma unroll
        for (int j = 0; j < VPT; j++) c += __popcll(__ballot(r[j] > v));
        if (lane == 0 && c) atomicAdd(steps + 32, c);
        int *const equal = steps + 64;                // [NV][BM_WAVES]
#pragma unroll
        for (int p = 0; p < NV; p++) {
            int e = 0;
#pragma unroll
            for (int k = 0; k < V; k++) e += __popcll(__ballot(r[V * p + k] == v));
            if (lane == 0) equal[BM_WAVES * p + wave] = e;
        }
        __syncthreads();
        const int missing = a.n - steps[32];
        int below = 0;                                // of v with lower indexes: those of the planes before, ...
#pragma unroll
        for (int p = 0; p < NV; p++) {
            int to = below;
#pragma unroll
            for (int w = 0; w < BM_WAVES; w++) {
                to += w < wave ? equal[BM_WAVES * p + w] : 0;
                below += equal[BM_WAVES * p + w];
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                const bm_u64 m = __ballot(r[V * p + k] == v);
                to += (int)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                const bool is = r[V * p + k] == v;
                if (r[V * p + k] > v || (is && to < missing)) {
                    const bm_u64 key = (bm_u64)r[V * p + k] << 32 | (0xffffffffu - (unsigned)(index(p) + k));
                    out[atomicAdd(&place, 1)] = key;
                    atomicMax(&first, key);
                }
                to += is;
            }
        }
        __syncthreads();
        result.count = a.n;
        result.best = first;
    }
    if (tid == 0) a.share[at] = result;
}

// ---------------------------------------------------------------------------
// A candidate is ordered by its score (64 bits), then by beam (the lower first), logit and token (the lower first).  Scores
// of one beam do not fall with the logit, so this is the order of the shares' lists, also where scores differ by
// less than 64 bits hold (beside a score of -1e30, or of +inf as the largest number).
// ---------------------------------------------------------------------------
#define BS_THREADS 1024
#define BS_WAVES (BS_THREADS / 64)
#define BS_LIST 4096
#define BS_COUNTED 256                // shares whose n-th largest is found by counting
#define BS_RANKED 128                 // candidates that are ranked as they are
#define BS_MANY 768
#define BS_ACTIVE 2048                // shares whose entries are looked at
#define BS_AT 60                      // bits of BsKey.at, in threes
#define BS_TOKEN ((1u << 20) - 1)

struct BsKey {
    bm_u64 score;                     // 0: none
    bm_u64 at;                        // 63 - beam in 6 bits, the logit's order in 32, 2^20 - 1 - token in 20
    __device__ __forceinline__ bool operator>(const BsKey &o) const { return score > o.score || (score == o.score && at > o.at); }
    __device__ __forceinline__ bool operator>=(const BsKey &o) const { return !(o > *this); }
};

__global__ __launch_bounds__(BS_THREADS) void beam_select(qk_beam_args a, int shares, const BmShare *share,
                                                          const bm_u64 *lists) {
    __shared__ double base[QK_BEAM_MAX];                         // score - log(sum); NaN: no candidates by logits
    __shared__ float most[QK_BEAM_MAX];                          // the largest logit
    __shared__ BsKey list[BS_LIST], nth;
    __shared__ int counts[3][8], count, n_active, active[BS_ACTIVE], entries[BS_ACTIVE], rank[BS_LIST], above[BS_WAVES], cut, kept;
    __shared__ bm_u64 lows[BS_WAVES], highs[BS_WAVES], least;
    int *const steps = rank;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = blockIdx.x, n = a.n_out;
    const int row0 = q * a.beams, cols = a.beams * shares, slots = bm_slots_log(n);
    share += (size_t)row0 * shares;
    lists += (size_t)row0 * shares << slots;
    const BmShare first = share[min(tid, cols - 1)];             // of what idle beams left nothing is looked at
    for (int b = wave; b < a.beams; b += BS_WAVES) {
        const BmShare *const s = share + (size_t)b * shares;
        const BmShare mx = s[min(lane, shares - 1)];
        const float score = a.score[row0 + b];
        const int end = a.ended ? a.ended[row0 + b] : -1;
        double v = NAN;
        if (fabsf(score) <= 3.402823466e38f && (unsigned)end >= (unsigned)a.vocab) {
            auto max_of = [](const BmShare &x) { return x.best ? bm_value(x.best) : -INFINITY; };
            float M = max_of(mx);
            for (int i = lane + 64; i < shares; i += 64) M = fmaxf(M, max_of(s[i]));
            M = wave_max(M);
            auto part = [&](const BmShare &x) {
                return x.best ? x.sum * exp((double)x.ref - (double)M) : 0.0;
            };
            double sum = lane < shares ? part(mx) : 0.0;
            for (int i = lane + 64; i < shares; i += 64) sum += part(s[i]);
            sum = bm_sum(sum);
            if (M > -INFINITY) v = (double)score - log(sum);
            if (lane == 0) most[b] = M;
        }
        if (lane == 0) base[b] = v;
    }
    if (tid == 0) count = n_active = 0;
    if (tid < 24) counts[tid / 8][tid % 8] = 0;
    __syncthreads();
    auto at_of = [](int b, unsigned order, unsigned token) {
        return (bm_u64)(QK_BEAM_MAX - 1 - b) << 52 | (bm_u64)order << 20 | (BS_TOKEN - token);
    };
    // (what is of no known index has the last: as good as that at least)
    auto key_of = [&](int b, bm_u64 e) {
        const double s = base[b];
        BsKey k = {0, 0};
        if (s == s && e) {
            k.score = bm_order(s + ((double)bm_value(e) - (double)most[b]));
            k.at = at_of(b, (unsigned)(e >> 32), (unsigned)e ? bm_index(e) : BS_TOKEN);
        }
        return k;
    };
    // beam b's candidate where it is at its end
    auto end_of = [&](int b) {
        BsKey k = {0, 0};
        if (b < a.beams && a.ended) {
            const float s = a.score[row0 + b];
            const int t = a.ended[row0 + b];
            if ((unsigned)t < (unsigned)a.vocab && fabsf(s) <= 3.402823466e38f)
                k = {bm_order((double)s), at_of(b, 0u, (unsigned)t)};
        }
        return k;
    };
    auto best_of = [&](int i, const BmShare &s) { return key_of((int)((unsigned)i / (unsigned)shares), s.best); };
    // a thread's largest candidate
    BsKey top = end_of(tid);
    if (tid < cols) {
        const BsKey k = best_of(tid, first);
        if (k > top) top = k;
    }
    for (int i = tid + BS_THREADS; i < cols; i += BS_THREADS) {
        const BsKey k = best_of(i, share[i]);
        if (k > top) top = k;
    }
    // A bound that at least n of the block's keys reach, and at most `enough` where it can be: the bits of the n-th
    // largest from the top, three at a time, until so few are left.  own(u): how many of the thread's keys reach u.
    // Its score is one of low .. high, so it has the bits that these begin with.
    auto bound = [&](int enough, bm_u64 low, bm_u64 high, auto own) {
        const int open = low == high ? 0 : (66 - __clzll((long long)(low ^ high))) / 3 * 3;
        BsKey t = {open < 64 ? high >> open << open : 0, 0};
        for (int b = BS_AT + open - 3, turn = 0; b >= 0; b -= 3, turn = turn == 2 ? 0 : turn + 1) {
            auto with = [&](unsigned k) {                        // t with k in the bits b .. b + 2
                BsKey u = t;
                if (b >= BS_AT) u.score |= (bm_u64)k << (b - BS_AT);
                else u.at |= (bm_u64)k << b;
                return u;
            };
            int mine = 0;                                        // of lane k: the wave's keys that reach with(k)
#pragma unroll
            for (int k = 1; k < 8; k++) {
                const int c = own(with(k));
                if (lane == k) mine = c;
            }
            if (lane > 0 && lane < 8 && mine) atomicAdd(&counts[turn][lane], mine);
            if (tid < 8) counts[turn == 2 ? 0 : turn + 1][tid] = 0;        // its last readers are two barriers back
            __syncthreads();
            int got = INT_MAX, most = 0;
#pragma unroll
            for (int k = 1; k < 8; k++) {
                const int c = counts[turn][k];
                if (c >= n) {
                    most = k;
                    got = c;
                }
            }
            t = with(most);
            if (got <= enough) break;
        }
        __syncthreads();
        if (tid < 24) counts[tid / 8][tid % 8] = 0;
        __syncthreads();
        return t;
    };
    // Candidates by their scores' places among BS_THREADS steps of one width from `from` to the best: `cut` is the
    // step from which on at least n of those counted are, `kept` how many.  count(add): the thread's.
    double from = 0.0, scale = 0.0;
    auto range = [&](bm_u64 lo, bm_u64 hi) {                     // steps from lo, no lower than e^-64 of the best
        const double best = bm_double(hi);
        from = lo ? fmax(bm_double(lo), best - 64.0) : best - 64.0;
        scale = best > from ? (BS_THREADS - 1) / (best - from) : 0.0;
    };
    auto step = [&](const BsKey &k) { return (int)fmin(fmax((bm_double(k.score) - from) * scale, 0.0), BS_THREADS - 1.0); };
    auto count_steps = [&](auto all) {
        steps[tid] = 0;
        if (tid == 0) cut = kept = 0;
        __syncthreads();
        all([&](const BsKey &k) { atomicAdd(steps + step(k), 1); });
        __syncthreads();
        const int here = steps[tid];
        int upto = here;                                         // of this step and those above it
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_down(upto, d, 64);
            if (lane + d < 64) upto += v;
        }
        if (lane == 0) above[wave] = upto;
        __syncthreads();
#pragma unroll
        for (int w = 1; w < BS_WAVES; w++) upto += w > wave ? above[w] : 0;
        if (upto >= n && upto - here < n) {                      // one thread's, or none's: fewer than n
            cut = tid;
            kept = upto;
        }
        __syncthreads();
    };
    // A bound that n of the threads' candidates reach, and few more: of few threads' the n-th largest, by counting
    BsKey T0 = {0, 0};
    bm_u64 best = top.score;
    if (max(cols, a.beams) <= BS_COUNTED) {
        constexpr int PARTS = BS_THREADS / BS_COUNTED;
        const int i = tid % BS_COUNTED, c = max(cols, a.beams);
        if (tid < c) list[tid] = top;
        if (tid < BS_COUNTED) rank[tid] = 0;
        __syncthreads();
        if (i < c) {
            const BsKey one = list[i];
            int larger = 0;
#pragma unroll 4
            for (int j = tid / BS_COUNTED; j < c; j += PARTS) larger += list[j] > one || (j < i && list[j] >= one);
            atomicAdd(rank + i, larger);
        }
        if (tid == 0) nth = BsKey{0, 0};
        __syncthreads();
        if (tid < c) {
            if (rank[tid] == n - 1) nth = top;
            if (rank[tid] == 0) highs[0] = top.score;
        }
        __syncthreads();
        T0 = nth;
        best = highs[0];
    } else if (n <= 16) {
        // of few places the waves' n-th largest do, by the scores' upper halves (4 beams, 4 places: 8.1 us, by steps 9.5)
        const unsigned high = (unsigned)(top.score >> 32), t = bm_bound<unsigned, 32>(high, n);
        unsigned most = high;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, d, 64));
        if (lane == 0) {
            highs[wave] = (bm_u64)most << 32 | 0xffffffffu;
            lows[wave] = (bm_u64)t << 32;
        }
        __syncthreads();
        best = 0;
#pragma unroll
        for (int w = 0; w < BS_WAVES; w++) {
            best = max(best, highs[w]);
            T0.score = max(T0.score, lows[w]);
        }
    } else {
        bm_u64 low = top.score ? top.score : ~0ull;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            best = max(best, __shfl_xor(best, d, 64));
            low = min(low, __shfl_xor(low, d, 64));
        }
        if (lane == 0) {
            highs[wave] = best;
            lows[wave] = low;
        }
        if (tid == 0) least = ~0ull;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BS_WAVES; w++) {
            best = max(best, highs[w]);
            low = min(low, lows[w]);
        }
        range(low, best);
        count_steps([&](auto add) {
            if (top.score) add(top);
        });
        if (kept > 64 + n) {                                     // equal ones, or nearly
            T0 = bound(64 + n, low, best, [&](const BsKey &u) { return (int)__popcll(__ballot(top >= u)); });
        } else if (kept) {
            if (top.score && step(top) >= cut) atomicMin(&least, top.score);
            __syncthreads();
            T0.score = least;
        }
    }
    __syncthreads();
    if (tid == 0) count = 0;
    for (int i = tid; i < cols; i += BS_THREADS) {
        const BmShare s = i == tid ? first : share[i];
        const BsKey k = best_of(i, s);
        // (what is of no known index may be of any)
        if (k.score > T0.score || (k.score && k.score == T0.score && (k.at | BS_TOKEN) >= T0.at)) {
            const int at = atomicAdd(&n_active, 1);
            if (at < BS_ACTIVE) {
                active[at] = i;
                entries[at] = s.count;
            }
        }
    }
    __syncthreads();
    // all candidates that may reach the bound: of the active shares (of all, where they are too many for a list), and ends
    const bool every = n_active > BS_ACTIVE;
    const long m = (long)(every ? cols : n_active) << slots;
    auto each = [&](auto take) {
        // four loads on their way at once, of what no share listed as well
        for (long i0 = tid; i0 < m; i0 += 4 * BS_THREADS) {
            bm_u64 e[4];
            int l[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const long i = min(i0 + u * BS_THREADS, m - 1);
                const int k = (int)(i >> slots), slot = (int)i & ((1 << slots) - 1);
                l[u] = every ? k : active[k];
                e[u] = lists[((size_t)l[u] << slots) + slot];
                if (i0 + u * BS_THREADS >= m || slot >= (every ? share[l[u]].count : entries[k])) e[u] = 0;
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int b = (int)((unsigned)l[u] / (unsigned)shares);
                if (i0 + u * BS_THREADS < m) take(key_of(b, e[u]));
            }
        }
        take(end_of(tid));
    };
    auto hit = [&](const BsKey &k) { return k.score && k >= T0; };
    each([&](const BsKey &k) {
        if (hit(k)) {
            const int at = atomicAdd(&count, 1);
            if (at < BS_LIST) list[at] = k;
        }
    });
    __syncthreads();
    range(T0.score, best);
    // fewer than n: all
    auto from_cut = [&](const BsKey &k) { return hit(k) && step(k) >= cut; };
    if (count > BS_LIST) {
        // candidates beyond the list (many shares that reach the bound many times over)
        count_steps([&](auto add) {
            each([&](const BsKey &k) {
                if (hit(k)) add(k);
            });
        });
        if (kept > BS_LIST) {
            T0 = bound(BS_LIST, T0.score, best, [&](const BsKey &u) {
                int c = 0;
                each([&](const BsKey &k) { c += k.score && k >= u; });
                return (int)wave_sum((float)c);
            });
            if (tid == 0) cut = 0;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        each([&](const BsKey &k) {
            if (from_cut(k)) list[atomicAdd(&count, 1)] = k;
        });
        __syncthreads();
        range(T0.score, best);
    }
    if (count > BS_RANKED) {
        // fewer of the list
        BsKey mine[BS_LIST / BS_THREADS];
#pragma unroll
        for (int j = 0; j < BS_LIST / BS_THREADS; j++) {
            const int i = tid + BS_THREADS * j;
            mine[j] = i < count ? list[i] : BsKey{0, 0};
        }
        count_steps([&](auto add) {
#pragma unroll
            for (int j = 0; j < BS_LIST / BS_THREADS; j++)
                if (mine[j].score) add(mine[j]);
        });
        if (kept > BS_MANY) {                                    // equal ones, or nearly
            T0 = bound(64 + n, T0.score, best, [&](const BsKey &u) {
                int c = 0;
#pragma unroll
                for (int j = 0; j < BS_LIST / BS_THREADS; j++) c += __popcll(__ballot(mine[j] >= u));
                return c;
            });
            if (tid == 0) cut = 0;
        }
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < BS_LIST / BS_THREADS; j++)
            if (from_cut(mine[j])) list[atomicAdd(&count, 1)] = mine[j];
        __syncthreads();
    }
    const int c = count;
    const size_t o = (size_t)q * n;
    // places by counting, `parts` threads an entry
    for (int i = tid; i < c; i += BS_THREADS) rank[i] = 0;
    __syncthreads();
    const int parts = c <= 64 ? BS_THREADS / 64 : c <= 256 ? BS_THREADS / 256 : 1, width = BS_THREADS / parts;
    for (int i = tid % width; i < c; i += width) {
        const BsKey key = list[i];
        int above = 0;
#pragma unroll 4
        for (int j = tid / width; j < c; j += parts) above += list[j] > key;
        atomicAdd(rank + i, above);
    }
    __syncthreads();
    for (int i = tid; i < c; i += BS_THREADS) {
        if (rank[i] >= n) continue;
        const BsKey key = list[i];
        a.parent[o + rank[i]] = row0 + QK_BEAM_MAX - 1 - (int)(key.at >> 52);
        a.token[o + rank[i]] = (int)(BS_TOKEN - ((unsigned)key.at & BS_TOKEN));
        a.score_out[o + rank[i]] = (float)bm_double(key.score);
    }
    for (int i = c + tid; i < n; i += BS_THREADS) {
        a.parent[o + i] = a.token[o + i] = -1;
        a.score_out[o + i] = -INFINITY;
    }
}

// Entries a thread: few for few rows, whose shares have to fill the card, and not too many for many places (8 x 20
// beams, 40 places: 8 entries 54 us, 16 46, 32 44; 8 x 16, 32 places: 43, 37, 39; 2 x 5 of 300, 64 places: 16, 16, 18).
static int vpt(int rows, int vocab, int n) {
    if (n > 16) return 16;
    return (long)rows * vocab < 4 << 20 ? 8 : 32;
}

static int row_shares(int vocab, int v) { return (vocab + BM_THREADS * v - 1) / (BM_THREADS * v); }

extern "C" size_t qk_beam_ws_bytes(int seqs, int beams, int vocab, int n_out) {
    const int rows = seqs * beams, shares = row_shares(vocab, vpt(rows, vocab, n_out));
    return (size_t)rows * shares * (sizeof(BmShare) + (sizeof(bm_u64) << bm_slots_log(n_out)));
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
    // even shares: one of few entries would leave groups of threads with few or none
    const int width = ((a->vocab + shares - 1) / shares + 7) / 8 * 8;
    BmShare *const share = (BmShare *)a->ws;
    bm_u64 *const lists = (bm_u64 *)(share + (size_t)rows * shares);
    // few rows: a chain of loads less; many: the bytes of idle ones
    const BmRows r = {a->logits, a->row_stride, a->vocab, a->n_out, shares, width, a->score, a->ended, share, lists,
                      (long)rows * a->vocab < 4 << 20};
    if (a->bf16) rows_launch<uint16_t>(r, rows, v, s);
    else rows_launch<float>(r, rows, v, s);
    beam_select<<<(unsigned)a->seqs, BS_THREADS, 0, s>>>(*a, shares, share, lists);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
