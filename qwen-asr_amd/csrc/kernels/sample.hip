// sample.hip - one token per row of logits: temperature, top-k, top-p, min-p,
// then a draw at a given random number.
//
// With M the row's largest logit, a_i = (M - l_i) / T and w_i = e^(-a_i):
//   top-k  the k entries that come first in the order (larger logit, then lower index);
//   top-p  of those, entry i while the weights before it sum to less than top_p times
//          the weight of them all (the first is always kept);
//   min-p  of those, the ones with w_i >= min_p;
//   token  the first index whose weights up to and including it sum to more than u
//          times the weight of all that is left.
//
// No sort: what the answer needs of the order is two thresholds.  Weights are
// held as integers, w_i 2^43 cut off (2^20 entries sum to less than 2^64), so sums do
// not depend on the order of the atomics and every launch sees the same ones; what
// is cut is below 2^-43 of the largest weight for each entry, against the 2^-24 of an
// fp32 exponential.  y_i = a_i log2(e) is held as the sum of two fp32 numbers (the
// difference and the product with their rounding errors), so the weight's only
// errors are those of v_exp_f32 (1 ulp) and of its argument's fraction (2^-25).
//
// Four launches over blocks of the row, each reading the row once (from the
// caches after the first time):
//   sample_max    largest and smallest finite logit of each block's share
//   sample_hist   count (for top-k) and weight (for top-p) of SM_BINS classes of y, evenly
//                 over the row's range (at most 32 log2(e): the last class weighs 0)
//   sample_pick   from the classes' running sums: which are kept whole, and which hold
//                 a threshold.  Entries of the latter go to a short list, the former
//                 are summed per 1024 entries
//   sample_draw   one block a row: orders the list by counting, finds both
//                 thresholds, and walks the sums down to the one entry
// A row whose threshold classes hold more than SM_CAND entries (nearly equal
// logits) takes a radix selection over the row in the last launch instead.
//
// Bound by four kernels in a row for one row (151936 entries: 4 + 5 + 7 + 7 us, where a
// call of one launch takes 8), and for many by three readings of the rows and the last
// kernel's one block a row (64 rows: 9 + 15 + 18 + 9 us, where one reading takes 8), more than by
// the arithmetic of the weights (about 40 vector instructions each, in hist for every
// entry, in pick for those kept: hist takes 10 of its 15 us without any).  Rows that take
// the first entry alone (temperature 0, top-k 1) ask for no classes: 17 us for one, 29 for 64.
#include "common.h"
#include "qk_kernels.h"
#include "qwen_asr_hip.h"

#include <math.h>

#define SM_BINS 2048
#define SM_SUB 1024               // entries per partial sum
#define SM_MAX_SUBS 1024          // so at most 2^20 entries
#define SM_CAND 1024
#define SM_MAX_BLOCKS 256
#define SM_ONE (1ull << 43)

struct SmPar {
    float M, c, c_lo;             // largest logit; log2(e) / T in two parts
    float scale;                  // classes per unit of y
    float lim, lim_lo;            // largest y that min-p keeps, in two parts
    float top_p;                  // >= 1: off
    int k;                        // 0: off
    int none;                     // no entry at all
};

struct SmRow {                    // one row's part of the workspace
    unsigned long long weight[SM_BINS];
    unsigned count[SM_BINS];
    float max[SM_MAX_BLOCKS], min[SM_MAX_BLOCKS];
    SmPar par;
    unsigned n_cand, pad[2];
    int lo, hi, bk;               // classes below lo are kept whole; lo .. hi and bk hold the thresholds
    unsigned count_k;             // entries before class bk
    unsigned long long weight_k, weight_lo, weight_all, pad2;   // before bk, before lo, of the row
    unsigned long long cand[SM_CAND];                           // the logit's bits, the index
    unsigned long long sub[SM_MAX_SUBS];
};

// the value as it counts: what is no number never does, -0 is 0
__device__ __forceinline__ float sm_clean(float l) { return l != l ? -INFINITY : l + 0.0f; }

__device__ __forceinline__ unsigned sm_key(float l) {
    const unsigned u = __float_as_uint(l);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

// the order: larger is earlier
__device__ __forceinline__ unsigned long long sm_comp(float l, int i) {
    return (unsigned long long)sm_key(l) << 32 | (0xffffffffu - (unsigned)i);
}

struct SmY {
    float y, lo;                  // y + lo
    int bin;                      // not falling with y
};

// Any l: what is -infinity or no number gets the last class, which weighs nothing.
__device__ __forceinline__ SmY sm_y(const SmPar &p, float l) {
    // M - l and its rounding error
    const float d0 = p.M - l, bb = d0 - p.M, e0 = (p.M - (d0 - bb)) - (l + bb);
    const bool top = l == p.M;                   // also inf - inf
    const float d = top ? 0.0f : d0, e = top ? 0.0f : e0;
    SmY r;
    r.y = d * p.c;
    r.lo = fmaf(e, p.c, fmaf(d, p.c_lo, fmaf(d, p.c, -r.y)));
    r.bin = (int)fminf(r.y * p.scale, (float)(SM_BINS - 1));
    return r;
}

__device__ __forceinline__ bool sm_likely(const SmPar &p, const SmY &v) {
    return (v.y - p.lim) + (v.lo - p.lim_lo) <= 0.0f;
}

__device__ __forceinline__ unsigned long long sm_weight(const SmY &v) {
    const float n = rintf(v.y);
    const float e = __builtin_amdgcn_exp2f(-((v.y - n) + v.lo));         // 2^(-1/2) .. 2^(1/2)
    const unsigned m = v.bin == SM_BINS - 1 ? 0u : (unsigned)(e * 16777216.0f);
    return ((unsigned long long)m << 19) >> ((int)n & 63);
}

__device__ __forceinline__ SmPar sm_par(const qk_sample_args &a, const SmRow &w, int row, int nb) {
    __shared__ float smx, smn;
    const float T = a.temperature ? a.temperature[row] : 1.0f, tp = a.top_p ? a.top_p[row] : 1.0f,
                mp = a.min_p ? a.min_p[row] : 0.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (threadIdx.x < 64) {
        float mx = -INFINITY, mn = INFINITY;
        for (int i = threadIdx.x; i < nb; i += 64) {
            mx = fmaxf(mx, w.max[i]);
            mn = fminf(mn, w.min[i]);
        }
        mx = wave_max(mx);
        mn = -wave_max(-mn);
        if (threadIdx.x == 0) {
            smx = mx;
            smn = mn;
        }
    }
    __syncthreads();
    SmPar p;
    p.M = smx;
    p.none = smx == -INFINITY;
    const bool greedy = !(T > 0.0f);
    const double c = fmin((greedy ? 1.0 : 1.0 / (double)T) * 1.4426950408889634074, 1e30);
    p.c = (float)c;
    p.c_lo = (float)(c - (double)p.c);
    if (greedy) k = 1;
    p.k = k <= 0 || k >= a.vocab ? 0 : k;
    p.top_p = tp != tp ? 1.0f : fmaxf(tp, 0.0f);
    p.lim = INFINITY;
    p.lim_lo = 0.0f;
    if (mp > 0.0f) {
        const double lim = -log2((double)fminf(mp, 1.0f));
        p.lim = (float)lim;
        p.lim_lo = (float)(lim - (double)p.lim);
    }
    if (p.k == 1) {                              // the first entry alone, whatever it weighs: no class is asked for
        p.top_p = 1.0f;
        p.lim = INFINITY;
        p.lim_lo = 0.0f;
    }
    const float range = (p.M - smn) * p.c * 1.000001f;       // the lowest entry is not in the last class
    p.scale = fminf((float)(SM_BINS - 1) / (range < 46.166242f ? range : 46.166242f), 1e30f);
    return p;
}

// inclusive sum over the wave: rows of 16 by shifts, then the rows' ends passed on
__device__ __forceinline__ unsigned long long sm_wave_scan(unsigned long long v) {
#define SM_STEP(CTRL, ROWS)                                                                                 \
    {                                                                                                       \
        const unsigned l = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, false);      \
        const unsigned h = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xF, false); \
        v += (unsigned long long)h << 32 | l;                                                               \
    }
    SM_STEP(0x111, 0xF) SM_STEP(0x112, 0xF) SM_STEP(0x114, 0xF) SM_STEP(0x118, 0xF)      // row_shr 1, 2, 4, 8
    SM_STEP(0x142, 0xA) SM_STEP(0x143, 0xC)                                              // row_bcast 15, 31
#undef SM_STEP
    return v;
}

// ... of the whole wave, in its last lane
__device__ __forceinline__ unsigned long long sm_wave_sum(unsigned long long v) { return sm_wave_scan(v); }

// exclusive sum over the block of one value per thread, and the sum of all
template <int NT>
__device__ __forceinline__ unsigned long long sm_scan(unsigned long long v, unsigned long long &total) {
    constexpr int NW = NT / 64;
    __shared__ unsigned long long ws[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned long long x = sm_wave_scan(v);
    __syncthreads();
    if (lane == 63) ws[wave] = x;
    __syncthreads();
    unsigned long long base = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        if (i < wave) base += ws[i];
        all += ws[i];
    }
    total = all;
    return base + x - v;
}

__global__ __launch_bounds__(256) void sample_max(qk_sample_args a, int nb) {
    const int row = blockIdx.x / nb, b = blockIdx.x % nb;
    SmRow &w = ((SmRow *)a.ws)[row];
    const float *x = a.logits + (size_t)row * a.row_stride;
    // the classes are cleared here, a launch before they are counted
    for (int i = b * 256 + threadIdx.x; i < SM_BINS; i += nb * 256) {
        w.weight[i] = 0;
        w.count[i] = 0;
    }
    if (b == 0 && threadIdx.x == 0) w.n_cand = 0;
    float mx = -INFINITY, mn = INFINITY;
#pragma unroll 8
    for (int i = b * 256 + threadIdx.x; i < a.vocab; i += nb * 256) {
        const float l = sm_clean(x[i]);
        mx = fmaxf(mx, l);
        if (l > -INFINITY) mn = fminf(mn, l);
    }
    __shared__ float smx[4], smn[4];
    mx = wave_max(mx);
    mn = -wave_max(-mn);
    if ((threadIdx.x & 63) == 0) {
        smx[threadIdx.x >> 6] = mx;
        smn[threadIdx.x >> 6] = mn;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        w.max[b] = fmaxf(fmaxf(smx[0], smx[1]), fmaxf(smx[2], smx[3]));
        w.min[b] = fminf(fminf(smn[0], smn[1]), fminf(smn[2], smn[3]));
    }
}

// Blocks of 1024 threads: each adds its classes to the row's with one atomic a
// class, so few large blocks.  The counts are left out without top-k, the weights
// without top-p.
__global__ __launch_bounds__(1024) void sample_hist(qk_sample_args a, int nb, int nh) {
    const int row = blockIdx.x / nh, b = blockIdx.x % nh;
    SmRow &w = ((SmRow *)a.ws)[row];
    __shared__ unsigned long long hw[SM_BINS];
    __shared__ unsigned hc[SM_BINS];
    for (int i = threadIdx.x; i < SM_BINS; i += 1024) {
        hw[i] = 0;
        hc[i] = 0;
    }
    const SmPar p = sm_par(a, w, row, nb);                   // its barrier orders the clearing, too
    if (b == 0 && threadIdx.x == 0) w.par = p;
    const bool counts = p.k > 1, weights = p.top_p < 1.0f;
    if (p.none || !(counts || weights)) return;              // nothing asks for the order
    const float *x = a.logits + (size_t)row * a.row_stride;
    constexpr int U = 4;
    for (int i0 = b * 1024 + threadIdx.x; i0 < a.vocab; i0 += nh * 1024 * U) {
        float l[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            const long i = i0 + (long)j * nh * 1024;
            l[j] = i < a.vocab ? x[i] : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < U; j++) {
            const SmY v = sm_y(p, l[j]);
            if (v.bin == SM_BINS - 1) continue;
            if (weights) atomicAdd(&hw[v.bin], sm_weight(v));
            if (counts) atomicAdd(&hc[v.bin], 1u);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SM_BINS; i += 1024) {
        if (hw[i]) atomicAdd(&w.weight[i], hw[i]);
        if (hc[i]) atomicAdd(&w.count[i], hc[i]);
    }
}

struct SmCut {
    int lo, hi, bk;
    unsigned count_k;
    unsigned long long weight_k, weight_lo, weight_all;
};

// which classes hold the thresholds (256 threads; n, v: this thread's SM_PER classes)
#define SM_PER (SM_BINS / 256)
__device__ __forceinline__ SmCut sm_cut(const SmPar &p, const unsigned (&n)[SM_PER],
                                        const unsigned long long (&v)[SM_PER]) {
    __shared__ SmCut sc;
    __shared__ unsigned long long s_end_k, ws[4][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool by_k = p.k > 0, by_p = p.top_p < 1.0f;
    unsigned nt = 0;
    unsigned long long vt = 0;
#pragma unroll
    for (int i = 0; i < SM_PER; i++) {
        nt += n[i];
        vt += v[i];
    }
    const unsigned long long ns = sm_wave_scan(nt), vs = sm_wave_scan(vt);
    if (lane == 63) {
        ws[wave][0] = ns;
        ws[wave][1] = vs;
    }
    if (threadIdx.x == 0) sc = {SM_BINS, -1, -1, 0, 0, 0, 0};
    __syncthreads();
    unsigned long long n0 = ns - nt, v0 = vs - vt, v_all = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        n0 += i < wave ? ws[i][0] : 0;
        v0 += i < wave ? ws[i][1] : 0;
        v_all += ws[i][1];
    }
    if (by_k) {
        // top-k ends in class bk; the last class weighs nothing, so an end there is none
        unsigned long long at = n0, vat = v0;
#pragma unroll
        for (int i = 0; i < SM_PER; i++) {
            const int b = threadIdx.x * SM_PER + i;
            if (b < SM_BINS - 1 && at < (unsigned)p.k && at + n[i] >= (unsigned)p.k) {
                sc.bk = b;
                sc.count_k = (unsigned)at;
                sc.weight_k = vat;
                s_end_k = vat + v[i];
                if (!by_p) {
                    sc.lo = sc.hi = b;
                    sc.weight_lo = vat;
                }
            }
            at += n[i];
            vat += v[i];
        }
        __syncthreads();
    }
    if (by_p) {
        // the weight that top-p is a share of lies between these; so does its end
        const int bk = by_k ? sc.bk : -1;
        const double wl = (double)(bk >= 0 ? sc.weight_k : v_all), wh = (double)(bk >= 0 ? s_end_k : v_all);
        const double tl = (double)p.top_p * wl, th = (double)p.top_p * wh;
        unsigned long long vat = v0;
#pragma unroll
        for (int i = 0; i < SM_PER; i++) {
            const int b = threadIdx.x * SM_PER + i;
            const double x0 = (double)vat, x1 = (double)(vat + v[i]);
            if (x1 >= tl && (x0 < tl || b == 0)) {
                sc.lo = b;
                sc.weight_lo = vat;
            }
            if (x1 >= th && (x0 < th || b == 0)) sc.hi = b;
            vat += v[i];
        }
        __syncthreads();
    }
    SmCut c = sc;
    c.weight_all = v_all;
    return c;
}

// A logit below which no entry is of a class up to the last one that is kept or listed, or,
// where all are kept, as likely as min-p asks; -infinity: none is left out.  d = M - l of class B
// or less has d c scale < B + 1 up to the few roundings of 2^-24 that sm_y makes: a part in 10^5 is
// more than those.
__device__ __forceinline__ float sm_cut_logit(const SmPar &p, const SmCut &c) {
    const int last = max(max(c.lo - 1, c.hi), c.bk);
    double d;
    if (last < SM_BINS - 2) d = (double)(last + 1) / ((double)p.scale * (double)p.c);
    else if (c.lo == SM_BINS && p.lim < INFINITY) d = ((double)p.lim + (double)p.lim_lo) / (double)p.c + 1e-30;
    else return -INFINITY;
    const double at = (double)p.M - d * 1.00001;
    float f = (float)at;
    if ((double)f > at) f = nextafterf(f, -INFINITY);
    return f == f ? f : -INFINITY;
}

__global__ __launch_bounds__(256) void sample_pick(qk_sample_args a, int nb) {
    const int row = blockIdx.x / nb, b = blockIdx.x % nb, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    SmRow &w = ((SmRow *)a.ws)[row];
    const float *x = a.logits + (size_t)row * a.row_stride;
    const int subs = (a.vocab + SM_SUB - 1) / SM_SUB;
    constexpr int PL = SM_SUB / 64;
    float l[PL];
    auto load = [&](int s) {
#pragma unroll
        for (int j = 0; j < PL; j++) {
            const int i = s * SM_SUB + 64 * j + lane;
            l[j] = i < a.vocab ? x[i] : -INFINITY;
        }
    };
    // what does not wait for the thresholds: the first entries, the classes
    int s = b * 4 + wave;
    if (s < subs) load(s);
    unsigned cn[SM_PER];
    unsigned long long cw[SM_PER];
#pragma unroll
    for (int i = 0; i < SM_PER; i++) {
        cn[i] = w.count[threadIdx.x * SM_PER + i];
        cw[i] = w.weight[threadIdx.x * SM_PER + i];
    }
    const SmPar p = w.par;
    if (p.none) return;
    const SmCut c = p.k == 1 ? SmCut{0, 0, 0, 0, 0, 0, 0} : sm_cut(p, cn, cw);       // the largest is in class 0
    if (b == 0 && threadIdx.x == 0) {
        w.lo = c.lo;
        w.hi = c.hi;
        w.bk = c.bk;
        w.count_k = c.count_k;
        w.weight_k = c.weight_k;
        w.weight_lo = c.weight_lo;
        w.weight_all = c.weight_all;
    }
    // the block's list, then one place in the row's for it all
    __shared__ unsigned long long list[SM_CAND];
    __shared__ unsigned n, at;
    if (threadIdx.x == 0) n = 0;
    __syncthreads();
    auto entry = [&](float x, int i, unsigned long long &sum) {
        const SmY v = sm_y(p, x);
        if (v.bin < c.lo) {
            // with a branch: an entry that is not kept costs no weight
            if (p.lim == INFINITY || sm_likely(p, v)) sum += sm_weight(v);
        } else if (v.bin <= c.hi || v.bin == c.bk) {
            const unsigned k = atomicAdd(&n, 1u);
            if (k < SM_CAND) list[k] = (unsigned long long)__float_as_uint(x) << 32 | (unsigned)i;
        }
    };
    // Logits below `cut` are in no class that is kept or listed.  The others of a partial sum are
    // packed in LDS first: few lanes of a wave have one, and all would wait for its weight (64 rows,
    // top-p: 49.7 us for the four launches, 51.8 without).
    const float cut = sm_cut_logit(p, c);
    __shared__ float qx[4][SM_SUB];
    __shared__ unsigned short qi[4][SM_SUB];
    for (; s < subs; s += nb * 4) {
        float now[PL];
#pragma unroll
        for (int j = 0; j < PL; j++) now[j] = l[j];
        if (s + nb * 4 < subs) load(s + nb * 4);
        unsigned long long sum = 0;
        if (cut == -INFINITY) {
#pragma unroll
            for (int j = 0; j < PL; j++) entry(now[j], s * SM_SUB + 64 * j + lane, sum);
        } else {
            int len = 0;
#pragma unroll
            for (int j = 0; j < PL; j++) {
                const bool hit = now[j] >= cut;
                const unsigned long long hits = __ballot(hit);
                if (hit) {
                    const int k = len + __popcll(hits & ((1ull << lane) - 1));
                    qx[wave][k] = now[j];
                    qi[wave][k] = (unsigned short)(64 * j + lane);
                }
                len += __popcll(hits);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            for (int k = lane; k < len; k += 64) entry(qx[wave][k], s * SM_SUB + qi[wave][k], sum);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        sum = sm_wave_sum(sum);
        if (lane == 63) w.sub[s] = sum;
    }
    __syncthreads();
    if (n == 0) return;
    if (threadIdx.x == 0) at = atomicAdd(&w.n_cand, n);
    __syncthreads();
    for (unsigned i = threadIdx.x; i < n && i < SM_CAND; i += 256)
        if (at + i < SM_CAND) w.cand[at + i] = list[i];
}

// The entry at which a running sum over the order reaches `target`, by counting
// 8 bits at a time over the row's entries that are >= least: counts (by_weight
// false) or weights.  Returns its place in the order and the weight up to and
// including it.
__device__ unsigned long long sm_select(const SmPar &p, const float *x, int vocab, unsigned long long least,
                                        bool by_weight, double target, unsigned long long &upto) {
    __shared__ unsigned long long hw[256];
    __shared__ unsigned hc[256];
    __shared__ int pick;
    __shared__ double base_s;
    __shared__ unsigned long long weight_s;
    unsigned long long prefix = 0, before = 0;
    double base = 0.0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) {
            hw[threadIdx.x] = 0;
            hc[threadIdx.x] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < vocab; i += 1024) {
            const float l = sm_clean(x[i]);
            if (l == -INFINITY) continue;
            const unsigned long long cp = sm_comp(l, i);
            if (cp < least || (shift < 56 && (cp >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
            const int d = (int)(cp >> shift) & 255;
            atomicAdd(&hw[d], sm_weight(sm_y(p, l)));
            atomicAdd(&hc[d], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            // the last digit that holds anything, if rounding leaves the target beyond the sum
            double at = base;
            unsigned long long wt = before;
            int last = 0;
            double last_at = at;
            unsigned long long last_wt = wt;
            bool found = false;
            for (int d = 255; d >= 0 && !found; d--) {
                if (!hc[d]) continue;
                last = d;
                last_at = at;
                last_wt = wt;
                at += by_weight ? (double)hw[d] : (double)hc[d];
                wt += hw[d];
                found = at >= target;
            }
            pick = last;
            base_s = last_at;
            weight_s = last_wt;
        }
        __syncthreads();
        prefix |= (unsigned long long)pick << shift;
        base = base_s;
        before = weight_s;
        __syncthreads();
    }
    const int i = (int)(0xffffffffu - (unsigned)prefix);
    upto = before + sm_weight(sm_y(p, sm_clean(x[i])));
    return prefix;
}

__global__ __launch_bounds__(1024) void sample_draw(qk_sample_args a) {
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    SmRow &w = ((SmRow *)a.ws)[row];
    // [0, n) in list order, padded; by rank; sums before each rank
    __shared__ __attribute__((aligned(16))) unsigned long long comp[SM_CAND], before[SM_CAND + 1], sub[SM_MAX_SUBS];
    __shared__ unsigned rank[SM_CAND];
    __shared__ int found;
    __shared__ unsigned long long base;
    const int subs = (a.vocab + SM_SUB - 1) / SM_SUB;
    const int lo = w.lo, hi = w.hi, bk = w.bk;
    const unsigned n = w.n_cand;
    const unsigned long long entry = t < (int)min(n, (unsigned)SM_CAND) ? w.cand[t] : 0;
    const unsigned long long sub_t = t < subs ? w.sub[t] : 0;
    float u = a.u[row];
    const SmPar p = w.par;
    if (p.none) {
        if (t == 0) a.tokens[row] = -1;
        return;
    }
    const float *x = a.logits + (size_t)row * a.row_stride;
    const bool slow = n > SM_CAND;               // block-uniform
    unsigned long long least = 0, all;
    unsigned long long mine = 0;                 // this thread's listed entry's weight, if it is kept
    const int index = (int)(unsigned)entry;
    sub[t] = sub_t;
    if (!slow && n > 0) {
        const float l = sm_clean(__uint_as_float((unsigned)(entry >> 32)));
        const SmY v = sm_y(p, l);
        const unsigned long long weight = sm_weight(v);
        bool keep = t < (int)n;
        // nothing real is 0: the padding is before nothing
        comp[t] = keep ? sm_comp(l, index) : 0;
        rank[t] = 0;
        before[t] = 0;
        __syncthreads();
        // the rank of each: groups of waves compare it with a part of the list each
        const int padded = (int)(n + 63) & ~63, parts = 1024 / padded, part = t / padded, i = t % padded;
        if (part < parts) {
            const unsigned long long me = comp[i];
            const int len = (padded / 2 + parts - 1) / parts * 2, j0 = part * len, j1 = min(j0 + len, padded);
            unsigned r = 0;
#pragma unroll 4
            for (int j = j0; j < j1; j += 2) {
                const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&comp[j]);
                r += (o.x > me) + (o.y > me);
            }
            if (r) atomicAdd(&rank[i], r);
        }
        __syncthreads();
        const unsigned my = rank[t];
        if (keep) before[my] = weight;
        __syncthreads();
        const unsigned long long sorted = before[t];
        const unsigned long long ahead_w = sm_scan<1024>(sorted, all);
        before[t] = ahead_w;
        if (t == 0) before[SM_CAND] = all;
        unsigned long long whole = w.weight_all;
        const unsigned ahead = (unsigned)__syncthreads_count(keep && v.bin < bk);    // listed entries of earlier classes
        if (bk >= 0) {
            const unsigned left = (unsigned)p.k - w.count_k;         // entries that class bk gives to the top k
            if (v.bin == bk) keep = keep && my - ahead < left;
            whole = w.weight_k + (before[min(ahead + left, n)] - before[ahead]);
        }
        if (p.top_p < 1.0f) {
            const unsigned long long sum = w.weight_lo + before[my];
            keep = keep && v.bin <= hi && ((double)sum < (double)p.top_p * (double)whole || sum == 0);
        }
        if (keep && sm_likely(p, v)) {
            mine = weight;
            atomicAdd(&sub[index / SM_SUB], mine);
        }
        __syncthreads();
    } else if (slow) {
        unsigned long long upto = 0;
        if (p.k > 0) least = sm_select(p, x, a.vocab, 0, false, (double)p.k, upto);
        if (p.top_p < 1.0f)
            least = sm_select(p, x, a.vocab, least, true, (double)p.top_p * (p.k > 0 ? (double)upto : (double)w.weight_all), upto);
        for (int s = wave; s < subs; s += 16) {
            unsigned long long sum = 0;
            for (int j = 0; j < SM_SUB / 64; j++) {
                const int i = s * SM_SUB + 64 * j + lane;
                const float l = i < a.vocab ? sm_clean(x[i]) : -INFINITY;
                if (l == -INFINITY || sm_comp(l, i) < least) continue;
                const SmY v = sm_y(p, l);
                if (sm_likely(p, v)) sum += sm_weight(v);
            }
            sum = sm_wave_sum(sum);
            if (lane == 63) sub[s] = sum;
        }
        __syncthreads();
    }
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    // the 1024 entries, then the entry, at which the sum passes u times all of it
    const unsigned long long s0 = sm_scan<1024>(sub[t], all);
    const double target = (double)u * (double)all;
    if ((double)s0 <= target && (double)(s0 + sub[t]) > target) {
        found = t;
        base = s0;
    }
    comp[t] = 0;
    __syncthreads();
    const int s = found;
    if (mine && index / SM_SUB == s) comp[index % SM_SUB] = mine;
    const int i = s * SM_SUB + t;
    const float l = i < a.vocab ? sm_clean(x[i]) : -INFINITY;
    __syncthreads();
    unsigned long long v = comp[t];
    if (l > -INFINITY) {
        const SmY y = sm_y(p, l);
        if ((slow ? sm_comp(l, i) >= least : y.bin < lo) && sm_likely(p, y)) v = sm_weight(y);
    }
    unsigned long long in_sub;
    const unsigned long long v0 = base + sm_scan<1024>(v, in_sub);
    if ((double)v0 <= target && (double)(v0 + v) > target) a.tokens[row] = i;
}

extern "C" size_t qk_sample_ws_bytes(int rows, int vocab) { return (size_t)rows * sizeof(SmRow); }

extern "C" int qk_sample_launch(const qk_sample_args *a, hipStream_t s) {
    // A wave of sample_pick takes a partial sum at a time and 4096 waves are there at
    // once: as many turns as that takes, and blocks of four waves for so many turns.
    const int subs = (a->vocab + SM_SUB - 1) / SM_SUB;
    const long turns = ((long)subs * a->rows + 4095) / 4096;
    int nb = (int)((subs + 4 * turns - 1) / (4 * turns));
    if (nb > SM_MAX_BLOCKS) nb = SM_MAX_BLOCKS;
    const unsigned blocks = (unsigned)(a->rows * nb);
    // 4096 entries a block at least, and about 512 blocks
    int nh = (a->vocab + 4095) / 4096;
    const int most_h = a->rows >= 512 ? 1 : 512 / a->rows;
    if (nh > most_h) nh = most_h;
    sample_max<<<blocks, 256, 0, s>>>(*a, nb);
    sample_hist<<<(unsigned)(a->rows * nh), 1024, 0, s>>>(*a, nb, nh);
    sample_pick<<<blocks, 256, 0, s>>>(*a, nb);
    sample_draw<<<a->rows, 1024, 0, s>>>(*a);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
