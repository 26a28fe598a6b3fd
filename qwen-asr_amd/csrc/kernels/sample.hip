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
// fp32 exponential.  a_i is computed in 64 bits, the exponential's fraction on the
// hardware (v_exp_f32, 1 ulp).
//
// Four launches over blocks of the row, each reading the row once (from the
// caches after the first time):
//   sample_max    largest and smallest finite logit of each block's share
//   sample_hist   count and weight of SM_BINS classes of a, evenly over the row's range
//                 (at most 32: the last class holds what weighs 0)
//   sample_pick   from the classes' running sums: which are kept whole, and which hold
//                 a threshold.  Entries of the latter go to a short list, the former
//                 are summed per 1024 entries
//   sample_draw   one block a row: orders the list by counting, finds both
//                 thresholds, and walks the sums down to the one entry
// A row whose threshold classes hold more than SM_CAND entries (nearly equal
// logits) takes a radix selection over the row in the last launch instead.
// Bound by launch latency for few rows; for many by reading the row and the
// 64-bit arithmetic on each entry.
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

struct SmRow {                    // one row's part of the workspace
    unsigned long long weight[SM_BINS];
    unsigned count[SM_BINS];
    float max[SM_MAX_BLOCKS], min[SM_MAX_BLOCKS];
    unsigned n_cand, slow, pad[2];
    int lo, hi, bk, pad1;         // classes below lo are kept whole; lo .. hi and bk hold the thresholds
    unsigned count_k;             // entries before class bk
    unsigned pad2;
    unsigned long long weight_k, weight_lo, weight_all;   // before bk, before lo, of the row
    unsigned cand[SM_CAND];
    unsigned long long sub[SM_MAX_SUBS];
};

struct SmPar {
    double M, inv_t, scale, lim;  // largest logit; 1 / T; classes per unit of a; largest a that min-p keeps
    float top_p;                  // >= 1: off
    int k;                        // 0: off
    bool none;                    // no entry at all
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

__device__ __forceinline__ double sm_a(const SmPar &p, float l) {
    if ((double)l == p.M) return 0.0;
    const double a = (p.M - (double)l) * p.inv_t;
    return a < 1e30 ? a : 1e30;                  // also where it is none (0 times infinity)
}

__device__ __forceinline__ int sm_bin(const SmPar &p, double a) {
    const double b = a * p.scale;
    return b < (double)(SM_BINS - 1) ? (int)b : SM_BINS - 1;
}

__device__ __forceinline__ unsigned long long sm_weight(double a) {
    if (!(a < 32.0)) return 0;
    const double y = a * 1.4426950408889634074;
    const int n = (int)(y + 0.5);
    const float e = __builtin_amdgcn_exp2f((float)((double)n - y));      // 2^(-1/2) .. 2^(1/2)
    return ((unsigned long long)(unsigned)(e * 16777216.0f) << 19) >> n;
}

__device__ __forceinline__ SmPar sm_par(const qk_sample_args &a, const SmRow &w, int row, int nb) {
    __shared__ float smx, smn;
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
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(T > 0.0f);
    p.inv_t = greedy ? 1.0 : 1.0 / (double)T;
    int k = a.top_k ? a.top_k[row] : 0;
    if (greedy) k = 1;
    p.k = k <= 0 || k >= a.vocab ? 0 : k;
    const float tp = a.top_p ? a.top_p[row] : 1.0f;
    p.top_p = tp != tp ? 1.0f : fmaxf(tp, 0.0f);
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    p.lim = mp > 0.0f ? -log((double)fminf(mp, 1.0f)) : 1e300;
    double range = (p.M - (double)smn) * p.inv_t;
    range = range < 32.0 ? range * (1.0 + 1e-9) : 32.0;       // also where it is none
    p.scale = (double)(SM_BINS - 1) / fmax(range, 1e-300);
    if (!(p.scale < 1e300)) p.scale = 1e300;
    __syncthreads();                             // the shared pair may be written again
    return p;
}

// exclusive sum over the block of one value per thread, and the sum of all
template <int NT, typename V>
__device__ __forceinline__ V sm_scan(V v, V &total) {
    constexpr int NW = NT / 64;
    __shared__ V ws[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    V x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const V y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) ws[wave] = x;
    __syncthreads();
    V base = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        if (i < wave) base += ws[i];
        all += ws[i];
    }
    total = all;
    return base + x - v;
}

__device__ __forceinline__ unsigned long long sm_wave_sum(unsigned long long v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
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
    if (b == 0 && threadIdx.x == 0) w.n_cand = w.slow = 0;
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

__global__ __launch_bounds__(256) void sample_hist(qk_sample_args a, int nb) {
    const int row = blockIdx.x / nb, b = blockIdx.x % nb;
    SmRow &w = ((SmRow *)a.ws)[row];
    const SmPar p = sm_par(a, w, row, nb);
    if (p.none || (p.k == 0 && p.top_p >= 1.0f)) return;     // nothing asks for the order
    __shared__ unsigned long long hw[SM_BINS];
    __shared__ unsigned hc[SM_BINS];
    for (int i = threadIdx.x; i < SM_BINS; i += 256) {
        hw[i] = 0;
        hc[i] = 0;
    }
    __syncthreads();
    const float *x = a.logits + (size_t)row * a.row_stride;
#pragma unroll 4
    for (int i = b * 256 + threadIdx.x; i < a.vocab; i += nb * 256) {
        const float l = sm_clean(x[i]);
        if (l == -INFINITY) continue;
        const double d = sm_a(p, l);
        const int c = sm_bin(p, d);
        atomicAdd(&hw[c], sm_weight(d));
        atomicAdd(&hc[c], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SM_BINS; i += 256)
        if (hc[i]) {
            atomicAdd(&w.weight[i], hw[i]);
            atomicAdd(&w.count[i], hc[i]);
        }
}

struct SmCut {
    int lo, hi, bk;
    unsigned count_k;
    unsigned long long weight_k, weight_lo, weight_all;
};

// which classes hold the thresholds (256 threads)
__device__ SmCut sm_cut(const SmPar &p, const SmRow &w) {
    constexpr int PER = SM_BINS / 256;
    SmCut c = {SM_BINS, -1, -1, 0, 0, 0, 0};
    if (p.k == 0 && p.top_p >= 1.0f) return c;
    __shared__ SmCut sc;
    __shared__ int s_lo, s_hi;
    __shared__ unsigned long long s_end_k;
    unsigned n[PER], nt = 0, n_all;
    unsigned long long v[PER], vt = 0, v_all;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        n[i] = w.count[threadIdx.x * PER + i];
        v[i] = w.weight[threadIdx.x * PER + i];
        nt += n[i];
        vt += v[i];
    }
    const unsigned n0 = sm_scan<256>(nt, n_all);
    const unsigned long long v0 = sm_scan<256>(vt, v_all);
    if (threadIdx.x == 0) {
        sc = c;
        sc.weight_all = v_all;
        s_lo = s_hi = SM_BINS - 1;
    }
    __syncthreads();
    // top-k ends in class bk; the last class weighs nothing, so an end there is none
    if (p.k > 0) {
        unsigned at = n0;
        unsigned long long vat = v0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int b = threadIdx.x * PER + i;
            if (b < SM_BINS - 1 && at < (unsigned)p.k && at + n[i] >= (unsigned)p.k) {
                sc.bk = b;
                sc.count_k = at;
                sc.weight_k = vat;
                s_end_k = vat + v[i];
            }
            at += n[i];
            vat += v[i];
        }
    }
    __syncthreads();
    const int bk = sc.bk;
    if (p.top_p < 1.0f) {
        // the weight that top-p is a share of lies between these; so does its end
        const double wl = bk >= 0 ? (double)sc.weight_k : (double)v_all, wh = bk >= 0 ? (double)s_end_k : (double)v_all;
        const double tl = (double)p.top_p * wl, th = (double)p.top_p * wh;
        unsigned long long vat = v0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int b = threadIdx.x * PER + i;
            const double x0 = (double)vat, x1 = (double)(vat + v[i]);
            if (x1 >= tl && (x0 < tl || b == 0)) s_lo = b;
            if (x1 >= th && (x0 < th || b == 0)) s_hi = b;
            vat += v[i];
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            sc.lo = s_lo;
            sc.hi = s_hi;
        }
    } else if (threadIdx.x == 0) {
        sc.lo = bk >= 0 ? bk : SM_BINS;
        sc.hi = bk;
    }
    __syncthreads();
    const int lo = sc.lo;
    unsigned long long vat = v0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (threadIdx.x * PER + i == lo) sc.weight_lo = vat;
        vat += v[i];
    }
    __syncthreads();
    return sc;
}

__global__ __launch_bounds__(256) void sample_pick(qk_sample_args a, int nb) {
    const int row = blockIdx.x / nb, b = blockIdx.x % nb, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    SmRow &w = ((SmRow *)a.ws)[row];
    const SmPar p = sm_par(a, w, row, nb);
    if (p.none) return;
    const SmCut c = sm_cut(p, w);
    if (b == 0 && threadIdx.x == 0) {
        w.lo = c.lo;
        w.hi = c.hi;
        w.bk = c.bk;
        w.count_k = c.count_k;
        w.weight_k = c.weight_k;
        w.weight_lo = c.weight_lo;
        w.weight_all = c.weight_all;
    }
    const float *x = a.logits + (size_t)row * a.row_stride;
    const int subs = (a.vocab + SM_SUB - 1) / SM_SUB;
    for (int s = b * 4 + wave; s < subs; s += nb * 4) {
        unsigned long long sum = 0;
#pragma unroll 4
        for (int j = 0; j < SM_SUB / 64; j++) {
            const int i = s * SM_SUB + 64 * j + lane;
            const float l = i < a.vocab ? sm_clean(x[i]) : -INFINITY;
            if (l == -INFINITY) continue;
            const double d = sm_a(p, l);
            const int cl = sm_bin(p, d);
            if (cl < c.lo) {
                if (d <= p.lim) sum += sm_weight(d);
            } else if (cl <= c.hi || cl == c.bk) {
                const unsigned at = atomicAdd(&w.n_cand, 1u);
                if (at < SM_CAND) w.cand[at] = (unsigned)i;
            }
        }
        sum = sm_wave_sum(sum);
        if (lane == 0) w.sub[s] = sum;
    }
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
            atomicAdd(&hw[d], sm_weight(sm_a(p, l)));
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
    upto = before + sm_weight(sm_a(p, sm_clean(x[i])));
    return prefix;
}

__global__ __launch_bounds__(1024) void sample_draw(qk_sample_args a, int nb) {
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    SmRow &w = ((SmRow *)a.ws)[row];
    const SmPar p = sm_par(a, w, row, nb);
    if (p.none) {
        if (t == 0) a.tokens[row] = -1;
        return;
    }
    const float *x = a.logits + (size_t)row * a.row_stride;
    __shared__ unsigned long long comp[SM_CAND], wt[SM_CAND], sub[SM_MAX_SUBS];
    __shared__ int found;
    const int subs = (a.vocab + SM_SUB - 1) / SM_SUB;
    const int lo = w.lo, hi = w.hi, bk = w.bk;
    const unsigned n = w.n_cand;
    const bool slow = n > SM_CAND;               // block-uniform
    unsigned long long least = 0, all;
    unsigned long long mine = 0;                 // this thread's listed entry's weight, if it is kept
    int index = -1;
    if (!slow) {
        sub[t] = t < subs ? w.sub[t] : 0;
        float l = 0.0f;
        double d = 0.0;
        int cl = SM_BINS;
        if (t < (int)n) {
            index = (int)w.cand[t];
            l = sm_clean(x[index]);
            d = sm_a(p, l);
            cl = sm_bin(p, d);
            comp[t] = sm_comp(l, index);
            wt[t] = sm_weight(d);
        }
        __syncthreads();
        unsigned before_n = 0;
        unsigned long long before_w = 0;
        if (t < (int)n) {
            const unsigned long long me = comp[t];
            for (unsigned j = 0; j < n; j++)
                if (comp[j] > me) {
                    before_n++;
                    before_w += wt[j];
                }
        }
        bool keep = t < (int)n;
        unsigned long long whole = w.weight_all;
        if (bk >= 0) {
            unsigned ahead;
            (void)sm_scan<1024>((unsigned)(keep && cl < bk), ahead);     // listed entries of earlier classes
            if (cl == bk) keep = keep && w.count_k + (before_n - ahead) < (unsigned)p.k;
            unsigned long long in_k;
            (void)sm_scan<1024>(keep && cl == bk ? wt[t] : 0ull, in_k);
            whole = w.weight_k + in_k;
        }
        if (p.top_p < 1.0f) {
            const unsigned long long before = w.weight_lo + before_w;
            keep = keep && cl <= hi && ((double)before < (double)p.top_p * (double)whole || before == 0);
        }
        if (keep && d <= p.lim) {
            mine = wt[t];
            atomicAdd(&sub[index / SM_SUB], mine);
        }
        __syncthreads();
    } else {
        unsigned long long upto = 0;
        if (p.k > 0) least = sm_select(p, x, a.vocab, 0, false, (double)p.k, upto);
        if (p.top_p < 1.0f)
            least = sm_select(p, x, a.vocab, least, true, (double)p.top_p * (p.k > 0 ? (double)upto : (double)w.weight_all), upto);
        for (int s = wave; s < SM_MAX_SUBS; s += 16) {
            unsigned long long sum = 0;
            if (s < subs)
                for (int j = 0; j < SM_SUB / 64; j++) {
                    const int i = s * SM_SUB + 64 * j + lane;
                    const float l = i < a.vocab ? sm_clean(x[i]) : -INFINITY;
                    if (l == -INFINITY || sm_comp(l, i) < least) continue;
                    const double d = sm_a(p, l);
                    if (d <= p.lim) sum += sm_weight(d);
                }
            sum = sm_wave_sum(sum);
            if (lane == 0) sub[s] = sum;
        }
        __syncthreads();
    }
    float u = a.u[row];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    // the 1024 entries, then the entry, at which the sum passes u times all of it
    const unsigned long long s0 = sm_scan<1024>(sub[t], all);
    const double target = (double)u * (double)all;
    if ((double)s0 <= target && (double)(s0 + sub[t]) > target) found = t;
    __syncthreads();
    const int s = found;
    __shared__ unsigned long long base;
    if (t == s) base = s0;
    __syncthreads();
    comp[t] = 0;
    __syncthreads();
    if (mine && index / SM_SUB == s) comp[index % SM_SUB] = mine;
    __syncthreads();
    unsigned long long v = comp[t];
    const int i = s * SM_SUB + t;
    if (i < a.vocab) {
        const float l = sm_clean(x[i]);
        if (l > -INFINITY) {
            const double d = sm_a(p, l);
            if (d <= p.lim && (slow ? sm_comp(l, i) >= least : sm_bin(p, d) < lo)) v = sm_weight(d);
        }
    }
    unsigned long long in_sub;
    const unsigned long long v0 = base + sm_scan<1024>(v, in_sub);
    if ((double)v0 <= target && (double)(v0 + v) > target) a.tokens[row] = i;
}

extern "C" size_t qk_sample_ws_bytes(int rows, int vocab) { return (size_t)rows * sizeof(SmRow); }

extern "C" int qk_sample_launch(const qk_sample_args *a, hipStream_t s) {
    // four partial sums a block at least, and about 1024 blocks
    const int subs = (a->vocab + SM_SUB - 1) / SM_SUB;
    int nb = (subs + 3) / 4;
    const int most = a->rows >= 1024 ? 1 : 1024 / a->rows;
    if (nb > most) nb = most;
    if (nb > SM_MAX_BLOCKS) nb = SM_MAX_BLOCKS;
    if ((long)a->rows * nb > 0x7fffffffL) return QWEN_HIP_EINVAL;
    const unsigned blocks = (unsigned)(a->rows * nb);
    sample_max<<<blocks, 256, 0, s>>>(*a, nb);
    sample_hist<<<blocks, 256, 0, s>>>(*a, nb);
    sample_pick<<<blocks, 256, 0, s>>>(*a, nb);
    sample_draw<<<a->rows, 1024, 0, s>>>(*a, nb);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
