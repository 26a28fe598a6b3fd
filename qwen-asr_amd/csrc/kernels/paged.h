// paged.h - device helpers shared by the kernels that work on a paged KV cache
// (paged_append.hip, paged_decode.hip, paged_prefill.hip).
//
// Pages are [n_pages][kv_heads][page_size][128] of fp32 or bf16, page_size a
// power of two.  Lengths, row starts and page ids are device data that no host
// check has seen: every use here is clamped, so that wrong values give wrong
// rows but never an access outside the buffers.
#pragma once
#include "common.h"
#include "qk_kernels.h"
#include "qwen_asr_hip.h"

#include <math.h>

#define PG_HD QWEN_HIP_HEAD_DIM

// Element offset of (page id, kv head, slot).  64 bits: a cache of a few
// hundred thousand positions passes 2^32 elements.
__device__ __forceinline__ size_t pg_offset(const qk_paged &a, int pid, int kvh, int pos) {
    const int slot = pos & ((1 << a.page_shift) - 1);
    return ((((size_t)pid * a.kv_heads + kvh) << a.page_shift) + slot) * PG_HD;
}

// Page id of position pos (0 <= pos < a.capacity) of sequence s, -1 where the
// table holds none
__device__ __forceinline__ int pg_page(const qk_paged &a, int s, int pos) {
    const int pid = a.table[(size_t)s * a.table_stride + (pos >> a.page_shift)];
    return (unsigned)pid < (unsigned)a.n_pages ? pid : -1;
}

// cached positions of sequence s, 0 for a negative length
__device__ __forceinline__ int pg_len(const qk_paged &a, int s) { return max(a.kv_len[s], 0); }

// Last s in [0, n) with key(s) <= x, -1 if there is none (key not falling): a
// G-ary search by an aligned group of G lanes, every lane the same x.  One
// dependent load for n <= G (64 sequences by a wave), where a binary search by
// one lane has log2(n).  All 64 lanes of the wave call it together.
template <int G, typename KEY>
__device__ __forceinline__ int pg_search(int n, long x, KEY key) {
    const int lane = threadIdx.x & 63, c = lane % G, base = lane - c;
    const unsigned long long gm = G == 64 ? ~0ull : (1ull << G) - 1;
    int lo = 0;
    bool none = false;
    for (int len = n, step; len > 0; len = step > 1 ? step : 0) {
        step = (len + G - 1) / G;
        const long at = (long)lo + (long)c * step;
        const bool le = at < n && (long)c * step < len && key((int)at) <= x;
        const int cnt = __popcll((__ballot(le) >> base) & gm);
        if (lo == 0 && cnt == 0 && len == n) none = true;
        lo += max(cnt - 1, 0) * step;
    }
    return none || n <= 0 ? -1 : min(lo, n - 1);
}

// two / four consecutive values of a row as floats
__device__ __forceinline__ float4 pg_load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 pg_load4(const uint16_t *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
}

// ... and back, rounded once to nearest even where the type is bf16
__device__ __forceinline__ void pg_store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void pg_store4(uint16_t *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(bf16_pack2(v.x, v.y), bf16_pack2(v.z, v.w));
}

// The running maximum to subtract: 0 while nothing was seen (2^(-inf - 0) = 0, where
// -inf - -inf is no number)
__device__ __forceinline__ float pg_ref(float m) { return m == -INFINITY ? 0.0f : m; }

#define PG_LOG2E 1.44269504088896341f
