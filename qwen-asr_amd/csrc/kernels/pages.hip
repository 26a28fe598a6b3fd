// pages.hip - the pages of a paged KV cache as a program's sequences change: page tables of
// sequences that continue others, pages for their next rows, copies of pages that two of
// them would write (in all layers), and accepted drafts that move up behind the past.
//
// Whole numbers and copies of bits: the results are exact.
//
// Measured (a device copy moves 4.8 to 5.1 TB/s): 64 beams of 131 to 701 positions, 28 layers, bf16, pages of 32: table
// 8 us (a chain of loads and barriers in one block), copies of 31 half pages, 112 MB read and written, 25 to 33 us; 4 beams
// of 530, fp32: 5 and 3 us, less than the two calls take.  A wave takes four rows of the table, 64 entries of each at
// a time, so wide tables of few rows are one wave's work: one row of 24 entries 5 us, of 1251 11, of 6251 39, of 62501
// 350; 64 rows of 1251 22, of 6251 71; and 1024 rows of 24, each compared with all others, 132.  Accepted drafts of 1
// and of 24 sequences, 28 layers: 9 us, a launch.
#include "paged.h"

#include <limits.h>

typedef uint32_t pages_u32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// paged_fork: row s of the new table continues row p = parent[s] of the old one.
//
//   keep     entries 0 .. ceil(len / P) - 1 of row p, len = kv_len[p], P positions a page
//   held     a page is held where an entry of the new table or the program (`outside`) names it
//   tail     the last kept page, where len % P > 0: new rows go to its free slots.  If the row has new
//            rows and another one holds the page as well, the row takes a copy; of the rows that have it
//            as their tail the one with the most slots of it keeps it (of several the last: what it
//            writes no other one has), unless a row holds it for positions past it
//   fresh    entries up to ceil((len + new) / P) and tails that are copied or no page: the pages that are
//            not held, lowest first, by row and entry
//
// Nothing is counted from call to call: what is held follows from the new table, so
// a page that no row names is free again.
//
// One block: the work is a few thousand table entries (64 rows of 24 pages) between barriers, and what is
// held is a bit a page, in LDS up to FK_LDS_PAGES pages, in the workspace beyond.  Rows are taken four at a time a wave, fresh
// pages a thread each (a thread a word of bits, its free ones in turn: 19 us for 64 beams instead of 8).
// ---------------------------------------------------------------------------
#define FK_THREADS 1024
#define FK_WAVES (FK_THREADS / 64)
#define FK_ROWS 4                                     // rows that a wave has on their way at once

// exclusive sum over the block's threads and the sum of all; part: FK_WAVES + 1 ints
__device__ __forceinline__ int fk_scan(int v, int *part, int &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int up = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(up, d, 64);
        if (lane >= d) up += o;
    }
    __syncthreads();                                  // part is free again
    if (lane == 63) part[wave] = up;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < FK_WAVES; i++) {
        const int p = part[i];
        before += i < wave ? p : 0;
        sum += p;
    }
    all = sum;
    return before + up - v;
}

struct FkRow {
    int first, count;                                 // entries that get fresh pages: first .. first + count - 1
    int tail;                                         // page that is copied to the first of them, -1: none
};

template <int LDS_WORDS>
__global__ __launch_bounds__(FK_THREADS) void paged_fork(qk_paged_fork_args a) {
    __shared__ unsigned bits[LDS_WORDS > 0 ? 2 * LDS_WORDS : 1];
    __shared__ __attribute__((aligned(16))) int tails[QK_PAGED_FORK_ROWS], parts[QK_PAGED_FORK_ROWS];
    __shared__ int offs[QK_PAGED_FORK_ROWS], ranks[FK_THREADS], part[FK_WAVES];
    __shared__ FkRow rows[QK_PAGED_FORK_ROWS];
    __shared__ unsigned long long over;               // pages that the table has no room for
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int words = (a.n_pages + 31) >> 5;
    unsigned *const held = LDS_WORDS > 0 ? bits : a.ws, *const whole = held + words;
    // in the workspace the bits are set and read past the first cache, which atomics do not go through
    auto get = [&](const unsigned *w) {
        if constexpr (LDS_WORDS > 0) return *w;
        else return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    auto set = [&](unsigned *w, int id) { atomicOr(w + (id >> 5), 1u << (id & 31)); };
    for (int i = tid; i < 2 * words; i += FK_THREADS) {
        if constexpr (LDS_WORDS > 0) held[i] = 0u;
        else __hip_atomic_store(held + i, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if constexpr (LDS_WORDS == 0) __threadfence();

    if (tid == 0) over = 0;

    // a thread a row: how much of it is kept
    const int P = 1 << a.page_shift;
    const bool on = tid < a.n_out;
    int p = -1, len = 0, fresh_rows = 0;
    if (on) {
        p = a.parent ? a.parent[tid] : tid;
        p = (unsigned)p < (unsigned)a.n_in ? p : -1;
        len = p >= 0 ? max(a.kv_len[p], 0) : 0;
        fresh_rows = a.new_rows ? max(a.new_rows[tid], 0) : 0;
    }
    const int kept = (int)min(((long)len + P - 1) >> a.page_shift, (long)a.stride);
    const int whole_pages = min(len >> a.page_shift, a.stride), slots = len & (P - 1);
    if (on) {
        tails[tid] = p;
        offs[tid] = -1;                               // the tail, once its wave has read it
        rows[tid] = {whole_pages, kept, -1};
        const long end = (long)len + fresh_rows;
        a.len_out[tid] = (int)min(end, (long)INT_MAX);
        *reinterpret_cast<int4 *>(a.copies + 4 * tid) = make_int4(-1, -1, 0, 0);
    }
    __syncthreads();
    // a wave FK_ROWS rows beside each other: their entries, and which pages they hold.  What the row before has said already
    // (beams share their first pages) is not said again: bits of one word are set one after the other.
    for (int s0 = wave * FK_ROWS; s0 < a.n_out; s0 += FK_WAVES * FK_ROWS) {
        for (int e = lane; e < a.stride; e += 64) {
            int id[FK_ROWS];
            bool in_whole[FK_ROWS];
#pragma unroll
            for (int j = 0; j < FK_ROWS; j++) {
                const int s = min(s0 + j, a.n_out - 1), from = tails[s];
                in_whole[j] = e < rows[s].first;
                id[j] = e < rows[s].count ? a.table[(size_t)max(from, 0) * a.stride + e] : -1;
            }
#pragma unroll
            for (int j = 0; j < FK_ROWS; j++) {
                if (s0 + j >= a.n_out) break;
                id[j] = (unsigned)id[j] < (unsigned)a.n_pages ? id[j] : -1;
                a.table_out[(size_t)(s0 + j) * a.stride + e] = id[j];
                if (id[j] < 0) continue;
                if (!in_whole[j]) offs[s0 + j] = id[j];          // the entry behind the whole pages
                if (j > 0 && id[j] == id[j - 1] && in_whole[j] == in_whole[j - 1]) continue;
                set(held, id[j]);
                if (in_whole[j]) set(whole, id[j]);
            }
        }
    }
    if (a.outside) {
        for (int i = tid; i < a.n_pages; i += FK_THREADS)
            if (a.outside[i]) {
                set(held, i);
                set(whole, i);
            }
    }
    if constexpr (LDS_WORDS == 0) __threadfence();
    __syncthreads();
    const int at = whole_pages;                       // the tail's entry, where it is in the table
    const bool has_tail = on && slots > 0 && at < a.stride;
    const int tail = has_tail ? offs[tid] : -1;
    tails[tid] = tail;                                // -1 behind the last row
    parts[tid] = slots;
    __syncthreads();
    // whether another row has more of the tail: `width` threads a part of the rows each
    ranks[tid] = 0;
    __syncthreads();
    int width = 64;
    while (width < a.n_out) width *= 2;
    const int mine = tid & (width - 1), my_tail = tails[mine], my_part = parts[mine];
    if (my_tail >= 0) {
        bool found = false;
        for (int j = 4 * (tid / width); j < a.n_out; j += 4 * (FK_THREADS / width)) {
            const int4 t = *reinterpret_cast<const int4 *>(tails + j), p = *reinterpret_cast<const int4 *>(parts + j);
            auto more = [&](int tail_j, int part_j, int i) {
                return tail_j == my_tail && (part_j > my_part || (part_j == my_part && i > mine));
            };
            found = found || more(t.x, p.x, j) || more(t.y, p.y, j + 1) || more(t.z, p.z, j + 2) || more(t.w, p.w, j + 3);
        }
        if (found) ranks[mine] = 1;
    }
    __syncthreads();
    const bool copied = tail >= 0 && fresh_rows > 0 && (ranks[tid] || (get(whole + (tail >> 5)) >> (tail & 31) & 1u));
    FkRow r = {kept, 0, -1};
    if (on) {
        const long need = ((long)len + fresh_rows + P - 1) >> a.page_shift;
        if (has_tail && fresh_rows > 0 && (copied || tail < 0)) r.first = at;
        r.count = fresh_rows > 0 ? max((int)min(need, (long)a.stride) - r.first, 0) : 0;
        const long room = max((long)a.stride, ((long)len + P - 1) >> a.page_shift);
        if (fresh_rows > 0 && need > room) atomicAdd(&over, (unsigned long long)(need - room));
        if (copied) {
            r.tail = tail;
            a.table_out[(size_t)tid * a.stride + at] = -1;
        }
        rows[tid] = r;
    }
    int total;
    const int off = fk_scan(r.count, part, total);
    if (on) offs[tid] = off;
    // free pages of this thread's words, in order
    const int per = (words + FK_THREADS - 1) / FK_THREADS, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    auto free_bits = [&](int w) {
        const unsigned f = ~get(held + w);
        return w == words - 1 && (a.n_pages & 31) ? f & ((1u << (a.n_pages & 31)) - 1) : f;
    };
    int free_pages = 0, all;
    for (int w = w0; w < w1; w++) free_pages += __popc(free_bits(w));
    ranks[tid] = fk_scan(free_pages, part, all);
    if (tid == 0) *a.missing = (int)min((long)over + max(total - all, 0), (long)INT_MAX);
    __syncthreads();
    // the last of n ascending numbers that is at most x (the first is 0)
    auto last_upto = [](const int *v, int n, int x) {
        int lo = 0;
        for (int step = 1 << (31 - __builtin_clz(n)); step > 0; step >>= 1)
            if (lo + step < n && v[lo + step] <= x) lo += step;
        return lo;
    };
    // a thread a fresh page: the row that takes it, and which it is
    for (int rank = tid; rank < min(total, all); rank += FK_THREADS) {
        const int s = last_upto(offs, a.n_out, rank), t = last_upto(ranks, min(words, FK_THREADS), rank);
        int k = rank - ranks[t], w = t * per;
        unsigned f = free_bits(w);
        while (k >= __popc(f)) {
            k -= __popc(f);
            f = free_bits(++w);
        }
        int bit = 0;                                  // the k-th of its bits
#pragma unroll
        for (int half = 16; half > 0; half >>= 1) {
            const int c = __popc(f & ((1u << half) - 1));
            if (k >= c) {
                k -= c;
                f >>= half;
                bit += half;
            }
        }
        const FkRow x = rows[s];
        a.table_out[(size_t)s * a.stride + x.first + (rank - offs[s])] = 32 * w + bit;
        if (x.tail >= 0 && rank == offs[s])
            *reinterpret_cast<int4 *>(a.copies + 4 * s) = make_int4(x.tail, 32 * w + bit, 0, parts[s]);
    }
}

#define FK_SMALL (1 << 16)                            // pages: 16 KB of bits
#define FK_LDS_PAGES (1 << 19)

extern "C" size_t qk_paged_fork_ws_bytes(int n_pages) {
    return n_pages > FK_LDS_PAGES ? 2 * sizeof(unsigned) * (((size_t)n_pages + 31) / 32) : 0;
}

extern "C" int qk_paged_fork_launch(const qk_paged_fork_args *a, hipStream_t s) {
    if (a->n_pages <= FK_SMALL) paged_fork<FK_SMALL / 32><<<1, FK_THREADS, 0, s>>>(*a);
    else if (a->n_pages <= FK_LDS_PAGES) paged_fork<FK_LDS_PAGES / 32><<<1, FK_THREADS, 0, s>>>(*a);
    else paged_fork<0><<<1, FK_THREADS, 0, s>>>(*a);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}

// ---------------------------------------------------------------------------
// paged_copy: slots first .. first + slots - 1 of a page to the same slots of another, keys and values
// of all kv heads and layers.  Block (copy, layer and K or V, share of the page's 16-byte pieces).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void paged_copy(qk_paged_layers L, const int *copies) {
    const int4 c = *reinterpret_cast<const int4 *>(copies + 4 * (size_t)blockIdx.x);
    if ((unsigned)c.x >= (unsigned)L.n_pages || (unsigned)c.y >= (unsigned)L.n_pages || c.x == c.y) return;
    if (c.z < 0 || c.w <= 0 || c.z > (1 << L.page_shift) - c.w) return;
    unsigned char *const base = (unsigned char *)(blockIdx.y & 1 ? L.v[blockIdx.y >> 1] : L.k[blockIdx.y >> 1]);
    const int row = L.row_bytes / 16;                 // pieces of a row
    const size_t head = (size_t)L.row_bytes << L.page_shift, page = head * L.kv_heads;
    const unsigned char *const from = base + c.x * page + (size_t)c.z * L.row_bytes;
    unsigned char *const to = base + c.y * page + (size_t)c.z * L.row_bytes;
    const long piece = (long)c.w * row, n = piece * L.kv_heads;      // of a kv head, in all
    const long step = 256L * gridDim.z;
    for (long i0 = 256L * blockIdx.z + threadIdx.x; i0 < n; i0 += 4 * step) {
        pages_u32x4 v[4];
        size_t at[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long i = min(i0 + j * step, n - 1), h = n >> 31 ? i / piece : (long)((unsigned)i / (unsigned)piece);
            at[j] = h * head + 16 * (size_t)(i - h * piece);
            v[j] = *reinterpret_cast<const pages_u32x4 *>(from + at[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i0 + j * step < n) *reinterpret_cast<pages_u32x4 *>(to + at[j]) = v[j];
    }
}

extern "C" int qk_paged_copy_launch(const qk_paged_layers *L, const int *copies, int n, hipStream_t s) {
    if (n > 0xffffff) return QWEN_HIP_EINVAL;         // a launch has fewer than 2^32 threads along an axis
    // about 4096 blocks, none of less than 1024 pieces of a whole page
    const long pieces = ((long)L->row_bytes / 16 * L->kv_heads) << L->page_shift, pairs = 2L * L->n_layers * n;
    long z = (4096 + pairs - 1) / pairs, most = (pieces + 1023) / 1024;
    z = z < most ? z : most;
    paged_copy<<<dim3((unsigned)n, 2 * L->n_layers, (unsigned)z), 256, 0, s>>>(*L, copies);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}

// ---------------------------------------------------------------------------
// paged_compact: of a sequence's n drafts (positions past .. past + n - 1) those of `path`, ascending, move to
// past, past + 1, ..  A thread owns 16 bytes of a row for all of them, in order and CP_ROWS at a time, loads
// before stores: draft path[i] >= i has not been written over when it is read.
// ---------------------------------------------------------------------------
#define CP_ROWS 8
#define CP_PART 256                                   // accepted drafts at a time

__global__ __launch_bounds__(256) void paged_compact(qk_paged_layers L, qk_paged pg, int *len_out, const int *path,
                                                     long path_stride, const int *n_path) {
    __shared__ int from[CP_PART], to[CP_PART], bad;
    const int s = blockIdx.x, tid = threadIdx.x;
    int n = 1;
    if (pg.row_start) {
        const int a = min(max(pg.row_start[s], 0), pg.rows), b = min(max(pg.row_start[s + 1], 0), pg.rows);
        n = max(b - a, 0);
    }
    const long past = (long)pg_len(pg, s) - n;
    const int want = (int)min((long)max(n_path[s], 0), min((long)n, path_stride));
    path += s * path_stride;
    unsigned char *const base = (unsigned char *)(blockIdx.y & 1 ? L.v[blockIdx.y >> 1] : L.k[blockIdx.y >> 1]);
    const int row = L.row_bytes / 16, col = (int)(256 * blockIdx.z + tid), h = col / row;
    const bool on = h < L.kv_heads;
    unsigned char *const mine = base + (((size_t)min(h, L.kv_heads - 1) << L.page_shift) * L.row_bytes) + 16 * (col % row);
    // a row of the cache (of kv head 0) by its position, -1: none.  The host has seen that rows fit an int.
    auto place = [&](long p) {
        if (p < 0 || p >= pg.capacity) return -1;
        const int id = pg_page(pg, s, (int)p);
        return id < 0 ? -1 : id * (L.kv_heads << L.page_shift) + (int)(p & ((1 << L.page_shift) - 1));
    };
    int count = 0;                                    // accepted so far
    for (int i0 = 0; i0 < want; i0 += CP_PART) {
        const int m = min(want - i0, CP_PART);
        __syncthreads();                              // the last part is read
        if (tid == 0) bad = m;
        __syncthreads();
        if (tid < m) {
            const int i = i0 + tid, d = path[i], before = i > 0 ? path[i - 1] : -1;
            // the list ends at an entry that is no draft, or none behind the one before
            if (d <= before || d >= n) atomicMin(&bad, tid);
            const bool stays = d == i || d < 0 || d >= n;
            from[tid] = stays ? -1 : place(past + d);
            to[tid] = stays ? -1 : place(past + i);
        }
        __syncthreads();
        const int good = bad;
        for (int j0 = 0; j0 < good; j0 += CP_ROWS) {
            pages_u32x4 v[CP_ROWS];
            int t[CP_ROWS];                           // the same for the block
#pragma unroll
            for (int j = 0; j < CP_ROWS; j++) {
                const int k = min(j0 + j, CP_PART - 1), f = __builtin_amdgcn_readfirstlane(from[k]);
                t[j] = f >= 0 && j0 + j < good ? __builtin_amdgcn_readfirstlane(to[k]) : -1;
                // what does not move is read at the pages' start, where it does no harm
                v[j] = *reinterpret_cast<const pages_u32x4 *>(mine + (size_t)max(t[j] < 0 ? -1 : f, 0) * L.row_bytes);
            }
#pragma unroll
            for (int j = 0; j < CP_ROWS; j++)
                if (on && t[j] >= 0) *reinterpret_cast<pages_u32x4 *>(mine + (size_t)t[j] * L.row_bytes) = v[j];
        }
        count += good;
        if (good < m) break;
    }
    if (blockIdx.y == 0 && blockIdx.z == 0 && tid == 0) len_out[s] = (int)max(past + count, 0L);
}

extern "C" int qk_paged_compact_launch(const qk_paged_layers *L, const qk_paged *pg, int *len_out, const int *path,
                                       long path_stride, const int *n_path, hipStream_t s) {
    const int cols = L->row_bytes / 16 * L->kv_heads;
    if ((long)cols > 0xffffL * 256 || pg->n_seqs > 0xffffff) return QWEN_HIP_EINVAL;
    paged_compact<<<dim3((unsigned)pg->n_seqs, 2 * L->n_layers, (cols + 255) / 256), 256, 0, s>>>(*L, *pg, len_out, path,
                                                                                                path_stride, n_path);
    return hipGetLastError() == hipSuccess ? 0 : QWEN_HIP_EDEVICE;
}
