// Which sequences hold which pages of a paged cache, kept on the device: forks, growth, ends, compaction, and the copies these need in
// every layer.
//
// holders[e] is how many table rows name page e (and what the caller adds to keep a page); 0: free.  A sequence's last page, where it
// is not full, is its own: a fork copies its rows for all children but one, so that none ever writes another's positions.  Pages are
// taken lowest first, in the order of sequences and positions, so results do not depend on the order in which blocks run.
//
// The tables are small and their updates a few dependent steps, bound by latency: one block does what needs an order (ranks of free
// pages by scans), the rows of a fork too unless they are many.  The copies are bound by memory: 16 bytes a thread, a block per (page,
// layer's keys or values).
// 16 x 8 beams over 28 layers of 4 heads of 128 in 8 bits: the tables 8 us, 62 MB copied in 25 (5.0 TB/s, a large copy's rate); 1.4 GB compacted
// in 553 us (5.1 TB/s).  A fork of 4 sequences takes 5 + 3.4 us, growth by one position each of 16 sequences 4.6, of 1024 11.
#pragma once
#include "sp_device.h"

namespace pages {

constexpr int THREADS = 256;               // per sequence, and of copies
constexpr int PER = 8;                     // pages of each thread at a time in the ordered steps
// Threads of the ordered steps: few where that does the tables and pages in a turn or two (a block of 16 waves starts later and its barriers
// take longer), else as many as a block has.
constexpr int FEW = 256, MANY = 1024;
constexpr int ROWS_IN_ONE = 16384;         // sequences x pages up to which a fork's one block makes the rows too
constexpr int SEQS_IN_ONE = 2048;

struct Move { int src, dst, rows; };       // pages, rows of each head
struct Pool {                              // see sp_page_pool
    const uint64_t *pools, *scales;
    int *table, *lengths, *holders, *missing;
    int64_t page_bytes, head_bytes, row_bytes;                         // strides
    int n_pools, n_pages, page, nkv, width_bytes, block, per_page, S, width;      // width_bytes: of a row's values
    int unit;                                                          // 16, 4 or 1: every row begins and ends on whole units of as many bytes
    // workspace
    int *counts;                           // moves; held pages; whether rows may have gaps (pages that were not found)
    int *fresh, *first;                    // [S] new lengths; [S + 1] places of each sequence's pages among those wanted
    int *rows;                             // [S][width] new table
    int *list;                             // [n_pages] free pages taken
    int *to;                               // [n_pages] where the pages of a compaction's moves go
    Move *moves;                           // [max(S, n_pages)]
};

// Exclusive sum over the block's N threads of one value each, and the total.
template <int N>
__device__ __forceinline__ int block_rank(int v, int *wave_sums, int &total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) wave_sums[wv] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int k = 0; k < N / 64; ++k) {
        const int w = wave_sums[k];
        before += k < wv ? w : 0;
        total += w;
    }
    return before + x - v;
}

// Holders of pages at .. at + PER - 1 (1 behind the last page).
__device__ __forceinline__ void load_holders(const int *holders, int n_pages, int at, int (&h)[PER]) {
    typedef int Vector __attribute__((ext_vector_type(PER), aligned(4)));
    if (at + PER <= n_pages) {
        const Vector v = *(const Vector *)(holders + at);
#pragma unroll
        for (int j = 0; j < PER; ++j) h[j] = v[j];
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) h[j] = at + j < n_pages ? holders[at + j] : 1;
    }
}

// The lowest `want` free pages in order to list; returns how many there are.
template <int N>
__device__ __forceinline__ int take_free(const int *holders, int n_pages, int want, int *list, int *wave_sums) {
    int found = 0;
    for (int e0 = 0; e0 < n_pages && found < want; e0 += N * PER) {
        const int at = e0 + (int)threadIdx.x * PER;
        int h[PER], mine = 0, total;
        load_holders(holders, n_pages, at, h);
#pragma unroll
        for (int j = 0; j < PER; ++j) mine += h[j] == 0;
        int rank = found + block_rank<N>(mine, wave_sums, total);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (h[j] == 0 && rank < want) list[rank++] = at + j;
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// ------------------------------------------------------------------------------------------------ fork
// A sequence's new row: its length, the pages that it holds in common with its parent, and rows of a last page to copy (0: none).
// A last page that the parent does not have is missing in its children too.
struct Child { int parent, len, keep, copy; };
__device__ __forceinline__ Child child_of(const Pool &a, int p) {
    if (p < 0 || p >= a.S) return {-1, 0, 0, 0};
    const int len = min(max(a.lengths[p], 0), a.width * a.page), full = len / a.page, rest = len - full * a.page;
    const bool has = rest && a.table[(int64_t)p * a.width + full] >= 0;
    return {p, len, full + (rest > 0), has ? rest : 0};
}
// Entry (s, j), where `now` was: e.
__device__ __forceinline__ void fork_entry(const Pool &a, int64_t at, int now, int e) {
    a.rows[at] = e;
    if (e != now) {
        if (now >= 0 && now < a.n_pages) atomicSub(&a.holders[now], 1);
        if (e >= 0 && e < a.n_pages) atomicAdd(&a.holders[e], 1);
    }
}
// A wave a sequence: the first child of a parent keeps its last page.
__global__ void __launch_bounds__(THREADS) k_fork_rows(Pool a, const int *parents) {
    const int s = blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (s >= a.S) return;
    Child c = child_of(a, parents[s]);
    bool earlier = false;
    if (c.copy)
        for (int i = lane; i < s; i += 64) earlier |= parents[i] == c.parent;
    if (__any(earlier)) --c.keep;
    else c.copy = 0;
    for (int j = lane; j < a.width; j += 64) {
        const int64_t at = (int64_t)s * a.width + j;
        fork_entry(a, at, a.table[at], j < c.keep ? a.table[(int64_t)c.parent * a.width + j] : -1);
    }
    if (lane == 0) {
        a.fresh[s] = c.len;
        a.first[s] = c.copy;
    }
}
// Pages for the copies, in the order of sequences.  One block; ROWS: it makes the rows too.
template <bool ROWS, int N>
__global__ void __launch_bounds__(N) k_fork(Pool a, const int *parents) {
    constexpr int M = ROWS ? SEQS_IN_ONE : 1;
    __shared__ int wave_sums[N / 64], parent_s[M], first_s[M], keep_s[M], full_s[M], copy_s[M];
    const int tid = threadIdx.x;
    if constexpr (ROWS) {
        for (int s = tid; s < a.S; s += N) first_s[s] = a.S;
        __syncthreads();
        for (int s = tid; s < a.S; s += N) {
            const Child c = child_of(a, parents[s]);
            if (c.copy) atomicMin(&first_s[c.parent], s);
            parent_s[s] = c.parent;
            keep_s[s] = c.keep;
            full_s[s] = c.len / a.page;
            copy_s[s] = c.copy;
            a.fresh[s] = c.len;
        }
        __syncthreads();
        for (int s = tid; s < a.S; s += N)
            if (copy_s[s]) {
                if (first_s[parent_s[s]] == s) copy_s[s] = 0;
                else --keep_s[s];
            }
        __syncthreads();
        constexpr int AT_ONCE = 4;
        const int entries = a.S * a.width;
        for (int i0 = tid; i0 < entries; i0 += N * AT_ONCE) {
            int now[AT_ONCE], e[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int i = min(i0 + k * N, entries - 1), s = i / a.width, j = i - s * a.width;
                now[k] = a.table[i];
                e[k] = a.table[j < keep_s[s] ? parent_s[s] * a.width + j : i];
                if (j >= keep_s[s]) e[k] = -1;
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k)
                if (i0 + k * N < entries) fork_entry(a, i0 + k * N, now[k], e[k]);
        }
        __syncthreads();
    }
    // first_s / a.first: rows of a last page to copy, then the place of the sequence among those that copy
    int wanted = 0;
    for (int s0 = 0; s0 < a.S; s0 += N) {
        const int s = s0 + tid, rest = s >= a.S ? 0 : ROWS ? copy_s[s] : a.first[s];
        int total;
        const int at = wanted + block_rank<N>(rest > 0, wave_sums, total);
        if (s < a.S) {
            if constexpr (ROWS) first_s[s] = at;
            if (rest > 0) {
                a.moves[at].rows = rest;
                if constexpr (!ROWS) a.moves[at].src = s;
            }
        }
        wanted += total;
    }
    __syncthreads();
    const int got = take_free<N>(a.holders, a.n_pages, wanted, a.list, wave_sums);
    auto place = [&](int s, int p, int full, int k) {
        const int src = a.table[(int64_t)p * a.width + full], dst = k < got ? a.list[k] : -1;
        if (dst >= 0) a.holders[dst] = 1;
        a.rows[(int64_t)s * a.width + full] = dst;
        a.moves[k].src = src;
        a.moves[k].dst = dst;
    };
    if constexpr (ROWS) {
        for (int s = tid; s < a.S; s += N)
            if (copy_s[s]) place(s, parent_s[s], full_s[s], first_s[s]);
    } else {
        for (int k = tid; k < wanted; k += N) {
            const int s = a.moves[k].src;
            place(s, parents[s], a.fresh[s] / a.page, k);
        }
    }
    if (tid == 0) {
        a.counts[0] = got;
        if (wanted > got) { *a.missing += wanted - got; a.counts[2] = 1; }
    }
}

// ------------------------------------------------------------------------------------------------ copies
// Rows 0 .. rows - 1 of every head of page src to page dst of one pool, with the scales of their blocks.
__device__ __forceinline__ void copy_page(const Pool &a, int pool, const Move &m) {
    if (m.src < 0 || m.src >= a.n_pages || m.dst < 0 || m.dst >= a.n_pages) return;
    uint8_t *const base = (uint8_t *)a.pools[pool];
    uint8_t *const to = base + m.dst * a.page_bytes;
    const uint8_t *const from = base + m.src * a.page_bytes;
    // runs of bytes: a head's rows where they lie side by side, else each row
    const bool side = a.row_bytes == a.width_bytes;
    const uint32_t run = side ? m.rows * a.width_bytes : a.width_bytes, runs = side ? a.nkv : a.nkv * m.rows;
    auto place = [&](uint32_t r) -> int64_t {
        if (side) return r * a.head_bytes;
        const uint32_t h = r / m.rows;
        return h * a.head_bytes + (r - h * m.rows) * a.row_bytes;
    };
    auto copy = [&](auto unit) {
        typedef decltype(unit) Unit;
        const uint32_t per = run / sizeof(Unit), total = per * runs;
        for (uint32_t i0 = threadIdx.x; i0 < total; i0 += THREADS * 4) {
            Unit v[4];
            int64_t at[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t i = min(i0 + k * THREADS, total - 1), r = i / per;
                at[k] = place(r) + (i - r * per) * (uint32_t)sizeof(Unit);
                v[k] = *(const Unit *)(from + at[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i0 + k * THREADS < total) *(Unit *)(to + at[k]) = v[k];
        }
    };
    if (a.unit == 16) copy(u32x4{});
    else if (a.unit == 4) copy(uint32_t{});
    else copy(uint8_t{});
    if (a.scales) {
        float *const s = (float *)a.scales[pool];
        const int blocks = (m.rows + a.block - 1) / a.block;
        for (int i = threadIdx.x; i < a.nkv * blocks; i += THREADS) {
            const int64_t at = (int64_t)(i / blocks) * a.per_page + i % blocks, page = (int64_t)a.nkv * a.per_page;
            s[m.dst * page + at] = s[m.src * page + at];
        }
    }
}
// The moves' copies, (move, pool) pairs over the grid's blocks.
__device__ __forceinline__ void copy_moves(const Pool &a, int moves) {
    const int64_t total = (int64_t)moves * a.n_pools;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int k = (int)(w / a.n_pools);
        copy_page(a, (int)(w - (int64_t)k * a.n_pools), a.moves[k]);
    }
}
// A fork's copies, and its tables.
__global__ void __launch_bounds__(THREADS) k_fork_copy(Pool a) {
    const int64_t entries = (int64_t)a.S * a.width, stride = (int64_t)gridDim.x * THREADS, first = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    for (int64_t i = first; i < entries; i += stride) a.table[i] = a.rows[i];
    for (int64_t s = first; s < a.S; s += stride) a.lengths[s] = a.fresh[s];
    copy_moves(a, a.counts[0]);
}

// ------------------------------------------------------------------------------------------------ growth, ends
// A length as the table can hold it: what a program set there never leads outside the table.
__device__ __forceinline__ int length_of(const Pool &a, int s) { return min(max(a.lengths[s], 0), a.width * a.page); }
__device__ __forceinline__ int pages_of(const Pool &a, int len) { return (int)(((uint32_t)len + a.page - 1) / (uint32_t)a.page); }
// counts[s] new positions of each sequence: pages for those that have none yet.  One block.
template <int N>
__global__ void __launch_bounds__(N) k_grow(Pool a, const int *counts) {
    __shared__ int wave_sums[N / 64], behind;
    const int tid = threadIdx.x, gaps = a.counts[2];
    if (tid == 0) behind = 0;
    int wanted = 0;
    for (int s0 = 0; s0 < a.S; s0 += N) {
        const int s = s0 + tid;
        int need = 0, now = -1, total;
        if (s < a.S) {
            const int len = length_of(a, s), grown = len + min(max(counts[s], 0), a.width * a.page - len), have = pages_of(a, len);
            need = pages_of(a, grown) - have;
            a.fresh[s] = grown;
            if (need) now = a.table[(int64_t)s * a.width + have];
        }
        const int at = wanted + block_rank<N>(need, wave_sums, total);
        if (s < a.S) a.first[s] = at;
        if (now >= 0) behind = 1;
        wanted += total;
    }
    if (tid == 0) a.first[a.S] = wanted;
    __syncthreads();
    auto each_new = [&](auto &&fn) {                                // fn(the place among those wanted, its entry); 16 threads a sequence
        for (int s = tid >> 4; s < a.S; s += N / 16) {
            const int at = a.first[s], n = a.first[s + 1] - at, have = pages_of(a, length_of(a, s));
            for (int j = tid & 15; j < n; j += 16) fn(at + j, (int64_t)s * a.width + have + j);
        }
    };
    // Pages that the entries still name, where a program has lowered a sequence's length, are given back first.  (A row without gaps names one in
    // the first of them if in any.)
    if (behind || gaps) {
        each_new([&](int, int64_t entry) {
            const int e = a.table[entry];
            if (e >= 0 && e < a.n_pages) atomicSub(&a.holders[e], 1);
        });
        __syncthreads();
    }
    const int got = take_free<N>(a.holders, a.n_pages, min(wanted, a.n_pages), a.list, wave_sums);
    each_new([&](int k, int64_t entry) {
        const int e = k < got ? a.list[k] : -1;
        a.table[entry] = e;
        if (e >= 0) a.holders[e] = 1;
    });
    __syncthreads();
    int over = 0;
    for (int s = tid; s < a.S; s += N) {
        over += length_of(a, s) + (int64_t)max(counts[s], 0) > a.fresh[s];
        a.lengths[s] = a.fresh[s];
    }
    if (over) atomicAdd(a.missing, over);
    if (tid == 0 && wanted > got) { atomicAdd(a.missing, wanted - got); a.counts[2] = 1; }
}
// Sequences that end: a block each.  (The same one twice gives its pages back once.)
__global__ void __launch_bounds__(THREADS) k_free(Pool a, const int *seqs) {
    const int s = seqs[blockIdx.x];
    if (s < 0 || s >= a.S) return;
    for (int j = threadIdx.x; j < a.width; j += blockDim.x) {
        const int e = atomicExch(&a.table[(int64_t)s * a.width + j], -1);
        if (e >= 0 && e < a.n_pages) atomicSub(&a.holders[e], 1);
    }
    if (threadIdx.x == 0) a.lengths[s] = 0;
}

// ------------------------------------------------------------------------------------------------ compaction
// Held pages at or behind U, the number of held pages, go to the free pages before it, in order.  One block.  places (may be NULL): where
// each page is afterwards.
template <int N>
__global__ void __launch_bounds__(N) k_compact(Pool a, int *places) {
    __shared__ int wave_sums[N / 64];
    const int tid = threadIdx.x;
    int held = 0;
    for (int e0 = 0; e0 < a.n_pages; e0 += N * PER) {
        const int at = e0 + tid * PER;
        int h[PER], mine = 0, total;
        load_holders(a.holders, a.n_pages, at, h);
#pragma unroll
        for (int j = 0; j < PER; ++j) mine += at + j < a.n_pages && h[j] != 0;
        block_rank<N>(mine, wave_sums, total);
        held += total;
    }
    int moves = 0;
    for (int e0 = held; e0 < a.n_pages; e0 += N * PER) {
        const int at = e0 + tid * PER;
        int h[PER], mine = 0, total;
        load_holders(a.holders, a.n_pages, at, h);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            h[j] = at + j < a.n_pages && h[j] != 0;
            mine += h[j];
        }
        int rank = moves + block_rank<N>(mine, wave_sums, total);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (h[j]) a.moves[rank++].src = at + j;
        moves += total;
    }
    const int low = take_free<N>(a.holders, held, moves, a.list, wave_sums);         // (as many as there are moves)
    for (int k = tid; k < low; k += N) {
        const int src = a.moves[k].src, dst = a.list[k];
        a.moves[k].dst = dst;
        a.moves[k].rows = a.page;
        a.to[src] = dst;
        a.holders[dst] = a.holders[src];
    }
    if (places)
        for (int e = tid; e < a.n_pages; e += N) places[e] = e;
    __syncthreads();
    if (places)
        for (int k = tid; k < low; k += N) places[a.moves[k].src] = a.moves[k].dst;
    for (int k = tid; k < low; k += N) a.holders[a.moves[k].src] = 0;
    if (tid == 0) { a.counts[0] = low; a.counts[1] = held; }
}
// The compaction's copies, and the pages behind the last held one in the tables.
__global__ void __launch_bounds__(THREADS) k_compact_copy(Pool a) {
    const int moves = a.counts[0], held = a.counts[1];
    const int64_t entries = (int64_t)a.S * a.width, stride = (int64_t)gridDim.x * THREADS;
    if (moves == 0) return;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < entries; i += stride) {
        const int e = a.table[i];
        if (e >= held && e < a.n_pages) a.table[i] = a.to[e];
    }
    copy_moves(a, moves);
}
// Whole pages by lists.
__global__ void __launch_bounds__(THREADS) k_copy(Pool a, const int *src, const int *dst) {
    copy_page(a, blockIdx.y, Move{src[blockIdx.x], dst[blockIdx.x], a.page});
}

}  // namespace pages
