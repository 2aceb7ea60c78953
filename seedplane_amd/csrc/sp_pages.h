// Which sequences hold which pages of a paged cache, kept on the device: forks, growth, ends, compaction, and the copies these need in
// every layer.
//
// holders[e] is how many table rows name page e (and what the caller adds to keep a page); 0: free.  A sequence's last page, where it
// is not full, is its own: a fork copies its rows for all children but one, so that none ever writes another's positions.  Pages are
// taken lowest first, in the order of sequences and positions, so results do not depend on the order in which blocks run.
//
// The tables are small and their updates a few dependent steps, bound by latency: one block does what needs an order (ranks of free
// pages by scans), a block per sequence what does not, and the last of those to finish goes on as the one.  The copies are bound by
// memory: 16 bytes a thread, a block per (page, layer's keys or values).
#pragma once
#include "sp_device.h"

namespace pages {

constexpr int THREADS = 256;               // per sequence, and of copies
constexpr int SCAN = 1024, PER = 8;        // threads of the ordered steps, pages of each at a time

struct Move { int src, dst, rows; };       // pages, rows of each head
struct Pool {                              // see sp_page_pool
    const uint64_t *pools, *scales;
    int *table, *lengths, *holders, *missing;
    int64_t page_bytes, head_bytes, row_bytes;                         // strides
    int n_pools, n_pages, page, nkv, width_bytes, block, per_page, S, width;      // width_bytes: of a row's values
    bool aligned;                                                      // every row to 16 bytes
    // workspace
    int *arrived;                          // [0] blocks that have finished, [1] moves
    int *fresh, *first;                    // [S] new lengths; [S + 1] places of each sequence's pages among those wanted
    int *rows;                             // [S][width] new table
    int *list;                             // [n_pages] free pages taken
    Move *moves;                           // [max(S, n_pages)]
};

// Exclusive sum over the block of one value per thread, and the total.  SCAN threads.
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
    for (int k = 0; k < SCAN / 64; ++k) {
        const int w = wave_sums[k];
        before += k < wv ? w : 0;
        total += w;
    }
    return before + x - v;
}

// The lowest `want` free pages in order to list; returns how many there are.  SCAN threads.
__device__ __forceinline__ int take_free(const int *holders, int n_pages, int want, int *list, int *wave_sums) {
    int found = 0;
    for (int e0 = 0; e0 < n_pages && found < want; e0 += SCAN * PER) {
        const int at = e0 + (int)threadIdx.x * PER;
        bool free[PER];
        int mine = 0, total;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            free[j] = at + j < n_pages && holders[at + j] == 0;
            mine += free[j];
        }
        int rank = found + block_rank(mine, wave_sums, total);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (free[j] && rank < want) list[rank++] = at + j;
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// Whether this block is the last of gridDim.x to come here; its thread then sees what the others wrote.
__device__ __forceinline__ bool last_block(int *arrived) {
    __shared__ int last_s;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const int n = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        last_s = n == (int)gridDim.x - 1;
        if (last_s) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (last_s) __threadfence();
    return last_s;
}

// ------------------------------------------------------------------------------------------------ fork
// A block per sequence: its new row, holders of what changes.  The last block then takes pages for the copies.
__global__ void __launch_bounds__(SCAN) k_fork(Pool a, const int *parents) {
    __shared__ int wave_sums[SCAN / 64], earlier;
    const int s = blockIdx.x, tid = threadIdx.x;
    {
        const int p = parents[s];
        const bool valid = p >= 0 && p < a.S;
        const int len = valid ? min(a.lengths[p], a.width * a.page) : 0, full = len / a.page, rest = len - full * a.page;
        if (tid == 0) earlier = 0;
        __syncthreads();
        if (valid && rest)
            for (int i = tid; i < s; i += blockDim.x)
                if (parents[i] == p) earlier = 1;
        __syncthreads();
        // (a last page that the parent does not have is missing in its children too)
        const bool copy = earlier && a.table[(int64_t)p * a.width + full] >= 0;
        const int keep = full + (rest && !copy);
        for (int j = tid; j < a.width; j += blockDim.x) {
            const int now = a.table[(int64_t)s * a.width + j], e = j < keep ? a.table[(int64_t)p * a.width + j] : -1;
            a.rows[(int64_t)s * a.width + j] = e;
            if (e != now) {
                if (now >= 0 && now < a.n_pages) atomicSub(&a.holders[now], 1);
                if (e >= 0 && e < a.n_pages) atomicAdd(&a.holders[e], 1);
            }
        }
        if (tid == 0) {
            a.fresh[s] = len;
            a.first[s] = copy ? rest : 0;
        }
    }
    if (!last_block(a.arrived)) return;
    // places of the copies, in order of sequences
    int wanted = 0;
    for (int s0 = 0; s0 < a.S; s0 += SCAN) {
        const int s = s0 + tid, rest = s < a.S ? a.first[s] : 0;
        int total;
        const int at = wanted + block_rank(rest > 0, wave_sums, total);
        if (rest > 0) a.moves[at] = {s, -1, rest};
        wanted += total;
    }
    __syncthreads();
    const int got = take_free(a.holders, a.n_pages, wanted, a.list, wave_sums);
    for (int k = tid; k < wanted; k += SCAN) {
        const int s = a.moves[k].src, full = a.fresh[s] / a.page, p = parents[s];
        const int src = a.table[(int64_t)p * a.width + full], dst = k < got ? a.list[k] : -1;
        if (dst >= 0) a.holders[dst] = 1;
        a.rows[(int64_t)s * a.width + full] = dst;
        a.moves[k].src = src;
        a.moves[k].dst = dst;
    }
    if (tid == 0) {
        a.arrived[1] = got;
        if (wanted > got) *a.missing += wanted - got;
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
    if (a.aligned) {
        const uint32_t per = run / 16, total = per * runs;
        for (uint32_t i0 = threadIdx.x; i0 < total; i0 += THREADS * 4) {
            u32x4 v[4];
            int64_t at[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t i = min(i0 + k * THREADS, total - 1), r = i / per;
                at[k] = place(r) + (i - r * per) * 16;
                v[k] = *(const u32x4 *)(from + at[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i0 + k * THREADS < total) *(u32x4 *)(to + at[k]) = v[k];
        }
    } else {
        const uint32_t total = run * runs;
        for (uint32_t i = threadIdx.x; i < total; i += THREADS) {
            const uint32_t r = i / run;
            const int64_t at = place(r) + (i - r * run);
            to[at] = from[at];
        }
    }
    if (a.scales) {
        float *const s = (float *)a.scales[pool];
        const int blocks = (m.rows + a.block - 1) / a.block;
        for (int i = threadIdx.x; i < a.nkv * blocks; i += THREADS) {
            const int64_t at = (int64_t)(i / blocks) * a.per_page + i % blocks, page = (int64_t)a.nkv * a.per_page;
            s[m.dst * page + at] = s[m.src * page + at];
        }
    }
}
// A fork's copies: block (copy, pool); the first pool's blocks write the tables too.
__global__ void __launch_bounds__(THREADS) k_fork_copy(Pool a) {
    const int pool = blockIdx.y, k = blockIdx.x;
    if (pool == 0) {
        for (int j = threadIdx.x; j < a.width; j += blockDim.x) a.table[(int64_t)k * a.width + j] = a.rows[(int64_t)k * a.width + j];
        if (threadIdx.x == 0) a.lengths[k] = a.fresh[k];
    }
    if (k < a.arrived[1]) copy_page(a, pool, a.moves[k]);
}

// ------------------------------------------------------------------------------------------------ growth, ends
// counts[s] new positions of each sequence: pages for those that have none yet.  One block.
__global__ void __launch_bounds__(SCAN) k_grow(Pool a, const int *counts) {
    __shared__ int wave_sums[SCAN / 64];
    const int tid = threadIdx.x;
    int wanted = 0;
    for (int s0 = 0; s0 < a.S; s0 += SCAN) {
        const int s = s0 + tid;
        int need = 0, total;
        if (s < a.S) {
            const int64_t len = a.lengths[s], grown = min(len + max(counts[s], 0), (int64_t)a.width * a.page);
            need = max(0, (int)((grown + a.page - 1) / a.page - (len + a.page - 1) / a.page));
            a.fresh[s] = (int)grown;
        }
        const int at = wanted + block_rank(need, wave_sums, total);
        if (s < a.S) a.first[s] = at;
        wanted += total;
    }
    if (tid == 0) a.first[a.S] = wanted;
    __syncthreads();
    const int got = take_free(a.holders, a.n_pages, min(wanted, a.n_pages), a.list, wave_sums);
    for (int s = tid >> 4; s < a.S; s += SCAN / 16) {                  // 16 threads a sequence
        const int at = a.first[s], n = a.first[s + 1] - at, have = (a.lengths[s] + a.page - 1) / a.page;
        for (int j = tid & 15; j < n; j += 16) {
            const int e = at + j < got ? a.list[at + j] : -1;
            a.table[(int64_t)s * a.width + have + j] = e;
            if (e >= 0) a.holders[e] = 1;
        }
    }
    __syncthreads();
    int over = 0;
    for (int s = tid; s < a.S; s += SCAN) {
        over += max(a.lengths[s] + (int64_t)max(counts[s], 0) - a.fresh[s], (int64_t)0) > 0;
        a.lengths[s] = a.fresh[s];
    }
    if (over) atomicAdd(a.missing, over);
    if (tid == 0 && wanted > got) atomicAdd(a.missing, wanted - got);
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
__global__ void __launch_bounds__(SCAN) k_compact(Pool a, int *places) {
    __shared__ int wave_sums[SCAN / 64];
    const int tid = threadIdx.x;
    int held = 0;
    for (int e0 = 0; e0 < a.n_pages; e0 += SCAN * PER) {
        const int at = e0 + tid * PER;
        int mine = 0, total;
#pragma unroll
        for (int j = 0; j < PER; ++j) mine += at + j < a.n_pages && a.holders[at + j] != 0;
        block_rank(mine, wave_sums, total);
        held += total;
    }
    int moves = 0;
    for (int e0 = held; e0 < a.n_pages; e0 += SCAN * PER) {
        const int at = e0 + tid * PER;
        bool used[PER];
        int mine = 0, total;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            used[j] = at + j < a.n_pages && a.holders[at + j] != 0;
            mine += used[j];
        }
        int rank = moves + block_rank(mine, wave_sums, total);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (used[j]) a.moves[rank++].src = at + j;
        moves += total;
    }
    const int low = take_free(a.holders, held, moves, a.list, wave_sums);         // (as many as there are moves)
    for (int k = tid; k < low; k += SCAN) {
        const int src = a.moves[k].src, dst = a.list[k];
        a.moves[k].dst = dst;
        a.moves[k].rows = a.page;
        a.holders[dst] = a.holders[src];
    }
    if (places)
        for (int e = tid; e < a.n_pages; e += SCAN) places[e] = e;
    __syncthreads();
    if (places)
        for (int k = tid; k < low; k += SCAN) places[a.moves[k].src] = a.moves[k].dst;
    for (int k = tid; k < low; k += SCAN) a.holders[a.moves[k].src] = 0;
    if (tid == 0) { a.arrived[1] = low; a.arrived[2] = held; }
}
// The compaction's copies, (pool, move) pairs over the grid, and the tables: a page behind the last held one is found among the moves,
// whose sources are in order.
__global__ void __launch_bounds__(THREADS) k_compact_copy(Pool a) {
    const int moves = a.arrived[1], held = a.arrived[2];
    const int64_t entries = (int64_t)a.S * a.width, stride = (int64_t)gridDim.x * blockDim.x;
    if (moves == 0) return;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < entries; i += stride) {
        const int e = a.table[i];
        if (e < held || e >= a.n_pages) continue;
        int lo = 0, hi = moves - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (a.moves[mid].src < e) lo = mid + 1;
            else hi = mid;
        }
        if (a.moves[lo].src == e) a.table[i] = a.moves[lo].dst;
    }
    const int64_t total = (int64_t)moves * a.n_pools;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int k = (int)(w / a.n_pools);
        copy_page(a, (int)(w - (int64_t)k * a.n_pools), a.moves[k]);
    }
}
// Whole pages by lists.
__global__ void __launch_bounds__(THREADS) k_copy(Pool a, const int *src, const int *dst) {
    copy_page(a, blockIdx.y, Move{src[blockIdx.x], dst[blockIdx.x], a.page});
}

}  // namespace pages
