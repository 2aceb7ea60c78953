// C ABI (include/seedplane_hip.h) of the page pool: forks, growth, ends and compaction of paged sequences.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <utility>

#include "sp_host.h"
#include "sp_pages.h"

namespace {

size_t up(size_t n) { return (n + 15) / 16 * 16; }

struct Places { size_t fresh, first, rows, list, to, moves, total; };
Places places_of(int64_t S, int64_t width, int64_t n_pages) {
    Places p{};
    p.fresh = 64;
    p.first = p.fresh + up(S * 4);
    p.rows = p.first + up((S + 1) * 4);
    p.list = p.rows + up(S * width * 4);
    p.to = p.list + up(n_pages * 4);
    p.moves = p.to + up(n_pages * 4);
    p.total = p.moves + up(std::max(S, n_pages) * sizeof(pages::Move));
    return p;
}
bool sizes_ok(int64_t S, int64_t width, int64_t n_pages) {
    return S >= 1 && S <= 65535 && width >= 1 && n_pages >= 1 && S * width < (1 << 30);
}

// Whether no two rows of the pool share a byte: taken from the smallest stride on, each dimension steps over all that those before it reach.
bool rows_apart(const sp_page_pool *p) {
    std::pair<int64_t, int> dims[] = {{p->page_stride, p->n_pages}, {p->head_stride, p->n_kv_heads}, {p->row_stride, p->page_size}};
    std::sort(std::begin(dims), std::end(dims));
    __int128 reach = p->head_dim;
    for (const auto &[stride, n] : dims) {
        if (n == 1) continue;
        if (stride < reach) return false;
        reach += (__int128)stride * (n - 1);
    }
    return true;
}

// gives: the call gives pages to sequences or takes them back, by their numbers alone.
pages::Pool pool_args(const sp_page_pool *p, bool gives = true) {
    require(p != nullptr, SP_EINVAL, "pool is NULL");
    require(sizes_ok(p->max_seqs, p->max_pages, p->n_pages), SP_EINVAL,
            "max_seqs must be in [1, 65535], max_pages and n_pages positive and max_seqs * max_pages below 2^30");
    const int b = p->dtype == SP_DT_F16 || p->dtype == SP_DT_BF16 ? 2 : p->dtype == SP_DT_E4M3 || p->dtype == SP_DT_I8 ? 1 : 0;
    require(b != 0, SP_EINVAL, "dtype must be SP_DT_F16, SP_DT_BF16, SP_DT_E4M3 or SP_DT_I8");
    require(p->n_pools >= 1 && p->n_pools <= 65535 && p->page_size >= 1 && p->n_kv_heads >= 1 && p->head_dim >= 1, SP_EINVAL,
            "the pool's sizes must be positive, n_pools at most 65535");
    require((double)p->page_size * p->n_kv_heads * p->head_dim * b < (double)(1u << 31) && (double)p->max_pages * p->page_size < (double)(1u << 31),
            SP_EINVAL, "a page must be below 2^31 bytes and a sequence below 2^31 positions");
    require((p->n_pages == 1 || p->page_stride >= p->head_dim) && (p->n_kv_heads == 1 || p->head_stride >= p->head_dim) &&
                (p->page_size == 1 || p->row_stride >= p->head_dim) && p->page_stride >= 0 && p->head_stride >= 0 && p->row_stride >= 0,
            SP_EINVAL, "the pool's strides are smaller than a row");
    require(!gives || rows_apart(p), SP_EINVAL, "the pool's pages lie on each other: it can only copy");
    require(p->pools_dev && p->table_dev && p->lengths_dev && p->holders_dev && p->missing_dev && p->workspace_dev, SP_EINVAL, "NULL pointer");
    require(((uintptr_t)p->workspace_dev & 15) == 0, SP_EINVAL, "the workspace must be aligned to 16 bytes");
    require((p->scale_block > 0) == (p->scales_dev != nullptr) && p->scale_block >= 0 &&
                (!p->scale_block || p->page_size % p->scale_block == 0), SP_EINVAL, "scales come with a scale_block that divides page_size");
    pages::Pool a{};
    a.pools = p->pools_dev; a.scales = p->scales_dev;
    a.table = p->table_dev; a.lengths = p->lengths_dev; a.holders = p->holders_dev; a.missing = p->missing_dev;
    a.page_bytes = p->page_stride * b; a.head_bytes = p->head_stride * b; a.row_bytes = p->row_stride * b;
    a.n_pools = p->n_pools; a.n_pages = p->n_pages; a.page = p->page_size; a.nkv = p->n_kv_heads; a.width_bytes = p->head_dim * b;
    a.block = p->scale_block; a.per_page = p->scale_block ? p->page_size / p->scale_block : 0;
    a.S = p->max_seqs; a.width = p->max_pages;
    // (a fork of 16 x 8 beams over 28 layers of 4 heads of 72 in 8 bits: by bytes 106 us, by 4 of them 42)
    const int64_t all = a.page_bytes | a.head_bytes | a.row_bytes | a.width_bytes;
    a.unit = !p->aligned16 || all % 4 ? 1 : all % 16 ? 4 : 16;
    const Places at = places_of(a.S, a.width, a.n_pages);
    uint8_t *const w = (uint8_t *)p->workspace_dev;
    a.counts = (int *)w;
    a.fresh = (int *)(w + at.fresh);
    a.first = (int *)(w + at.first);
    a.rows = (int *)(w + at.rows);
    a.list = (int *)(w + at.list);
    a.to = (int *)(w + at.to);
    a.moves = (pages::Move *)(w + at.moves);
    return a;
}

// Blocks of up to `moves` copies in every pool: one each, up to four times as many as the chip holds (1.4 GB moved: 571 us, by 2048 blocks 586).
int copy_blocks(const pages::Pool &a, int64_t moves) { return (int)std::min<int64_t>(std::max<int64_t>(moves * a.n_pools, 1), 8192); }
bool few(const pages::Pool &a) { return a.S <= pages::FEW && a.n_pages <= 2 * pages::FEW * pages::PER && (int64_t)a.S * a.width <= 8 * pages::FEW; }

}  // namespace

extern "C" {

size_t sp_pages_workspace(int32_t max_seqs, int32_t max_pages, int32_t n_pages) {
    return sizes_ok(max_seqs, max_pages, n_pages) ? places_of(max_seqs, max_pages, n_pages).total : 0;
}

int sp_op_pages_fork(const sp_page_pool *pool, const int32_t *parents_dev, void *stream) {
    return guarded([&] {
        const pages::Pool a = pool_args(pool);
        require(parents_dev != nullptr, SP_EINVAL, "NULL pointer");
        const hipStream_t st = (hipStream_t)stream;
        if ((int64_t)a.S * a.width <= pages::ROWS_IN_ONE && a.S <= pages::SEQS_IN_ONE) {
            if (few(a)) hipLaunchKernelGGL((pages::k_fork<true, pages::FEW>), dim3(1), dim3(pages::FEW), 0, st, a, parents_dev);
            else hipLaunchKernelGGL((pages::k_fork<true, pages::MANY>), dim3(1), dim3(pages::MANY), 0, st, a, parents_dev);
        } else {
            constexpr int per = pages::THREADS / 64;
            hipLaunchKernelGGL(pages::k_fork_rows, dim3((a.S + per - 1) / per), dim3(pages::THREADS), 0, st, a, parents_dev);
            HIPCHK(hipGetLastError());
            hipLaunchKernelGGL((pages::k_fork<false, pages::MANY>), dim3(1), dim3(pages::MANY), 0, st, a, parents_dev);
        }
        HIPCHK(hipGetLastError());
        hipLaunchKernelGGL(pages::k_fork_copy, dim3(copy_blocks(a, a.S)), dim3(pages::THREADS), 0, st, a);
        HIPCHK(hipGetLastError());
    });
}

int sp_op_pages_grow(const sp_page_pool *pool, const int32_t *counts_dev, void *stream) {
    return guarded([&] {
        const pages::Pool a = pool_args(pool);
        require(counts_dev != nullptr, SP_EINVAL, "NULL pointer");
        if (few(a)) hipLaunchKernelGGL(pages::k_grow<pages::FEW>, dim3(1), dim3(pages::FEW), 0, (hipStream_t)stream, a, counts_dev);
        else hipLaunchKernelGGL(pages::k_grow<pages::MANY>, dim3(1), dim3(pages::MANY), 0, (hipStream_t)stream, a, counts_dev);
        HIPCHK(hipGetLastError());
    });
}

int sp_op_pages_free(const sp_page_pool *pool, int32_t n_seqs, const int32_t *seqs_dev, void *stream) {
    return guarded([&] {
        const pages::Pool a = pool_args(pool);
        require(n_seqs >= 0, SP_EINVAL, "n_seqs must not be negative");
        if (n_seqs == 0) return;
        require(seqs_dev != nullptr, SP_EINVAL, "NULL pointer");
        hipLaunchKernelGGL(pages::k_free, dim3(n_seqs), dim3(pages::THREADS), 0, (hipStream_t)stream, a, seqs_dev);
        HIPCHK(hipGetLastError());
    });
}

int sp_op_pages_compact(const sp_page_pool *pool, int32_t *places_dev, void *stream) {
    return guarded([&] {
        const pages::Pool a = pool_args(pool);
        if (few(a)) hipLaunchKernelGGL(pages::k_compact<pages::FEW>, dim3(1), dim3(pages::FEW), 0, (hipStream_t)stream, a, places_dev);
        else hipLaunchKernelGGL(pages::k_compact<pages::MANY>, dim3(1), dim3(pages::MANY), 0, (hipStream_t)stream, a, places_dev);
        HIPCHK(hipGetLastError());
        hipLaunchKernelGGL(pages::k_compact_copy, dim3(copy_blocks(a, a.n_pages / 2)), dim3(pages::THREADS), 0, (hipStream_t)stream, a);
        HIPCHK(hipGetLastError());
    });
}

int sp_op_pages_copy(const sp_page_pool *pool, int32_t n_copies, const int32_t *src_dev, const int32_t *dst_dev, void *stream) {
    return guarded([&] {
        const pages::Pool a = pool_args(pool, false);
        require(n_copies >= 0, SP_EINVAL, "n_copies must not be negative");
        if (n_copies == 0) return;
        require(src_dev && dst_dev, SP_EINVAL, "NULL pointer");
        hipLaunchKernelGGL(pages::k_copy, dim3(n_copies, a.n_pools), dim3(pages::THREADS), 0, (hipStream_t)stream, a, src_dev, dst_dev);
        HIPCHK(hipGetLastError());
    });
}

}  // extern "C"
