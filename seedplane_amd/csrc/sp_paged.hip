// C ABI (include/seedplane_hip.h) of the operators around a paged K/V cache: rotation, append, shared-prefix attention.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>
#include <type_traits>

#include "sp_host.h"
#include "sp_blocks.h"
#include "sp_paged.h"
#include "sp_paged_plan.h"
#include "sp_rotate.h"

using namespace paged;

namespace {

bool is_capturing(hipStream_t st) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    HIPCHK(hipStreamIsCapturing(st, &cs));
    return cs != hipStreamCaptureStatusNone;
}

int bytes_of(int dt) { return dt == SP_DT_F32 ? 4 : dt == SP_DT_E4M3 || dt == SP_DT_I8 ? 1 : 2; }
bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

Rotation rotation_of(const sp_rotary *r, int hd) {
    if (!r) return Rotation{nullptr, 0, 0, 1.f};
    require(r->inv_freq_dev != nullptr, SP_EINVAL, "inv_freq_dev is NULL");
    require(r->rot_dim >= 2 && r->rot_dim % 2 == 0 && r->rot_dim <= hd, SP_EINVAL,
            "rot_dim must be even and in [2, head_dim]");
    require(r->layout == SP_ROPE_HALF || r->layout == SP_ROPE_INTERLEAVED, SP_EINVAL,
            "layout must be SP_ROPE_HALF or SP_ROPE_INTERLEAVED");
    return Rotation{r->inv_freq_dev, r->rot_dim, r->layout == SP_ROPE_INTERLEAVED, r->factor};
}

// Vectors of 8 values are used where every vector of the operands is aligned to 16 bytes (8 for a type of 8 bits).
bool wide_ok(const void *p, int dt, int64_t row, int64_t head) {
    return aligned(p, bytes_of(dt) == 1 ? 8 : 16) && row % 8 == 0 && head % 8 == 0;
}

// The bytes of [rows][heads][hd] values at strides row and head (elements); empty where there are none.
struct Span {
    uintptr_t lo = 0, hi = 0, row = 0, width = 0;            // first and last + 1 byte; row stride, bytes of a row from its start
    bool folded = false;                                     // rows or heads lie on top of each other, or run backwards
};
Span span_of(const void *p, int dt, int64_t rows, int64_t heads, int64_t hd, int64_t row, int64_t head) {
    Span s;
    const int b = bytes_of(dt);
    s.folded = (rows > 1 && row < hd) || (heads > 1 && head < hd) ||
               (rows > 1 && heads > 1 && row < (heads - 1) * head + hd && head < (rows - 1) * row + hd);
    if (s.folded || !rows || !heads) return s;
    s.lo = (uintptr_t)p;
    s.width = ((heads - 1) * head + hd) * b;
    s.row = row * b;
    s.hi = s.lo + (rows - 1) * s.row + s.width;
    return s;
}
// Whether two spans may share a byte: they do not where their rows have one stride and lie beside each other in it.
bool overlap(const Span &a, const Span &b) {
    if (a.lo >= b.hi || b.lo >= a.hi) return false;
    if (a.row != b.row || !a.row || a.width > a.row || b.width > b.row) return true;
    const uintptr_t off = b.lo >= a.lo ? (b.lo - a.lo) % a.row : (a.row - (a.lo - b.lo) % a.row) % a.row;
    return off < a.width || off + b.width > a.row;
}
bool may_overlap(const Span &out, const void *p, int dt, int64_t rows, int64_t heads, int64_t hd, int64_t row, int64_t head) {
    const Span in = span_of(p, dt, rows, heads, hd, row, head);
    if (!in.folded) return overlap(out, in);
    // rows or heads of the input repeat (stride 0, sliding windows): its outer bytes
    const int b = bytes_of(dt);
    const int64_t r = (rows - 1) * row, h = (heads - 1) * head;
    const intptr_t lo = (intptr_t)p + (std::min<int64_t>(r, 0) + std::min<int64_t>(h, 0)) * b;
    const intptr_t hi = (intptr_t)p + (std::max<int64_t>(r, 0) + std::max<int64_t>(h, 0) + hd) * b;
    return lo < (intptr_t)out.hi && (intptr_t)out.lo < hi;
}
// A cache's keys or values, from the first byte to the last.
Span pool_of(const sp_paged_kv *kv, const void *p) {
    Span s;
    s.lo = (uintptr_t)p;
    s.hi = s.lo + (uintptr_t)((kv->n_pages - 1) * kv->page_stride + (kv->n_kv_heads - 1) * kv->head_stride +
                              (kv->page_size - 1) * kv->row_stride + kv->head_dim) * bytes_of(kv->dtype);
    return s;
}
void check_output(const Span &out) { require(!out.folded, SP_EINVAL, "the output's rows or heads lie on top of each other"); }

// Rows of a block and its threads: about 256 threads a block, whole rows.
void shape_of(int per_row, int rows, int &per_block, int &threads) {
    per_block = std::max(1, std::min(rows, 256 / per_row));
    threads = std::min(ROT_THREADS, (per_block * per_row + 63) / 64 * 64);
}

template <class F>
void for_input(int dt, bool wide, F &&fn) {
    if (dt == SP_DT_F32) { if (wide) fn((float *)nullptr, std::integral_constant<int, 8>{}); else fn((float *)nullptr, std::integral_constant<int, 1>{}); }
    else if (dt == SP_DT_F16) { if (wide) fn((f16 *)nullptr, std::integral_constant<int, 8>{}); else fn((f16 *)nullptr, std::integral_constant<int, 1>{}); }
    else { if (wide) fn((bf16 *)nullptr, std::integral_constant<int, 8>{}); else fn((bf16 *)nullptr, std::integral_constant<int, 1>{}); }
}

void check_cache(const sp_paged_kv *kv) {
    require(kv && kv->k_dev && kv->v_dev, SP_EINVAL, "NULL cache");
    const bool codes = kv->dtype == SP_DT_E4M3 || kv->dtype == SP_DT_I8;
    require(kv->dtype == SP_DT_F16 || kv->dtype == SP_DT_BF16 || codes, SP_EINVAL,
            "the cache's dtype must be SP_DT_F16, SP_DT_BF16, SP_DT_E4M3 or SP_DT_I8");
    require(kv->n_pages >= 1 && kv->page_size >= 1 && kv->n_kv_heads >= 1 && kv->head_dim >= 2, SP_EINVAL,
            "the cache's sizes must be positive");
    require((kv->n_pages == 1 || kv->page_stride >= kv->head_dim) && (kv->n_kv_heads == 1 || kv->head_stride >= kv->head_dim) &&
                (kv->page_size == 1 || kv->row_stride >= kv->head_dim) && kv->page_stride >= 0 && kv->head_stride >= 0 && kv->row_stride >= 0,
            SP_EINVAL, "the cache's strides are smaller than a row");
    int64_t reach = kv->head_dim, more = 0;
    const int64_t dims[3][2] = {{kv->n_pages, kv->page_stride}, {kv->n_kv_heads, kv->head_stride}, {kv->page_size, kv->row_stride}};
    for (const auto &d : dims)
        require(!__builtin_mul_overflow(d[0] - 1, d[1], &more) && more < ((int64_t)1 << 60) && (reach += more) < ((int64_t)1 << 60),
                SP_EINVAL, "the cache is too large");
    require(codes == (kv->k_scale_dev != nullptr) && codes == (kv->v_scale_dev != nullptr),
            SP_EINVAL, "a cache of 8 bits has k_scale_dev and v_scale_dev, others have none");
    require(kv->scale_block >= 0 && (kv->scale_block == 0 || codes), SP_EINVAL, "only caches of 8 bits have a scale_block");
    require(kv->dtype != SP_DT_I8 || kv->scale_block, SP_EINVAL, "an int8 cache has a scale_block");
    require(kv->scale_block % SCALE_KEYS == 0 && kv->scale_block <= MOST_BLOCK && (!kv->scale_block || kv->page_size % kv->scale_block == 0),
            SP_EINVAL, "scale_block must be a multiple of 16 up to 128 that divides page_size");
    require(!kv->scale_block || (double)kv->n_pages * kv->n_kv_heads * (kv->page_size / kv->scale_block) < 1e15, SP_EINVAL, "the cache is too large");
}

// The scales of a cache in blocks, of keys or of values.
Span scales_of(const sp_paged_kv *kv, const float *p) {
    Span s;
    s.lo = (uintptr_t)p;
    s.hi = s.lo + (uintptr_t)kv->n_pages * kv->n_kv_heads * (kv->page_size / kv->scale_block) * sizeof(float);
    return s;
}

// Rows of blocks with scales of their own: see sp_blocks.h.  a: the append's arguments as for other caches.
void append_blocks(const sp_paged_kv *kv, AppendArgs &a, int dtype, bool wide, hipStream_t st) {
    BlockAppendArgs b{};
    (AppendArgs &)b = a;
    b.kscale = const_cast<float *>(kv->k_scale_dev); b.vscale = const_cast<float *>(kv->v_scale_dev);      // (written with scale_block alone)
    b.block = kv->scale_block; b.per_page = kv->page_size / kv->scale_block;
    b.by_block = PageDivisor(b.block); b.by_page = PageDivisor(kv->page_size);
    b.by_key = PageDivisor(a.units + a.tail); b.by_value = PageDivisor(a.vecs);
    // Blocks that the call is likely to write: of many sequences (a step) one each, else its rows side by side.  Where there is one for every
    // other row a workgroup looks at one row, else at several, most of which follow one of the same block; heads are split while the
    // blocks are too few to fill the chip.  (A step of 1024 sequences, 28 / 4 heads of 128: 14.2 us a call; by 4 rows and single heads twice that.)
    // The host knows a call's sequences only by the table's height, so that a prompt beside a tall table is laid out as a step: 1777 rows of one
    // sequence 47 us with a table of 1024, 14.6 with its own row; 300 rows 20 and 13.
    // More than 4096 rows: the search of all rows for each block comes to count, so that a workgroup takes several blocks with one search
    // (131072 rows of 16 sequences 595 us, by single searches 1154; 8192 38 and 40; 1777 18 and 14).
    const int runs = std::max(1, std::min(a.rows, std::max(a.rows / b.block, a.n_seq)));
    b.find = a.rows > 4096;
    b.chunk = b.find ? std::min(MOST_CHUNK, std::max(b.block, a.rows / 512)) : 2 * (int64_t)runs >= a.rows ? 1 : std::max(1, a.rows / 256);
    b.chunks = (a.rows + b.chunk - 1) / b.chunk;
    b.splits = std::max((a.nkv + BLOCK_HEADS - 1) / BLOCK_HEADS, std::min(a.nkv, 256 / runs));
    b.heads = (a.nkv + b.splits - 1) / b.splits;
    b.splits = (a.nkv + b.heads - 1) / b.heads;
    // the queries' rows are the plain append's, without keys and values
    b.turned = a.nq * a.units;
    b.rest = a.nq * a.tail;
    b.per_row = b.turned + b.rest;
    int query_blocks = 0;
    size_t lds = (size_t)b.block * (a.rot.rot / 2) * sizeof(float2);
    if (a.nq) {
        b.by_row = Divisor(b.per_row);
        b.per_block = std::max(1, std::min(a.rows, 256 / b.per_row));
        query_blocks = (a.rows + b.per_block - 1) / b.per_block;
        lds = std::max(lds, (size_t)b.per_block * (sizeof(int64_t) + (a.rot.rot / 2) * sizeof(float2)));
    }
    launch_block_append(dtype, wide, b, query_blocks, lds, st);
}

}  // namespace

struct sp_attn_plan {
    int NH = 0, NKV = 0, HD = 0, max_rows = 0, max_seqs = 0, device = 0;
    // device block: header [16] (items, tokens, most records of a token) and token records; then, at item_at, the items, and backwards
    // from there the list of tokens that are no range
    int32_t *dev = nullptr;
    size_t tok_at = 0, item_at = 0, words = 0;
    int32_t *staging[2] = {};            // pinned images of the block, used in turn
    hipEvent_t copied[2] = {};
    bool used[2] = {};
    int turn = 0;
    // the last set()
    bool set = false, joined = false;
    int n_items = 0, n_tok = 0, n_seq = 0, max_kv = 0, most_parts = 0;

    void release() {
        for (int i = 0; i < 2; ++i) {
            if (copied[i]) { (void)hipEventSynchronize(copied[i]); (void)hipEventDestroy(copied[i]); }
            if (staging[i]) (void)hipHostFree(staging[i]);
        }
        dev_free(dev);
    }
};

namespace {

constexpr size_t HEADER = 16;

// The plan's shape and where its tables lie (words).
void lay_out(sp_attn_plan &p) {
    p.tok_at = HEADER;
    p.item_at = (p.tok_at + (size_t)p.max_rows * (sizeof(TokenRecs) / 4 + 1) + 15) / 16 * 16;
    p.words = p.item_at + (size_t)items_bound(p.max_rows, p.NKV) * (sizeof(Item) / 4);
}

void check_shape(int NH, int NKV, int HD, int max_rows, int max_seqs) {
    require(NH >= 1 && NH <= 65535 && NKV >= 1 && NH % NKV == 0 && NH / NKV <= MAX_GROUP, SP_EINVAL,
            "n_heads must be at most 65535 and a multiple of n_kv_heads with at most 32 query heads per kv head");
    require(HD == 64 || HD == 128, SP_EINVAL, "head_dim must be 64 or 128");
    require(max_rows >= 1 && max_seqs >= 1 && max_seqs <= 65535 && (int64_t)max_rows * NH <= (1 << 27), SP_EINVAL,
            "max_rows and max_seqs must be positive, max_seqs at most 65535 and max_rows * n_heads at most 2^27");
}

// The checks of sp_attn_plan_set / sp_attn_plan_items; returns the number of tokens.
int check_lengths(int n_seq, const int32_t *q_len, const int32_t *kv_len, int n_groups, const int32_t *size, const int32_t *shared,
                  int max_rows, int max_seqs) {
    require(q_len && kv_len && (n_groups == 0 || (size && shared)), SP_EINVAL, "NULL pointer");
    require(n_seq >= 1 && n_seq <= max_seqs, SP_EINVAL, "n_seq must be in [1, max_seqs]");
    int64_t tokens = 0;
    for (int s = 0; s < n_seq; ++s) {
        require(q_len[s] >= 0 && kv_len[s] >= 0 && kv_len[s] < ALL_SEEN, SP_EINVAL, "q_len and kv_len must be in [0, 2^30)");
        tokens += q_len[s];
    }
    require(tokens <= max_rows, SP_EINVAL, "the queries exceed max_rows");
    require(n_groups >= 0 && n_groups <= n_seq, SP_EINVAL, "n_groups must be in [0, n_seq]");
    int64_t at = 0;
    for (int g = 0; g < n_groups; ++g) {
        require(size[g] >= 1 && at + size[g] <= n_seq && shared[g] >= 0, SP_EINVAL,
                "a group has at least one sequence, a shared length of at least 0, and the groups are the n_seq sequences in order");
        for (int s = (int)at; s < at + size[g]; ++s)
            require(q_len[s] == 0 || kv_len[s] >= shared[g], SP_EINVAL, "a sequence is shorter than its group's shared length");
        at += size[g];
    }
    require(n_groups == 0 || at == n_seq, SP_EINVAL, "the groups do not cover the n_seq sequences");
    return (int)tokens;
}

void tables_of(int NH, int NKV, int HD, int n_seq, const int32_t *q_len, const int32_t *kv_len, int n_groups, const int32_t *size,
               const int32_t *shared, PlanTables &t) {
    std::vector<int32_t> one, none;
    if (n_groups == 0) {                                     // no sharing: every sequence a group of its own
        one.assign(n_seq, 1);
        none.assign(n_seq, 0);
        make_plan(NH, NKV, HD, n_seq, q_len, kv_len, n_seq, one.data(), none.data(), t);
    } else {
        make_plan(NH, NKV, HD, n_seq, q_len, kv_len, n_groups, size, shared, t);
    }
}

template <class T, int KV, int HD>
void launch_items(const AttnArgs &a, int grid, hipStream_t st) {
    hipLaunchKernelGGL((k_paged_attn<T, KV, HD>), dim3(grid), dim3(256), attn_smem<KV>, st, a);
}
template <class T>
void launch_typed(bool kv8, int HD, const AttnArgs &a, int grid, hipStream_t st) {
    if (kv8) { if (HD == 128) launch_items<T, KV_E4M3, 128>(a, grid, st); else launch_items<T, KV_E4M3, 64>(a, grid, st); }
    else { if (HD == 128) launch_items<T, KV_16, 128>(a, grid, st); else launch_items<T, KV_16, 64>(a, grid, st); }
}
// A wave joins a (token, head) whose records it has in flight at once; more are shared by the block's four waves (15 records of 96
// tokens x 28 heads: 8.1 us by four, 5.1 by one).
// (A captured launch leaves the choice to the kernel.)
template <class T, int HD>
void launch_join(const JoinArgs &j, int tokens, bool capturing, int most_parts, hipStream_t st) {
    if (capturing) hipLaunchKernelGGL((k_paged_join<T, HD, 0>), dim3(tokens, j.NH), dim3(256), 0, st, j);
    else if (most_parts > JOIN_BATCH<HD>) hipLaunchKernelGGL((k_paged_join<T, HD, 4>), dim3(tokens, j.NH), dim3(256), 0, st, j);
    else hipLaunchKernelGGL((k_paged_join<T, HD, 1>), dim3(tokens, (j.NH + 3) / 4), dim3(256), 0, st, j);
}

// Blocks of a captured launch, whose item counts may change between replays: each block walks the items grid by grid.
constexpr int CAPTURED_GRID = 512;

}  // namespace

extern "C" {

int sp_op_rotate(const sp_rotary *rotary, int32_t dtype, int32_t n_rows, int32_t n_heads, int32_t head_dim, const void *x_dev,
                 int64_t x_row, int64_t x_head, void *out_dev, int64_t out_row, int64_t out_head, const int32_t *pos_dev,
                 void *stream) {
    return guarded([&] {
        require(dtype == SP_DT_F32 || dtype == SP_DT_F16 || dtype == SP_DT_BF16, SP_EINVAL,
                "dtype must be SP_DT_F32, SP_DT_F16 or SP_DT_BF16");
        require(n_rows >= 0 && n_heads >= 1 && head_dim >= 2 && head_dim <= 1024 && (int64_t)n_heads * head_dim < (1 << 16),
                SP_EINVAL, "n_rows must not be negative, head_dim in [2, 1024] and n_heads * head_dim below 2^16");
        require(rotary != nullptr, SP_EINVAL, "rotary is NULL");
        const Rotation rot = rotation_of(rotary, head_dim);
        if (n_rows == 0) return;
        require(x_dev && out_dev && pos_dev, SP_EINVAL, "NULL pointer");
        const bool in_place = x_dev == out_dev && x_row == out_row && x_head == out_head;
        const Span to = span_of(out_dev, dtype, n_rows, n_heads, head_dim, out_row, out_head);
        check_output(to);
        require(in_place || !may_overlap(to, x_dev, dtype, n_rows, n_heads, head_dim, x_row, x_head), SP_EINVAL,
                "the output overlaps the input");
        RotateArgs a{};
        a.rot = rot;
        a.x = x_dev; a.out = out_dev;
        a.x_row = x_row; a.x_head = x_head; a.out_row = out_row; a.out_head = out_head;
        a.pos = pos_dev;
        a.rows = n_rows; a.heads = n_heads;
        const bool wide = wide_ok(x_dev, dtype, x_row, x_head) && wide_ok(out_dev, dtype, out_row, out_head) &&
                          rot.rot % 16 == 0 && head_dim % 8 == 0;
        const int vec = wide ? 8 : 1;
        a.units = rot.rot / 2 / vec;
        a.per_head = a.units + (in_place ? 0 : (head_dim - rot.rot) / vec);
        a.per_row = n_heads * a.per_head;
        a.by_row = Divisor(a.per_row); a.by_head = Divisor(a.per_head); a.by_half = Divisor(rot.rot / 2);
        int threads;
        shape_of(a.per_row, n_rows, a.per_block, threads);
        for_input(dtype, wide, [&](auto *t, auto v) {
            hipLaunchKernelGGL((k_rotate<std::remove_pointer_t<decltype(t)>, decltype(v)::value>),
                               dim3((n_rows + a.per_block - 1) / a.per_block), dim3(threads),
                               (size_t)a.per_block * (rot.rot / 2) * sizeof(float2), (hipStream_t)stream, a);
        });
        HIPCHK(hipGetLastError());
    });
}

int sp_op_paged_append(const sp_paged_kv *kv, const sp_rotary *rotary, int32_t dtype, int32_t n_rows, int32_t n_heads,
                       const void *q_dev, int64_t q_row, int64_t q_head, const void *k_dev, int64_t k_row, int64_t k_head,
                       const void *v_dev, int64_t v_row, int64_t v_head, const int32_t *pos_dev, const int32_t *seq_dev,
                       const int32_t *at_dev, const int32_t *table_dev, int32_t n_seq, int32_t max_pages, void *q_out_dev,
                       int32_t q_out_dtype, int64_t q_out_row, int64_t q_out_head, void *stream) {
    return guarded([&] {
        check_cache(kv);
        require(dtype == SP_DT_F32 || dtype == SP_DT_F16 || dtype == SP_DT_BF16, SP_EINVAL,
                "dtype must be SP_DT_F32, SP_DT_F16 or SP_DT_BF16");
        const int hd = kv->head_dim, nq = q_dev ? n_heads : 0;
        require(hd <= 1024 && n_rows >= 0 && (!q_dev || n_heads >= 1) && (std::max(nq, 0) + 2 * (int64_t)kv->n_kv_heads) * hd < (1 << 16),
                SP_EINVAL, "n_rows must not be negative, head_dim at most 1024 and the values of a row below 2^16");
        require((q_dev != nullptr) == (q_out_dev != nullptr), SP_EINVAL, "q_dev and q_out_dev come together");
        require(!q_dev || q_out_dtype == SP_DT_F32 || q_out_dtype == SP_DT_F16 || q_out_dtype == SP_DT_BF16, SP_EINVAL,
                "q_out_dtype must be SP_DT_F32, SP_DT_F16 or SP_DT_BF16");
        require(n_seq >= 1 && max_pages >= 1, SP_EINVAL, "n_seq and max_pages must be positive");
        const Rotation rot = rotation_of(rotary, hd);
        require(!kv->scale_block || (kv->scale_block * (int64_t)rot.rot <= 16384 && kv->scale_block * (int64_t)hd < (1 << 16)), SP_EINVAL,
                "scale_block * rot_dim must be at most 16384 and scale_block * head_dim below 65536");
        require(!kv->scale_block || (int64_t)max_pages * kv->page_size <= (1 << 30), SP_EINVAL, "a table over blocks must be of at most 2^30 positions");
        if (n_rows == 0) return;
        require(k_dev && v_dev && seq_dev && at_dev && table_dev && (!rotary || pos_dev), SP_EINVAL, "NULL pointer");
        require(kv->k_dev != kv->v_dev, SP_EINVAL, "keys and values need memory of their own");
        for (const void *p : {kv->k_dev, kv->v_dev}) {
            const Span pool = pool_of(kv, p);
            require(!may_overlap(pool, k_dev, dtype, n_rows, kv->n_kv_heads, hd, k_row, k_head) &&
                        !may_overlap(pool, v_dev, dtype, n_rows, kv->n_kv_heads, hd, v_row, v_head) &&
                        (!q_dev || (!may_overlap(pool, q_dev, dtype, n_rows, nq, hd, q_row, q_head) &&
                                    !may_overlap(pool, q_out_dev, q_out_dtype, n_rows, nq, hd, q_out_row, q_out_head))),
                    SP_EINVAL, "the queries, keys or values overlap the cache");
        }
        if (kv->scale_block) {
            const Span ks = scales_of(kv, kv->k_scale_dev), vs = scales_of(kv, kv->v_scale_dev);
            require(!overlap(ks, vs), SP_EINVAL, "keys' and values' scales need memory of their own");
            for (const Span &s : {ks, vs})
                require(!overlap(s, pool_of(kv, kv->k_dev)) && !overlap(s, pool_of(kv, kv->v_dev)) &&
                            !may_overlap(s, k_dev, dtype, n_rows, kv->n_kv_heads, hd, k_row, k_head) &&
                            !may_overlap(s, v_dev, dtype, n_rows, kv->n_kv_heads, hd, v_row, v_head) &&
                            (!q_dev || (!may_overlap(s, q_dev, dtype, n_rows, nq, hd, q_row, q_head) &&
                                        !may_overlap(s, q_out_dev, q_out_dtype, n_rows, nq, hd, q_out_row, q_out_head))),
                        SP_EINVAL, "the scales overlap the cache, queries, keys or values");
        }
        if (q_dev) {
            const bool in_place = q_dev == q_out_dev && q_out_dtype == dtype && q_row == q_out_row && q_head == q_out_head;
            const Span to = span_of(q_out_dev, q_out_dtype, n_rows, nq, hd, q_out_row, q_out_head);
            check_output(to);
            require((in_place || !may_overlap(to, q_dev, dtype, n_rows, nq, hd, q_row, q_head)) &&
                        !may_overlap(to, k_dev, dtype, n_rows, kv->n_kv_heads, hd, k_row, k_head) &&
                        !may_overlap(to, v_dev, dtype, n_rows, kv->n_kv_heads, hd, v_row, v_head),
                    SP_EINVAL, "the rotated queries overlap an input");
        }
        AppendArgs a{};
        a.rot = rot;
        a.q = q_dev; a.k = k_dev; a.v = v_dev;
        a.q_out = q_out_dev; a.kc = kv->k_dev; a.vc = kv->v_dev;
        a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
        a.qo_row = q_out_row; a.qo_head = q_out_head;
        a.ks = kv->k_scale_dev; a.vs = kv->v_scale_dev;
        a.pos = pos_dev; a.seq = seq_dev; a.at = at_dev; a.table = table_dev;
        a.rows = n_rows; a.nq = nq; a.nkv = kv->n_kv_heads; a.hd = hd; a.qo_dt = q_out_dtype; a.kv_dt = kv->dtype;
        a.n_seq = n_seq; a.max_pages = max_pages; a.n_pages = kv->n_pages; a.page_size = kv->page_size;
        a.page_stride = kv->page_stride; a.head_stride = kv->head_stride; a.row_stride = kv->row_stride;
        const bool wide = (!q_dev || (wide_ok(q_dev, dtype, q_row, q_head) && wide_ok(q_out_dev, q_out_dtype, q_out_row, q_out_head))) &&
                          wide_ok(k_dev, dtype, k_row, k_head) && wide_ok(v_dev, dtype, v_row, v_head) &&
                          wide_ok(kv->k_dev, kv->dtype, kv->page_stride, kv->head_stride) &&
                          wide_ok(kv->v_dev, kv->dtype, kv->row_stride, 0) &&
                          rot.rot % 16 == 0 && hd % 8 == 0;
        const int vec = wide ? 8 : 1;
        a.units = rot.rot / 2 / vec;
        a.tail = (hd - rot.rot) / vec;
        a.vecs = hd / vec;
        a.turned = (nq + a.nkv) * a.units;
        a.rest = (nq + a.nkv) * a.tail;
        a.per_row = a.turned + a.rest + a.nkv * a.vecs;
        a.by_row = Divisor(a.per_row); a.by_units = Divisor(a.units); a.by_tail = Divisor(a.tail); a.by_vecs = Divisor(a.vecs);
        a.by_half = Divisor(rot.rot / 2);
        if (kv->scale_block) {
            append_blocks(kv, a, dtype, wide, (hipStream_t)stream);
            return;
        }
        int threads;
        shape_of(a.per_row, n_rows, a.per_block, threads);
        for_input(dtype, wide, [&](auto *t, auto v) {
            hipLaunchKernelGGL((k_append<std::remove_pointer_t<decltype(t)>, decltype(v)::value>),
                               dim3((n_rows + a.per_block - 1) / a.per_block), dim3(threads),
                               (size_t)a.per_block * (sizeof(int64_t) + (rot.rot / 2) * sizeof(float2)), (hipStream_t)stream, a);
        });
        HIPCHK(hipGetLastError());
    });
}

int sp_op_paged_read(const sp_paged_kv *kv, int32_t dtype, int32_t n_rows, const int32_t *seq_dev, const int32_t *at_dev,
                     const int32_t *table_dev, int32_t n_seq, int32_t max_pages, void *k_out_dev, int64_t k_row, int64_t k_head,
                     void *v_out_dev, int64_t v_row, int64_t v_head, void *stream) {
    return guarded([&] {
        check_cache(kv);
        require(dtype == SP_DT_F32 || dtype == SP_DT_F16 || dtype == SP_DT_BF16, SP_EINVAL,
                "dtype must be SP_DT_F32, SP_DT_F16 or SP_DT_BF16");
        const int hd = kv->head_dim, nkv = kv->n_kv_heads;
        require(n_rows >= 0 && n_seq >= 1 && max_pages >= 1 && hd <= 1024 && 2 * (int64_t)nkv * hd < (1 << 16), SP_EINVAL,
                "n_rows must not be negative, n_seq and max_pages positive, head_dim at most 1024 and the values of a row below 2^16");
        if (n_rows == 0) return;
        require(seq_dev && at_dev && table_dev && k_out_dev && v_out_dev, SP_EINVAL, "NULL pointer");
        const Span k = span_of(k_out_dev, dtype, n_rows, nkv, hd, k_row, k_head), v = span_of(v_out_dev, dtype, n_rows, nkv, hd, v_row, v_head);
        check_output(k);
        check_output(v);
        require(!overlap(k, v), SP_EINVAL, "the outputs overlap each other");
        for (const Span &s : {k, v})
            require(!overlap(s, pool_of(kv, kv->k_dev)) && !overlap(s, pool_of(kv, kv->v_dev)) &&
                        (!kv->scale_block || (!overlap(s, scales_of(kv, kv->k_scale_dev)) && !overlap(s, scales_of(kv, kv->v_scale_dev)))),
                    SP_EINVAL, "an output overlaps the cache");
        ReadArgs a{};
        a.kc = kv->k_dev; a.vc = kv->v_dev; a.k_out = k_out_dev; a.v_out = v_out_dev;
        a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
        a.ks = kv->k_scale_dev; a.vs = kv->v_scale_dev;
        a.seq = seq_dev; a.at = at_dev; a.table = table_dev;
        a.rows = n_rows; a.nkv = nkv; a.kv_dt = kv->dtype;
        a.n_seq = n_seq; a.max_pages = max_pages; a.n_pages = kv->n_pages; a.page_size = kv->page_size;
        a.block = kv->scale_block; a.per_page = a.block ? kv->page_size / a.block : 0;
        a.page_stride = kv->page_stride; a.head_stride = kv->head_stride; a.row_stride = kv->row_stride;
        const bool wide = wide_ok(k_out_dev, dtype, k_row, k_head) && wide_ok(v_out_dev, dtype, v_row, v_head) &&
                          wide_ok(kv->k_dev, kv->dtype, kv->page_stride, kv->head_stride) &&
                          wide_ok(kv->v_dev, kv->dtype, kv->row_stride, 0) && hd % 8 == 0;
        a.vecs = hd / (wide ? 8 : 1);
        a.per_row = 2 * nkv * a.vecs;
        // (a vector a thread while blocks do not fill the chip eight times over, then READ_AHEAD: 131072 rows of 4 heads of 128 from int8
        // 101 us, by single vectors 136; 1777 rows 4.5 either way)
        const bool many = (double)n_rows * a.per_row > 8.0 * 256 * ROT_THREADS * READ_AHEAD;
        a.per_block = std::max(1, std::min({n_rows, ROT_THREADS, ROT_THREADS * (many ? READ_AHEAD : 1) / a.per_row}));
        a.by_row = Divisor(a.per_row); a.by_vecs = Divisor(a.vecs);
        launch_read(dtype, wide, a, (hipStream_t)stream);
    });
}

int sp_attn_plan_create(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_rows, int32_t max_seqs,
                        sp_attn_plan **out) {
    if (!out) { sp_call_error() = "out is NULL"; return SP_EINVAL; }
    *out = nullptr;
    sp_attn_plan *p = nullptr;
    const int rc = guarded([&] {
        check_shape(n_heads, n_kv_heads, head_dim, max_rows, max_seqs);
        p = new sp_attn_plan();
        p->NH = n_heads; p->NKV = n_kv_heads; p->HD = head_dim; p->max_rows = max_rows; p->max_seqs = max_seqs;
        lay_out(*p);
        HIPCHK(hipGetDevice(&p->device));
        p->dev = dev_alloc<int32_t>(p->words);
        HIPCHK(hipMemset(p->dev, 0, HEADER * sizeof(int32_t)));
        for (int i = 0; i < 2; ++i) {
            HIPCHK(hipHostMalloc((void **)&p->staging[i], p->words * sizeof(int32_t), hipHostMallocDefault));
            HIPCHK(hipEventCreateWithFlags(&p->copied[i], hipEventDisableTiming));
        }
    });
    if (rc != SP_OK) {
        if (p) { p->release(); delete p; }
        return rc;
    }
    *out = p;
    return SP_OK;
}

void sp_attn_plan_destroy(sp_attn_plan *p) {
    if (!p) return;
    p->release();
    delete p;
}

int sp_attn_plan_set(sp_attn_plan *p, int32_t n_seq, const int32_t *q_len, const int32_t *kv_len, int32_t n_groups,
                     const int32_t *group_size, const int32_t *group_shared, void *stream) {
    return guarded([&] {
        require(p != nullptr, SP_EINVAL, "plan is NULL");
        check_lengths(n_seq, q_len, kv_len, n_groups, group_size, group_shared, p->max_rows, p->max_seqs);
        const hipStream_t st = (hipStream_t)stream;
        require(!is_capturing(st), SP_ESTATE, "a plan is not set in a stream capture: captured calls read the tables of the last set");
        PlanTables t;
        tables_of(p->NH, p->NKV, p->HD, n_seq, q_len, kv_len, n_groups, group_size, group_shared, t);
        const int turn = p->turn;
        if (p->used[turn]) HIPCHK(hipEventSynchronize(p->copied[turn]));
        int32_t *img = p->staging[turn];
        std::memset(img, 0, HEADER * sizeof(int32_t));
        img[0] = (int32_t)t.items.size();
        img[1] = (int32_t)t.toks.size();
        img[2] = t.most_parts;
        p->set = false;                                  // until the tables are on their way
        // header and token records lie side by side: one copy; then the list and the items
        std::memcpy(img + p->tok_at, t.toks.data(), t.toks.size() * sizeof(TokenRecs));
        // (the list ends where the items begin: the kernel has no pointer of its own for it)
        const size_t list_at = p->item_at - t.list.size();
        std::reverse_copy(t.list.begin(), t.list.end(), img + list_at);
        std::memcpy(img + p->item_at, t.items.data(), t.items.size() * sizeof(Item));
        HIPCHK(hipMemcpyAsync(p->dev, img, (HEADER + t.toks.size() * (sizeof(TokenRecs) / 4)) * 4, hipMemcpyHostToDevice, st));
        if (!t.items.empty())
            HIPCHK(hipMemcpyAsync(p->dev + list_at, img + list_at, t.list.size() * 4 + t.items.size() * sizeof(Item),
                                  hipMemcpyHostToDevice, st));
        HIPCHK(hipEventRecord(p->copied[turn], st));
        p->used[turn] = true;
        p->turn = turn ^ 1;
        p->n_items = (int)t.items.size();
        p->most_parts = t.most_parts;
        p->n_tok = (int)t.toks.size();
        p->n_seq = n_seq;
        p->max_kv = t.max_kv;
        p->joined = t.joined;
        p->set = true;
    });
}

int sp_attn_plan_items(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t n_seq, const int32_t *q_len, const int32_t *kv_len,
                       int32_t n_groups, const int32_t *group_size, const int32_t *group_shared, int32_t capacity,
                       int32_t *items, int32_t *n_items, int32_t *token_recs, int64_t *n_records) {
    return guarded([&] {
        check_shape(n_heads, n_kv_heads, head_dim, 1, 1);
        require(n_items != nullptr, SP_EINVAL, "n_items is NULL");
        check_lengths(n_seq, q_len, kv_len, n_groups, group_size, group_shared, (1 << 27) / n_heads, 65535);
        PlanTables t;
        tables_of(n_heads, n_kv_heads, head_dim, n_seq, q_len, kv_len, n_groups, group_size, group_shared, t);
        *n_items = (int32_t)t.items.size();
        if (n_records) *n_records = t.records;
        if (items) {
            require(capacity >= *n_items, SP_ECAPACITY, "capacity is smaller than the number of items");
            if (!t.items.empty()) std::memcpy(items, t.items.data(), t.items.size() * sizeof(Item));
        }
        if (token_recs && !t.toks.empty()) std::memcpy(token_recs, t.toks.data(), t.toks.size() * sizeof(TokenRecs));
    });
}

size_t sp_attn_plan_workspace(const sp_attn_plan *p) {
    if (!p) return 0;
    return (size_t)records_bound(p->max_rows, p->NH) * ((size_t)p->HD * sizeof(float) + sizeof(f32x4));
}

int sp_op_paged_attention(const sp_attn_plan *p, const sp_paged_kv *kv, int32_t dtype, int32_t n_rows, const void *q_dev, int64_t q_row,
                          int64_t q_head, const int32_t *table_dev, int32_t n_seq, int32_t max_pages, float scale, void *out_dev,
                          int64_t out_row, int64_t out_head, float *lse_dev, void *workspace_dev, void *stream) {
    return guarded([&] {
        require(p != nullptr, SP_EINVAL, "plan is NULL");
        check_cache(kv);
        require(dtype == SP_DT_F16 || dtype == SP_DT_BF16, SP_EINVAL, "dtype must be SP_DT_F16 or SP_DT_BF16");
        require(kv->dtype == dtype || bytes_of(kv->dtype) == 1, SP_EINVAL, "the cache's dtype must be the queries', SP_DT_E4M3 or SP_DT_I8");
        require(kv->n_kv_heads == p->NKV && kv->head_dim == p->HD, SP_EINVAL, "the cache's heads are not the plan's");
        require(scale > 0.f && std::isfinite(scale), SP_EINVAL, "scale must be positive");
        require(p->set, SP_ESTATE, "the plan has no lengths: call sp_attn_plan_set first");
        require(n_rows >= p->n_tok, SP_EINVAL, "the queries have fewer rows than the plan");
        require(n_seq >= p->n_seq && max_pages >= 1, SP_EINVAL, "the page table has fewer sequences than the plan");
        require((int64_t)max_pages * kv->page_size >= p->max_kv, SP_EINVAL, "the page table is too short for the plan's lengths");
        const int64_t hd = kv->head_dim;
        require(kv->page_stride % hd == 0 && kv->head_stride % hd == 0 && kv->row_stride % hd == 0, SP_EINVAL,
                "the cache's strides must be multiples of head_dim");
        constexpr int64_t MOST = (int64_t)1 << 32;
        require(kv->page_stride / hd < MOST && kv->head_stride / hd < MOST && kv->row_stride / hd < MOST &&
                    (double)(kv->n_pages - 1) * (kv->page_stride / hd) + (double)(kv->n_kv_heads - 1) * (kv->head_stride / hd) +
                            (double)(kv->page_size - 1) * (kv->row_stride / hd) < (double)MOST,
                SP_EINVAL, "the pool must be below 2^32 rows");
        int dev = 0;
        HIPCHK(hipGetDevice(&dev));
        require(dev == p->device, SP_EINVAL, "the plan belongs to another device than the current one");
        const hipStream_t st = (hipStream_t)stream;
        const bool capturing = is_capturing(st);
        if (capturing ? n_rows == 0 : p->n_tok == 0) return;           // (a captured call serves later sets too)
        require(q_dev && out_dev && table_dev && workspace_dev, SP_EINVAL, "NULL pointer");
        require(aligned(q_dev, 16) && q_row % 8 == 0 && q_head % 8 == 0, SP_EINVAL, "queries must be aligned to 16 bytes");
        {
            const Span to = span_of(out_dev, dtype, n_rows, p->NH, p->HD, out_row, out_head);
            check_output(to);
            require(!may_overlap(to, q_dev, dtype, n_rows, p->NH, p->HD, q_row, q_head), SP_EINVAL, "the output overlaps the queries");
            require(!overlap(to, pool_of(kv, kv->k_dev)) && !overlap(to, pool_of(kv, kv->v_dev)) &&
                        (!kv->scale_block || (!overlap(to, scales_of(kv, kv->k_scale_dev)) && !overlap(to, scales_of(kv, kv->v_scale_dev)))),
                    SP_EINVAL, "the output overlaps the cache");
        }
        require(aligned(out_dev, 8) && out_row % 4 == 0 && out_head % 4 == 0, SP_EINVAL, "outputs must be aligned to 8 bytes");
        require(aligned(kv->k_dev, 16) && aligned(kv->v_dev, 16) && kv->head_dim * bytes_of(kv->dtype) % 16 == 0,
                SP_EINVAL, "the cache's pages must be aligned to 16 bytes");
        require(aligned(workspace_dev, 16), SP_EINVAL, "the workspace must be aligned to 16 bytes");
        BlockArgs a{};
        a.q = q_dev; a.out = out_dev; a.lse = lse_dev;
        a.q_row = q_row; a.q_head = q_head; a.out_row = out_row; a.out_head = out_head;
        a.k = (const uint8_t *)kv->k_dev; a.v = (const uint8_t *)kv->v_dev; a.ks = kv->k_scale_dev; a.vs = kv->v_scale_dev;
        a.rows = n_rows; a.n_seq = n_seq;
        a.table = table_dev; a.max_pages = max_pages; a.n_pages = kv->n_pages; a.page_size = kv->page_size;
        a.page_rows = (uint32_t)(kv->page_stride / hd); a.head_rows = (uint32_t)(kv->head_stride / hd);
        a.slot_rows = (uint32_t)(kv->row_stride / hd);
        a.NH = p->NH; a.G = p->NH / p->NKV;
        a.by_g = Divisor(a.G);
        a.by_page = PageDivisor(kv->page_size);
        a.scale = scale * LOG2E;
        const size_t recs = (size_t)records_bound(p->max_rows, p->NH);
        a.ml = (f32x4 *)workspace_dev;
        a.po = (float *)(a.ml + recs);
        const bool kv8 = kv->dtype == SP_DT_E4M3;
        a.items = (const Item *)(p->dev + p->item_at);
        a.n_items = capturing ? p->dev : nullptr;
        const int grid = capturing ? CAPTURED_GRID : p->n_items;
        if (grid && kv->scale_block) {
            a.per_page = kv->page_size / kv->scale_block;
            a.by_block = PageDivisor(kv->scale_block);
            launch_block_items(dtype, kv->dtype, p->HD, a, grid, st);
        } else if (grid) {
            if (dtype == SP_DT_F16) launch_typed<f16>(kv8, p->HD, a, grid, st);
            else launch_typed<bf16>(kv8, p->HD, a, grid, st);
            HIPCHK(hipGetLastError());
        }
        if (p->joined || capturing) {
            const JoinArgs j{(const TokenRecs *)(p->dev + p->tok_at), p->dev + 1, a.po, a.ml, out_dev, lse_dev, out_row, out_head,
                             n_rows, p->NH, a.G};
            const int tokens = capturing ? std::min(n_rows, p->max_rows) : p->n_tok;
            if (dtype == SP_DT_F16) {
                if (p->HD == 128) launch_join<f16, 128>(j, tokens, capturing, p->most_parts, st);
                else launch_join<f16, 64>(j, tokens, capturing, p->most_parts, st);
            } else {
                if (p->HD == 128) launch_join<bf16, 128>(j, tokens, capturing, p->most_parts, st);
                else launch_join<bf16, 64>(j, tokens, capturing, p->most_parts, st);
            }
            HIPCHK(hipGetLastError());
        }
    });
}

}  // extern "C"
