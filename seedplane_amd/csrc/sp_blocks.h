// A paged cache of 8-bit codes with a scale for each block of positions and K/V head: appending to it, and reading positions back.
//
// A block is `block` positions of a page (a multiple of 16 that divides the page); a value is code * scale of its block and head.  Codes
// are int8 (whole numbers up to 127) or e4m3 (up to 448).  A call finds the rows that it brings to a block, whatever their order, and
// takes scale = max |x| / largest code over them.  A block whose first position is among them begins anew; any other keeps what it
// holds, its scale only grows, and where it does the codes that the call does not write are rounded once more, by old / new scale.
//
// What bounds it: a step is a chain of dependent accesses (row, table entry beside the search, values, scale, codes): 16 rows of 12 / 2 / 2
// heads of 128 take 6.1 us, their reading back 3.6, where an empty launch takes 2.3; a prompt of 1777 rows of 28 / 4 / 4 heads, 26 MB of
// values, takes 15.2 us, 13.3 of them without queries: the blocks' chains (the search of all rows, angles, which the workgroups of a block's single
// heads form each for itself, largest magnitudes, codes, with barriers between), beside which the queries' rows run, one a workgroup (rotated alone
// they take 5.8); its reading back 4.5 (14 MB).
//
// A workgroup takes a chunk of rows of the call (a row whose block an earlier row has is left to that row's workgroup), keys or
// values, and some heads: it looks up its block's rows among all of the call's, lists the slots that have one, takes the largest magnitude per
// head, then the codes (a step of 1024 sequences on blocks of 128: 24 us, by all slots 88; 16384 rows of prompts, whose slots all have one, 2 us
// more than without the list).
// Values are read twice unless a thread has but one item of them: a block of 64 positions of one head alone is 8192 values.  Long
// calls (FIND) look up the rows of all a chunk's blocks at once.  They are bound by the blocks' chains of barriers (16384 rows of 28 / 4 / 4
// heads 79 us, 38 of them without queries, where the bytes take 56 and 10), so their registers are held to those of 6 waves: with 5
// waves the blocks gain less than the queries' rows behind them lose (83).  Keys and values have loops of their own: one for both
// had more uniform values than scalar registers hold (16 rows 7.0 us instead of 6.0, 16384 89 instead of 78).
// Rows in order of time put more rows between a chunk's blocks than MOST_FOUND, and every run of a block's rows, here single rows, searches all
// of them: 8192 rows of 4 sequences 74 us on blocks of 16 and 99 of 32 (by sequence 37, 35), of 64 sequences 200, 587, of 128 1740 (73).
#pragma once
#include "sp_paged.h"

namespace paged {

constexpr int READ_AHEAD = 4;                                          // vectors of a thread in flight, reading back
constexpr int MOST_BLOCK = 128;                                        // positions of a block at most
constexpr int BLOCK_HEADS = 64;                                        // heads of a workgroup at most
constexpr int SEARCHED = 4;                                            // rows that a thread looks at at once
constexpr int MOST_CHUNK = 256, MOST_FOUND = 512;                      // rows of a chunk; of the call that may be of its blocks
constexpr float MOST_SCALE = 0x1p60f;                                  // (scales within 2^-60 .. 2^60: attention takes their products)

struct BlockAppendArgs : AppendArgs {                                  // ks, vs are not used; units, tail, vecs are a head's
    float *kscale, *vscale;                                            // [n_pages][nkv][per_page]
    int block, per_page;
    PageDivisor by_block, by_page;
    int chunk, chunks, splits, heads;                                  // rows of a workgroup, their number; workgroups over heads, heads of each
    PageDivisor by_key, by_value;                                      // vectors of a slot: keys (pairs of them where rotated), values
    bool find;                                                         // rows of a chunk's blocks are looked up at once
};
struct ReadArgs {
    const void *kc, *vc;
    void *k_out, *v_out;
    int64_t k_row, k_head, v_row, v_head;
    const float *ks, *vs;                                              // scales per head, per block, or NULL
    const int *seq, *at, *table;
    int rows, nkv, kv_dt, per_block, vecs, per_row;
    int n_seq, max_pages, n_pages, page_size, block, per_page;         // block 0: scales per head
    int64_t page_stride, head_stride, row_stride;
    Divisor by_row, by_vecs;
};

__attribute__((visibility("hidden"))) void launch_block_items(int dtype, int kv_dtype, int HD, const BlockArgs &a, int grid, hipStream_t st);
__attribute__((visibility("hidden"))) void launch_block_append(int dtype, bool wide, const BlockAppendArgs &a, int query_blocks, size_t lds, hipStream_t st);
__attribute__((visibility("hidden"))) void launch_read(int dtype, bool wide, const ReadArgs &a, hipStream_t st);

// ------------------------------------------------------------------------------------------------ codes
// N fp32 values (already over their scale) as codes of kind I8 or e4m3, and codes as fp32.
template <bool I8, int N>
__device__ __forceinline__ void store_codes(uint8_t *p, const float *v) {
    if constexpr (!I8) {
        store_values<N>(p, 0, SP_DT_E4M3, v);
    } else {
        int c[N];
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = (int)rintf(fminf(fmaxf(v[i], -127.f), 127.f));
        if constexpr (N == 1) p[0] = (uint8_t)c[0];
        else {
            u32x2 w;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[i] = (c[4 * i] & 0xff) | (c[4 * i + 1] & 0xff) << 8 | (c[4 * i + 2] & 0xff) << 16 | (uint32_t)c[4 * i + 3] << 24;
            *(u32x2 *)p = w;
        }
    }
}
__device__ __forceinline__ float e4m3_value(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8(code, 0); }
template <bool I8, int N>
__device__ __forceinline__ void load_codes(const uint8_t *p, float *v) {
    if constexpr (N == 1) {
        v[0] = I8 ? (float)(int8_t)p[0] : e4m3_value(p[0]);
    } else {
        const u32x2 w = *(const u32x2 *)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = w[i / 4] >> (8 * (i % 4));
            v[i] = I8 ? (float)(int8_t)c : e4m3_value(c & 0xff);
        }
    }
}

// ------------------------------------------------------------------------------------------------ append
template <bool FIND>
struct BlockShared {
    int slot[MOST_BLOCK];                                              // the row that brings each position of the block (the last one), -1
    uint32_t most[BLOCK_HEADS];                                        // bits of the largest magnitude
    float scale[BLOCK_HEADS], inverse[BLOCK_HEADS], keep[BLOCK_HEADS]; // new scale, 1 / scale; old / new (1: codes stay)
    int earlier, moved;                                                // rows before the workgroup's own; whether codes that stay move
    int here, list[MOST_BLOCK];                                        // slots that have a row
    int found, row[FIND ? MOST_FOUND : 1], seq[FIND ? MOST_FOUND : 1], at[FIND ? MOST_FOUND : 1];       // the call's rows that may be of a block of the chunk (FIND)
};

// The largest magnitude of N values, as bits: a NaN is above all (int8), or left out (e4m3, which holds it as itself).
template <bool I8, int N>
__device__ __forceinline__ uint32_t magnitude(const float *v, uint32_t most) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
        most = I8 || b <= 0x7f800000u ? max(most, b) : most;
    }
    return most;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}

// Whether row i is of block b of sequence s.
__device__ __forceinline__ bool of_block(const BlockAppendArgs &a, int seq, int at, int s, int b) {
    return seq == s && at >= 0 && at < (1 << 30) && at / a.by_block == b;
}

// The block of row r, which does not follow a row of the same block.
template <class T, int VEC, bool I8, bool FIND, bool KEYS>
__device__ __forceinline__ void append_block(const BlockAppendArgs &a, int r, int head0, BlockShared<FIND> &sh, float2 *cs) {
    const int tid = threadIdx.x, s = a.seq[r], p = a.at[r];
    if (s < 0 || s >= a.n_seq || p < 0 || p >= (1 << 30)) return;
    const int b = p / a.by_block, page = p / a.by_page;
    if (page >= a.max_pages) return;
    const int e = a.table[(int64_t)s * a.max_pages + page];            // (awaited after the search)
    __syncthreads();                                                   // the block before has been written
    for (int i = tid; i < a.block; i += ROT_THREADS) sh.slot[i] = -1;
    if (tid < a.heads) sh.most[tid] = 0;
    if (tid == 0) { sh.earlier = 0; sh.moved = 0; sh.here = 0; }
    __syncthreads();
    auto look = [&](int i, int seq, int at) {
        if (!of_block(a, seq, at, s, b)) return;
        if (i < r) sh.earlier = 1;
        else atomicMax(&sh.slot[at - b * a.block], i);
    };
    if (FIND && sh.found <= MOST_FOUND) {
        for (int i = tid; i < sh.found; i += ROT_THREADS) look(sh.row[i], sh.seq[i], sh.at[i]);
    } else {
        for (int i0 = tid; i0 < a.rows; i0 += ROT_THREADS * SEARCHED) {
            int seq[SEARCHED], at[SEARCHED];
#pragma unroll
            for (int k = 0; k < SEARCHED; ++k) {
                const int i = min(i0 + k * ROT_THREADS, a.rows - 1);
                seq[k] = a.seq[i];
                at[k] = a.at[i];
            }
#pragma unroll
            for (int k = 0; k < SEARCHED; ++k) look(min(i0 + k * ROT_THREADS, a.rows - 1), seq[k], at[k]);
        }
    }
    __syncthreads();
    if (sh.earlier || e < 0 || e >= a.n_pages) return;
    const int heads = min(a.heads, a.nkv - head0), half = a.rot.rot >> 1;
    const int64_t block_of_page = b - (int64_t)page * a.per_page;
    float *const scale = (KEYS ? a.kscale : a.vscale) + ((int64_t)e * a.nkv + head0) * a.per_page + block_of_page;      // of head h: at h * per_page
    const float old = tid < heads ? scale[(int64_t)tid * a.per_page] : 0.f;
    const bool begun = sh.slot[0] >= 0;
    if (tid < MOST_BLOCK) {                                            // (whole waves)
        const bool here = tid < a.block && sh.slot[tid] >= 0;
        const uint64_t who = __ballot(here);
        int first = 0;
        if ((tid & 63) == 0) first = atomicAdd(&sh.here, __popcll(who));
        first = __builtin_amdgcn_readfirstlane(first);
        if (here) sh.list[first + __popcll(who & (((uint64_t)1 << (tid & 63)) - 1))] = tid;
    }
    __syncthreads();
    // item: head h, slot i that has a row, and vector u of it (keys: a rotated pair of vectors, or one of the rest)
    const int here = __builtin_amdgcn_readfirstlane(sh.here);          // (at least row r's)
    Divisor by_here;
    by_here.d = here;
    by_here.inverse = 0xffffffffu / here + 1;                          // (rounded up, as the constructor's; not used for 1)
    const PageDivisor by = KEYS ? a.by_key : a.by_value;
    const int per = KEYS ? a.units + a.tail : a.vecs, total = here * per, items = heads * total;
    uint8_t *const pool = (uint8_t *)(KEYS ? a.kc : a.vc) + e * a.page_stride + head0 * a.head_stride +
                          (int64_t)(p - page * a.page_size - (p - b * a.block)) * a.row_stride;
    struct Item { int h, i, row, turn, at1, at2; bool two; };
    auto item_of = [&](int k) -> Item {
        Item x;
        const int q = k / by, u = k - q * per;
        x.h = q / by_here;
        x.i = sh.list[q - x.h * here];
        x.row = sh.slot[x.i];
        x.two = KEYS && u < a.units;
        x.turn = x.i * half + u * VEC;
        if (x.two) unit_offsets<VEC>(a.rot, u, x.at1, x.at2);
        else x.at1 = x.at2 = KEYS ? a.rot.rot + (u - a.units) * VEC : u * VEC;
        return x;
    };
    typedef T Vector __attribute__((ext_vector_type(VEC)));
    Vector raw1, raw2;
    float v1[VEC], v2[VEC];
    auto fetch = [&](const Item &x) {
        const int64_t row = x.row;
        const T *src = KEYS ? (const T *)a.k + row * a.k_row + (int64_t)(head0 + x.h) * a.k_head
                            : (const T *)a.v + row * a.v_row + (int64_t)(head0 + x.h) * a.v_head;
        raw1 = *(const Vector *)(src + x.at1);
        if constexpr (KEYS) raw2 = *(const Vector *)(src + x.at2);
    };
    auto values = [&](const Item &x) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            v1[i] = (float)raw1[i];
            if constexpr (KEYS) v2[i] = (float)raw2[i];
        }
        if constexpr (KEYS)
            if (x.two) turn_unit<VEC>(a.rot, cs + x.turn, v1, v2);
    };
    if (KEYS && half) {
        for (int k = tid; k < here * half; k += ROT_THREADS) {
            const int o = k / a.by_half, j = k - o * half, i = sh.list[o];
            cs[i * half + j] = turn_of(a.rot, a.pos[sh.slot[i]], j);
        }
        __syncthreads();
    }
    for (int k0 = 0; k0 < items; k0 += ROT_THREADS) {
        const Item x = item_of(min(k0 + tid, items - 1));              // (past the last: the last again, its largest does not change)
        fetch(x);
        values(x);
        uint32_t most = magnitude<I8, VEC>(v1, 0);
        if constexpr (KEYS) most = magnitude<I8, VEC>(v2, most);
        if (total % 64 == 0) {                                         // a wave's items are of one head
            most = wave_umax(most);
            if ((tid & 63) == 0 && most) atomicMax(&sh.most[x.h], most);
        } else if (most) {
            atomicMax(&sh.most[x.h], most);
        }
    }
    __syncthreads();
    if (tid < heads) {
        const float most = __uint_as_float(sh.most[tid]);
        const float made = most > MOST_SCALE * (I8 ? 127.f : 448.f) ? MOST_SCALE : most / (I8 ? 127.f : 448.f);
        // (comparisons that leave a NaN where it is: of int8's new values, or held since the block began)
        float grown = made < LEAST_SCALE ? LEAST_SCALE : made;
        if (!begun && !(old <= grown)) grown = grown != grown ? grown : old;
        sh.scale[tid] = grown;
        sh.inverse[tid] = 1.f / grown;
        const float keep = begun || grown == old ? 1.f : old / grown;
        sh.keep[tid] = keep;
        if (keep != 1.f) sh.moved = 1;
        scale[(int64_t)tid * a.per_page] = grown;
    }
    __syncthreads();
    // Quotients by the scale: the product with its reciprocal alone, rounded twice, puts values half way between two codes to either side; what is
    // left of the value behind it (one fused step, exact), taken in once more, gives the rounded quotient.  (Bounded in between, so that infinities
    // leave infinity, not NaN.  It costs 16384 rows 1.7 us of 79, a division of the compiler's 2.8.)
    auto scaled = [&](uint8_t *to, int h, int at1, int at2, bool two) {
        const float s = sh.scale[h], inverse = sh.inverse[h];
        auto quotient = [&](float v) {
            const float q = fminf(fmaxf(v * inverse, -512.f), 512.f);
            return __builtin_fmaf(__builtin_fmaf(-q, s, v), inverse, q);
        };
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            v1[i] = quotient(v1[i]);
            if constexpr (KEYS) v2[i] = quotient(v2[i]);
        }
        store_codes<I8, VEC>(to + at1, v1);
        if constexpr (KEYS)
            if (two) store_codes<I8, VEC>(to + at2, v2);
    };
    for (int k = tid; k < items; k += ROT_THREADS) {
        const Item x = item_of(k);
        if (items > ROT_THREADS) fetch(x);                             // (else its values are still here)
        if (FIND || items > ROT_THREADS) values(x);                    // (FIND: turned again, for the registers)
        scaled(pool + x.h * a.head_stride + x.i * a.row_stride, x.h, x.at1, x.at2, x.two);
    }
    // what the call does not write, of heads whose scale has grown (vectors of a whole head, whatever turns)
    if (sh.moved) {
        const int vecs = a.vecs, all = heads * a.block * vecs;
        for (int k = tid; k < all; k += ROT_THREADS) {
            const int q = k / a.by_value, h = q / a.by_block, i = q - h * a.block;
            const float f = sh.keep[h];
            if (sh.slot[i] >= 0 || f == 1.f) continue;
            uint8_t *const to = pool + h * a.head_stride + i * a.row_stride + (k - q * vecs) * VEC;
            float v[VEC];
            load_codes<I8, VEC>(to, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] *= f;
            store_codes<I8, VEC>(to, v);
        }
    }
}

// Rows of the call that are of the sequences and blocks between the least and largest of the chunk's, to sh.found.  (Every wave looks at the
// chunk's rows itself.)
__device__ __forceinline__ void find_rows(const BlockAppendArgs &a, int first, int last, BlockShared<true> &sh) {
    const int tid = threadIdx.x, lane = tid & 63;
    int s0 = 0x7fffffff, s1 = -1, p0 = 0x7fffffff, p1 = -1;
    for (int r = first + lane; r < last; r += 64) {
        const int s = a.seq[r], p = a.at[r];
        if (s < 0 || s >= a.n_seq || p < 0 || p >= (1 << 30)) continue;
        s0 = min(s0, s); s1 = max(s1, s);
        p0 = min(p0, p); p1 = max(p1, p);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        s0 = min(s0, __shfl_xor(s0, o)); s1 = max(s1, __shfl_xor(s1, o));
        p0 = min(p0, __shfl_xor(p0, o)); p1 = max(p1, __shfl_xor(p1, o));
    }
    if (tid == 0) sh.found = 0;
    __syncthreads();
    if (s1 < 0) return;
    p0 = p0 / a.by_block * a.block;
    p1 = p1 / a.by_block * a.block + (a.block - 1);
    auto look = [&](int i, int seq, int at) {
        if (seq < s0 || seq > s1 || at < p0 || at > p1) return;
        const int k = atomicAdd(&sh.found, 1);
        if (k < MOST_FOUND) { sh.row[k] = i; sh.seq[k] = seq; sh.at[k] = at; }
    };
    typedef int Four __attribute__((ext_vector_type(4), aligned(4)));
    const int whole = a.rows / 4 * 4;
    constexpr int STEP = ROT_THREADS * 4;
    for (int i0 = tid * 4; i0 < whole; i0 += STEP * 4) {
        Four seq[4], at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = min(i0 + k * STEP, whole - 4);
            seq[k] = *(const Four *)(a.seq + i);
            at[k] = *(const Four *)(a.at + i);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i0 + k * STEP >= whole) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) look(i0 + k * STEP + j, seq[k][j], at[k][j]);
        }
    }
    if (whole + tid < a.rows) look(whole + tid, a.seq[whole + tid], a.at[whole + tid]);
    __syncthreads();
}

template <class T, int VEC, bool I8, bool FIND, bool KEYS>
__device__ __forceinline__ void append_chunk(const BlockAppendArgs &a, int chunk, int split, BlockShared<FIND> &sh, float2 *cs) {
    const int first = chunk * a.chunk, last = min(a.rows, first + a.chunk);
    if constexpr (FIND) find_rows(a, first, last, sh);
    // the chunk's rows that begin a run of a block's rows (every wave finds the same)
    for (int r0 = first; r0 < last; r0 += 64) {
        const int r = r0 + (int)(threadIdx.x & 63);
        bool begins = r < last;
        if (begins && r > 0) {
            const int s = a.seq[r], p = a.at[r];
            begins = p < 0 || p >= (1 << 30) || !of_block(a, a.seq[r - 1], a.at[r - 1], s, p / a.by_block);
        }
        for (uint64_t runs = __ballot(begins); runs; runs &= runs - 1)
            append_block<T, VEC, I8, FIND, KEYS>(a, r0 + __builtin_ctzll(runs), split * a.heads, sh, cs);
    }
}

// Blocks: chunks x (keys, values) x splits of the heads, then the queries' rows.
template <class T, int VEC, bool I8, bool FIND>
__global__ void __launch_bounds__(ROT_THREADS, FIND ? 6 : 1) k_append_blocks(BlockAppendArgs a) {
    extern __shared__ __align__(16) unsigned char block_smem[];
    __shared__ BlockShared<FIND> sh;
    const int parts = 2 * a.splits, n = a.chunks * parts;
    const int block = blockIdx.x;
    if (block >= n) {
        append_rows<T, VEC>(a, block - n, block_smem);
        return;
    }
    const int chunk = block / parts, part = block - chunk * parts;
    if (part < a.splits) append_chunk<T, VEC, I8, FIND, true>(a, chunk, part, sh, (float2 *)block_smem);
    else append_chunk<T, VEC, I8, FIND, false>(a, chunk, part - a.splits, sh, (float2 *)block_smem);
}

// ------------------------------------------------------------------------------------------------ read
// Rows of a cache as dense values: row r's keys and values at position at[r] of sequence seq[r]; zeros where it has no place.
template <class C, int N>
__device__ __forceinline__ void load_cached(const void *p, int64_t at, int kv_dt, float *v) {
    if (kv_dt == SP_DT_I8) load_codes<true, N>((const uint8_t *)p + at, v);
    else if (kv_dt == SP_DT_E4M3) load_codes<false, N>((const uint8_t *)p + at, v);
    else if (kv_dt == SP_DT_F16) load_values<f16, N>((const f16 *)p + at, v);
    else load_values<bf16, N>((const bf16 *)p + at, v);
}
template <class T, int VEC>
__global__ void __launch_bounds__(ROT_THREADS) k_paged_read(ReadArgs a) {
    __shared__ int64_t from[ROT_THREADS];                              // [rows of the block]: element offset in the pools, or -1
    __shared__ int64_t scale_at[ROT_THREADS];
    const int row0 = blockIdx.x * a.per_block, n = min(a.per_block, a.rows - row0), total = n * a.per_row;
    for (int k = threadIdx.x; k < n; k += blockDim.x) {
        const int s = a.seq[row0 + k], p = a.at[row0 + k];
        int64_t at = -1, sc = 0;
        if (s >= 0 && s < a.n_seq && p >= 0 && p / a.page_size < a.max_pages) {
            const int e = a.table[(int64_t)s * a.max_pages + p / a.page_size];
            if (e >= 0 && e < a.n_pages) {
                at = e * a.page_stride + (p % a.page_size) * a.row_stride;
                if (a.block) sc = (int64_t)e * a.nkv * a.per_page + p % a.page_size / a.block;
            }
        }
        from[k] = at;
        scale_at[k] = sc;
    }
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < total; i0 += ROT_THREADS * READ_AHEAD) {
        float v[READ_AHEAD][VEC], f[READ_AHEAD];
        int64_t to[READ_AHEAD];
        bool keys[READ_AHEAD];
#pragma unroll
        for (int u = 0; u < READ_AHEAD; ++u) {
            const int i = i0 + u * ROT_THREADS;
            if (i >= total) break;
            const int r = i / a.by_row, k = i - r * a.per_row, w = k / a.by_vecs, at = (k - w * a.vecs) * VEC;
            keys[u] = w < a.nkv;
            const int h = keys[u] ? w : w - a.nkv;
            const int64_t row = row0 + r;
            to[u] = (keys[u] ? row * a.k_row + h * a.k_head : row * a.v_row + h * a.v_head) + at;
            f[u] = 1.f;
            if (from[r] < 0) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[u][j] = 0.f;
            } else {
                load_cached<T, VEC>(keys[u] ? a.kc : a.vc, from[r] + h * a.head_stride + at, a.kv_dt, v[u]);
                const float *scales = keys[u] ? a.ks : a.vs;
                if (scales) f[u] = scales[scale_at[r] + (a.block ? (int64_t)h * a.per_page : h)];
            }
        }
#pragma unroll
        for (int u = 0; u < READ_AHEAD; ++u) {
            if (i0 + u * ROT_THREADS >= total) break;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[u][j] *= f[u];
            store_values<VEC>(keys[u] ? a.k_out : a.v_out, to[u], dtype_of<T>(), v[u]);
        }
    }
}

}  // namespace paged
