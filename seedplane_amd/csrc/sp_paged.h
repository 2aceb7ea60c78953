// Attention over a paged K/V cache for batches whose sequences share a prefix.
//
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions j that query i sees, the keys cut into parts (items of
// the host's plan, sp_paged_plan.h); a part leaves (m, l, o) and parts are joined by weights exp(m - M), so a prefix shared by
// many sequences is read once for all of their queries and the rest of each sequence apart.
//
// One item: rows (queries x heads of one K/V head) against a range of positions.  Scores are computed transposed, S^T = K Q^T,
// on 32x32x16 MFMAs: the accumulator then has a query per lane and keys in its registers, so maxima and sums run in the
// lane's own registers (one exchange between the wave's halves per tile), and exp(S^T) is, without moving, the B operand of
// O^T = V^T P^T, if V^T's columns are taken in the same key order: the LDS transpose reads give V^T from rows of V.
//
// Keys and values go from the pages to LDS by direct copies (16 bytes a lane; no registers), two tiles deep.  A row's 16-byte
// pieces are stored permuted by its index (the copy fetches them so), which keeps both kinds of reads off each other's banks.
// Waves stand side by side over rows (WM) and over keys (4 / WM): 1 x 4 for the few rows of a decode step, 4 x 1 for
// many.  Scores, maxima, sums and outputs are fp32, in the records of parts too; P is rounded to the queries' type, which its
// product with V takes on the matrix cores (half a step of each weight).
//
// What bounds it.  Few rows: memory; 64 sequences x 4096 positions, 28 / 4 heads of 128 in bf16, 537 MB: 102 us, 5.3 TB/s, the rate of
// a large copy (e4m3 50 us).  Many rows: the products and the other vector instructions, of which little runs at once; 128 tiles of
// 126 rows x 4 heads on the same 4096 positions: 166 us, 813 TFLOP/s, 57 % of a large library product, the matrix cores busy 49 % and
// the vector unit's issue 50 % of the waves' time, both at once 12 %.  Part of that is the order within a wave: the first 32 keys'
// exponentials and the tile's maxima have no product beside them, only the second 32 keys' exponentials do.  (Per score one
// exponential, scaling, sum, comparison and half a rounding against a product's 4 HD operations; LDS is used 24 % of the time, without
// conflicts.  Tried, when this batch took 178 us: four tiles deep with 32 keys 243, sums of rounded weights by dot products 181,
// priorities 172 to 182, blocks of 8 waves whose halves take turns multiplying and weighing 188.)
//
// Caches with a scale per block of positions and head (sp_blocks.h) run the same items: the scales of the table's positions come to LDS by
// copies of 4 bytes in front of the tiles', each wave makes its own positions' terms of them behind the first scores, and a block's largest
// score is scaled instead of every score.  64 sequences x 4096 positions, 28 / 4 heads of 128: int8 52.7 us, e4m3 51.2 (268 MB and 8 of
// scales, 5.2 and 5.4 TB/s).  int8 takes five (fp16) or six (bf16) instructions for four codes where e4m3 takes two: a wave that shares a
// tile's rows with others brings its part of the tile to 16 bits for all of them, codes going through registers a tile ahead and
// being written behind products (6 prompts of 12 / 2 heads of 128 70 us; before other steps 73, each wave for itself 80, a barrier more instead of the registers 77;
// e4m3 each for itself 63, once for all 69; the same positions in 16 bits 55).  Tried for waves of their own: keys' codes left 1152 above their
// values as operands, scores begun at what that adds: 8 sequences of 20000 to 40000 positions 65.0 -> 64.2 us then, not kept.
#pragma once
#include "sp_paged_plan.h"
#include "sp_rotate.h"

namespace paged {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// key / d for keys below 2^30: m = ceil(2^(30 + l) / d) with 2^l >= d exceeds 2^(30 + l) / d by less than 2^l / d, so
// key m / 2^(30 + l) exceeds key / d by less than 1 / d; m is at most 2^31 as 2^(l - 1) < d.  (Straight code: a launch fetches its
// instructions anew, and a branch over a division cost a lone token's call over 733 positions 0.17 us of 8.95.)
struct PageDivisor {
    uint32_t m;
    int l;
    PageDivisor() = default;
    explicit PageDivisor(uint32_t d) : l(0) {
        while (((uint64_t)1 << l) < d) ++l;
        m = (uint32_t)((((uint64_t)1 << (30 + l)) + d - 1) / d);
    }
};
__device__ __forceinline__ int operator/(int key, PageDivisor d) { return (int)(__umulhi((uint32_t)key << 2, d.m) >> d.l); }

struct AttnArgs {
    const void *q;
    void *out;
    float *lse;                       // [rows][NH] or NULL
    int64_t q_row, q_head, out_row, out_head;
    const uint8_t *k, *v;
    const float *ks, *vs;             // e4m3: scale per K/V head
    const int *table;                 // [n_seq][max_pages]
    int rows, n_seq, max_pages, n_pages, page_size;      // rows of q and out, of the table; its width; the pool
    uint32_t page_rows, head_rows, slot_rows;     // strides of the pool in rows of head_dim values
    int NH, G;
    Divisor by_g;
    PageDivisor by_page;
    float scale;                      // of the scores, times log2(e)
    const Item *items;
    const int *n_items;               // NULL: one block per item
    // Records: [rows][HD] unnormalised outputs, and [rows] (m in log2 units, l, a factor of the outputs).  Sums stay in fp32: as
    // fp16 shares of a row's largest one (half the traffic; a decode step of 32 requests on 8192 shared positions 1.1 us of 23.5
    // less) a column far below the row's largest loses its bits, and all of them below 2^-25 of it
    float *po;
    f32x4 *ml;
};

// What a cache holds: the queries' type, e4m3 with a scale per K/V head, and e4m3 or int8 with a scale per block of positions and head.
enum { KV_16 = 0, KV_E4M3 = 1, KV_E4M3_BLOCKS = 2, KV_I8_BLOCKS = 3 };
constexpr bool in_blocks(int kv) { return kv >= KV_E4M3_BLOCKS; }
struct BlockArgs : AttnArgs {         // ks, vs: [n_pages][n_kv][per_page]
    int per_page;                     // blocks of a page
    PageDivisor by_block;
};
template <int KV> using ArgsOf = std::conditional_t<in_blocks(KV), BlockArgs, AttnArgs>;
constexpr int SCALE_KEYS = 16;        // blocks are whole runs of this many positions
constexpr float LEAST_SCALE = 0x1p-60f;

template <class T> struct Mma;
template <> struct Mma<f16> {
    typedef f16x8 frag;
    static constexpr uint32_t INF = 0x7c00;                            // bits of infinity
    static constexpr float LAZY = 0.f;
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pair(uint32_t codes, bool hi) {          // two e4m3 codes of a dword's half
        return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true))
                  : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false));
    }
};
template <> struct Mma<bf16> {
    typedef bf16x8 frag;
    static constexpr uint32_t INF = 0x7f80;
    static constexpr float LAZY = 8.f;
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pair(uint32_t codes, bool hi) {
        return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true))
                  : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false));
    }
};
template <class T>
__device__ __forceinline__ typename Mma<T>::frag from_e4m3(u32x2 c) {       // exact: e4m3 is a subset of fp16 and of bf16
    const u32x4 w = {Mma<T>::pair(c.x, false), Mma<T>::pair(c.x, true), Mma<T>::pair(c.y, false), Mma<T>::pair(c.y, true)};
    return __builtin_bit_cast(typename Mma<T>::frag, w);
}

// int8 codes, exact in both types: fp16 from bytes under the exponent of 1024 (q8_pair), bf16, whose 8 bits of fraction do not hold
// that sum, by way of fp32 (the upper half is the value).
template <class T>
__device__ __forceinline__ typename Mma<T>::frag from_i8(u32x2 c) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (std::is_same<T, f16>::value) {
            const uint32_t u = c[i] ^ 0x80808080u;
            w[2 * i] = __builtin_bit_cast(uint32_t, q8_pair(u, 0x04010400u));
            w[2 * i + 1] = __builtin_bit_cast(uint32_t, q8_pair(u, 0x04030402u));
        } else {
            uint32_t f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = __float_as_uint((float)(int8_t)(c[i] >> (8 * j)));
            w[2 * i] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
            w[2 * i + 1] = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
        }
    }
    return __builtin_bit_cast(typename Mma<T>::frag, w);
}

// Piece (16 bytes) c of row k lies at piece c ^ piece_swap<NCH>(k).  Reads of one piece of 16 rows and transpose reads of a
// pair of pieces of 4 rows each fall on distinct banks (rows of 256, 128 and 64 bytes).
template <int NCH>
__device__ __forceinline__ int piece_swap(int k) {
    if constexpr (NCH == 16) return ((k & 3) << 2) | ((k >> 1) & 2) | ((k >> 3) & 1);
    else if constexpr (NCH == 8) return ((k & 2) << 1) | ((k >> 1) & 2) | ((k >> 3) & 1);
    else return ((k >> 1) & 2) | ((k >> 3) & 1);
}

// One 16-byte global-to-LDS copy per lane: lane i's 16 bytes at g land at LDS byte address lds + 16 i.  Inline asm so that the
// compiler does not make every LDS read wait for the copies in flight; copies_wait counts them.  The hardware needs one
// wait state between the scalar write of M0 (the LDS address) and the copy.
__device__ __forceinline__ void copy_to_lds(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds) : "memory");
}
// The same of 4 bytes a lane: lane i's land at lds + 4 i.
__device__ __forceinline__ void copy_dword_to_lds(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "s"(lds) : "memory");
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The other half's value of lane ^ 32, combined.
__device__ __forceinline__ float half_max(float v) {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float half_sum(float v) {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// LDS of a block: tiles (64 KiB), which the join over key waves reuses, the pool rows of the next TABLE_KEYS positions, the
// key waves' (m, l).  Two blocks share a CU (8 waves: one block's loads and exponentials beside the other's matrix products).
constexpr int TABLE_KEYS = 2048;
constexpr int TILE_SMEM = 65536;
template <int KV> constexpr int attn_smem = TILE_SMEM + (in_blocks(KV) ? TABLE_KEYS / SCALE_KEYS * 5 * 4 : 0);
struct AttnShared {                                                    // beside the tiles
    uint32_t rows[TABLE_KEYS];                                         // pool row of each position (0 where there is none)
    uint32_t seen[TABLE_KEYS / 32];                                    // which positions exist
    int nonfinite;                                                     // values cleared at the border
    float2 ml[4][32];
};

// WIDE: codes are brought to 16 bits on the way, once for all row waves.
template <bool KV8, int HD, int WM, bool WIDE = false>
struct AttnTile {
    static constexpr int WK = 4 / WM;                                  // waves over keys
    static constexpr int RB = HD * (KV8 ? 1 : 2), NCH = RB / 16;       // bytes and pieces of a row
    static constexpr int KT = WM == 2 || (WM == 1 && RB == 256) ? 32 : 64;      // keys of a tile (of one group of WM waves)
    static constexpr int STAGES = WM == 1 ? 1 : 2;
    static constexpr int TILE = KT * (WIDE ? HD * 2 : RB);             // LDS bytes of a tile's keys (and of its values)
    static constexpr int ALL = KT * NCH / 64;                          // copies of a tile's keys, and of its values
    static constexpr int COPIES = ALL / WM;                            // ... of a wave
    static constexpr int QUADS = HD / 8;                               // 4-value pieces of a lane's half of a row
    static constexpr int JOIN = 4 * 32 * HD * 4;                       // LDS of the join over the key waves
    static_assert(ALL >= WM && ALL % WM == 0, "whole copies");
    static_assert(WK * STAGES * 2 * TILE <= TILE_SMEM && JOIN <= TILE_SMEM, "LDS plan");
    static_assert(TABLE_KEYS % (WK * KT) == 0, "whole rounds of the row table");
};

// x, of which the compiler knows nothing: what is computed from it stays where it is written.  Addresses of copies and of rare
// paths would otherwise be kept in registers over the loops, which need theirs for the accumulators.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <class V>
__device__ __forceinline__ __attribute__((address_space(3))) V *lds_at(uint32_t address) {
    return (__attribute__((address_space(3))) V *)(size_t)address;
}

template <class T, int KV, int HD, int WM>
__device__ __forceinline__ void run_item(const ArgsOf<KV> &a, const Item &w, unsigned char *smem, AttnShared &sh) {
    constexpr bool KV8 = KV != KV_16, BLOCKS = in_blocks(KV), I8 = KV == KV_I8_BLOCKS;
    constexpr bool WIDE = I8 && WM > 1;
    typedef AttnTile<KV8, HD, WM, WIDE> TL;
    typedef Mma<T> M;
    typedef typename M::frag frag;
    constexpr int KT = TL::KT, RB = TL::RB, NCH = TL::NCH, WK = TL::WK, NS = HD / 16, ND = HD / 32, SUB = KT / 32;
    constexpr int RPC = 64 / NCH;                                      // rows of one copy
    constexpr bool OP8 = KV8 && !WIDE;                                 // what the products' operands are read from: codes,
    constexpr int ORB = WIDE ? HD * 2 : RB, ONCH = ORB / 16;           // bytes and pieces of a row
    // (blocks: what is computed from it stays inside the item, else the values that all kinds share are kept over the loop of items and int8's
    // larger tiles, with codes in registers, go to scratch memory: a captured step of 64 x 4096 56.3 us instead of 51.6)
    const int tid0 = BLOCKS ? opaque(threadIdx.x) : threadIdx.x;
    const int lane = tid0 & 63, wv = __builtin_amdgcn_readfirstlane(tid0 >> 6);
    const int col = lane & 31, h = lane >> 5;                          // the lane's query row; its half of every 8 keys
    const int rw = wv % WM, kw = wv / WM;
    unsigned char *const buf0 = smem + kw * (TL::STAGES * 2 * TL::TILE);       // [stage][keys, values] of this key wave
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
        (uint32_t)(size_t)((__attribute__((address_space(3))) unsigned char *)buf0));

    // The chain of an item is its table's entries, their rows of the pool, the copies: the entries are asked for first.
    const int *table = a.table + (int64_t)w.seq * a.max_pages;
    auto page_of = [&](int key) { return key / a.by_page; };           // (of no meaning behind the last key, where it is not used)
    auto entry_of = [&](int key, int page) { return key < w.k1 && w.seq < a.n_seq && page < a.max_pages ? table[page] : -1; };
    if (threadIdx.x == 0) sh.nonfinite = 0;
    // (with blocks the tiles begin on whole SCALE_KEYS; positions before the item's first do not exist for it)
    const int k0 = BLOCKS ? w.k0 & -SCALE_KEYS : w.k0;
    // of each SCALE_KEYS positions of the table: (kc, lv) and iv (see make_terms), and the scales as they lie in the cache, keys', values'
    constexpr int BLOCKS_OF = TABLE_KEYS / SCALE_KEYS;
    float *const terms = (float *)(smem + TILE_SMEM), *const inverses = terms + 2 * BLOCKS_OF, *const raw_scales = inverses + BLOCKS_OF;
    const int key0 = k0 + (int)threadIdx.x, page0 = page_of(key0), entry0 = entry_of(key0, page0);

    const int row = rw * 32 + col;
    // (a captured call may meet tables set later: its own sizes bound every access)
    const int rt = row / a.by_g;
    int at = w.tok0 + rt;
    if (__builtin_expect(w.list >= 0, 0)) {
        at = ((const int *)a.items)[-1 - (w.list + min(rt, w.ntok - 1))];      // (the list lies before the items, backwards)
        asm volatile("" : "+v"(at));                                   // (awaited here: behind the branch every item would wait for its entries)
    }
    const bool live = row < w.ntok * a.G && at < a.rows;
    const int tok = live ? rt : 0, hh = live ? row - rt * a.G : 0;
    frag qf[NS];
    {
        const T *q = (const T *)a.q + (int64_t)(live ? at : min(w.tok0, a.rows - 1)) * a.q_row + (int64_t)(w.kvh * a.G + hh) * a.q_head + 8 * h;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = *(const frag *)(q + 16 * s);
    }
    // the row sees positions < lim; rows behind the tile's last compute along and are never stored.  lo and hi: the least and
    // the greatest of the wave's rows (its first and last token)
    const int lim = live ? min(w.k1, w.pos0 + tok + 1) : w.k1;
    const int lo = min(w.k1, w.pos0 + (rw * 32) / a.by_g + 1);
    const int hi = rw * 32 < w.ntok * a.G ? min(w.k1, w.pos0 + min(w.ntok - 1, (rw * 32 + 31) / a.by_g) + 1) : 0;
    const float sc = KV == KV_E4M3 ? a.scale * a.ks[w.kvh] : a.scale;

    const int swz = piece_swap<ONCH>(col);
    const int tg = (lane >> 4) & 1, ti = lane & 15;                    // which 16 of 32 dims; lane within them

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] = 0.f;
    float m = -INFINITY, l = 0.f;                                      // m in log2 units; l of the lane's own keys

    // copies of tile t of the row table (this wave's share) to LDS address `to`, keys or values.  Row kr of the tile is copied by
    // lanes of copy kr / RPC; the swap of its pieces is the lane's own, xor one that the copy alone decides.
    const int copy0 = rw * TL::COPIES * RPC + lane / NCH;
    const uint32_t piece0 = (uint32_t)((lane % NCH) ^ piece_swap<NCH>(copy0)) << 4;
    auto rows_of = [&](int t, uint32_t *r) {
        const uint32_t *rows = sh.rows + t * KT + copy0;
#pragma unroll
        for (int c = 0; c < TL::COPIES; ++c) r[c] = rows[c * RPC];
    };
    auto offset_of = [&](uint32_t r, int c) -> uint64_t {                // (keys and values at the same place; rows of 2^n bytes)
        const uint32_t low = r * RB + ((uint32_t)opaque(piece0) ^ (uint32_t)(piece_swap<NCH>(c * RPC) << 4));
        return (uint64_t)(r >> (32 - __builtin_ctz(RB))) << 32 | low;
    };
    auto copy_row = [&](const uint8_t *pool, uint64_t offset, uint32_t to, int c) {
        copy_to_lds(pool + offset, to + (rw * TL::COPIES + c) * 1024);
    };
    auto copy_tile = [&](const uint8_t *pool, int t, uint32_t to) {
        uint32_t r[TL::COPIES];
        rows_of(t, r);
#pragma unroll
        for (int c = 0; c < TL::COPIES; ++c) copy_row(pool, offset_of(r[c], c), to, c);
    };
    // which of 32 positions exist (block b of the row table)
    auto seen_of = [&](int b) -> uint32_t { return __builtin_amdgcn_readfirstlane(sh.seen[b]); };
    // Values that a weight of 0 may meet must be finite (each wave its own copies): those without a position, which are row 0 of
    // the pool, become zeros; so do infinities and NaNs of the border's tiles, which hold keys that some rows see and some
    // do not, and the rows that see them get them at the end.
    const int border = w.ntok > 1 ? k0 + max(min(w.k1, w.pos0 + 1) - k0, 0) / KT * KT : w.k1;
    auto clear_values = [&](int vb, int t, int t0, uint32_t all) {
        if (I8 || (all == ~0u && t0 < border)) return;                 // (every int8 code is finite)
        const int ln = opaque(lane);
#pragma unroll 1
        for (int c = 0; c < TL::COPIES; ++c) {
            const int n = rw * TL::COPIES + c, kr = n * RPC + ln / NCH;
            u32x4 *const at = (u32x4 *)(buf0 + vb + n * 1024 + ln * 16);
            u32x4 v = {0, 0, 0, 0};
            if ((sh.seen[t * SUB + kr / 32] >> (kr & 31)) & 1) {
                if (t0 < border) continue;
                v = *at;
                bool any = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t big = KV8 ? ((v[i] & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u
                                             : ((v[i] & 0x7fff7fffu) + (0x8000u - M::INF) * 0x10001u) >> 15 & 0x00010001u;
                    v[i] &= ~(big * (KV8 ? 0xffu : 0xffffu));
                    any |= big != 0;
                }
                if (!any) continue;
                sh.nonfinite = 1;
            }
            *at = v;
        }
        lds_wait();
    };
    // 32 keys at a time: scores (kb: their rows), then maxima, weights, outputs (vb: their rows).  The lane's operands: LDS addresses in
    // the wave's first tile, kb and vb constants beside them, so that reads need no address of their own
    uint32_t ka[NS], va[2][ND];
#pragma unroll
    for (int p = 0; p < NS; ++p) ka[p] = lds0 + (OP8 ? col * ORB + (((swz ^ p) << 4) | (h << 3)) : col * ORB + ((h ^ swz ^ (2 * p)) << 4));
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if constexpr (OP8) {
            const int rr = ti >> 1, key = 8 * (rr >> 2) + 4 * h + (rr & 3);
            va[0][d] = va[1][d] = lds0 + key * ORB + (((2 * d + tg) ^ piece_swap<ONCH>(key)) << 4) + ((ti & 1) << 3);
        } else {
            const int key = 4 * h + (ti >> 2), c = 4 * d + 2 * tg + ((ti >> 1) & 1);
            va[0][d] = lds0 + key * ORB + ((c ^ piece_swap<ONCH>(key)) << 4) + ((ti & 1) << 3);
            va[1][d] = lds0 + (key + 8) * ORB + ((c ^ piece_swap<ONCH>(key + 8)) << 4) + ((ti & 1) << 3);
        }
    }
    // (sums for good: the compiler would add the wave's part again at every read)
#pragma unroll
    for (int p = 0; p < NS; ++p) asm volatile("" : "+v"(ka[p]));
#pragma unroll
    for (int d = 0; d < ND; ++d) asm volatile("" : "+v"(va[0][d]), "+v"(va[1][d]));
    // operands as LDS gives them, and as the products take them: e4m3 is converted when it is used, after the wait for it
    typedef std::conditional_t<OP8, u32x2, u32x4> raw;
    auto widened = [&](u32x2 x) -> frag {
        if constexpr (I8) return from_i8<T>(x);
        else return from_e4m3<T>(x);
    };
    auto cooked = [&](raw x) -> frag {
        if constexpr (OP8) return widened(x);
        else return __builtin_bit_cast(frag, x);
    };
    auto value_raw = [&](int vb, int y, int d) -> raw {           // keys 16 y .. + 15
        if constexpr (OP8) {
            return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                lds_at<i32x2>(va[0][d] + vb + 16 * y * ORB)));
        } else {
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(va[0][d] + vb + 16 * y * ORB));
            const s16x4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(va[1][d] + vb + 16 * y * ORB));
            const u32x2 xx = __builtin_bit_cast(u32x2, x), zz = __builtin_bit_cast(u32x2, z);
            return (u32x4){xx.x, xx.y, zz.x, zz.y};
        }
    };
    auto read_keys = [&](int kb, raw (&k)[NS]) {
#pragma unroll
        for (int p = 0; p < NS; ++p) k[p] = *lds_at<raw>(ka[p] + kb);
    };
    auto read_values = [&](int vb, int y, raw (&v)[ND]) {
#pragma unroll
        for (int d = 0; d < ND; ++d) v[d] = value_raw(vb, y, d);
    };
    auto scores = [&](const raw (&k)[NS], f32x16 &s) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
        for (int p = 0; p < NS; ++p) s = M::run(cooked(k[p]), qf[p], s);
    };
    // With blocks: a key's score is s kc, its weight times its values' scale is 2^(s kc + lv), and that weight over the scale is the
    // weight itself.  Exponents are taken of s kc + lv: then what is rounded to T for the product with the values is at most 1
    // however the scales of a row's blocks differ, and the sum of weights takes the scale out again (iv) in fp32.  As kc is positive a
    // block's largest s is that of its exponents too.
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    struct Terms { f32x2 kc[SUB], lv[SUB], iv[SUB]; };                 // of keys 0 .. 15 and 16 .. 31
    // A wave's own copies of scales, which have landed, as terms: 4 of each 256 positions of the table.
    auto make_terms = [&]() {
        if constexpr (BLOCKS) {
            constexpr int PER = 64 / SCALE_KEYS, ROUND = 256 / SCALE_KEYS;
            const int ln = opaque(lane);
            if (ln < TABLE_KEYS / 256 * PER) {
                const int b = ln / PER * ROUND + wv * PER + ln % PER;
                const float vs = raw_scales[BLOCKS_OF + b];
                // (a scale of 0, of pages that were never written, stands for the least one; a NaN reaches the rows that see it)
                const float v = vs < LEAST_SCALE ? LEAST_SCALE : vs;
                const float ks = raw_scales[b], k = ks < LEAST_SCALE ? LEAST_SCALE : ks;
                *(float2 *)(terms + 2 * b) = make_float2(k * a.scale, __builtin_amdgcn_logf(v));
                inverses[b] = v < INFINITY ? 1.f / v : 0.f;
            }
        }
    };
    // masks a tile's scores, positions from t0, and brings the running maximum up to date; returns the exponent's base
    auto maxima = [&](f32x16 (&s)[SUB], int t, int t0, const uint32_t (&seen)[SUB], Terms &x) -> float {
        if constexpr (BLOCKS) {
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const f32x4 y = *(const f32x4 *)(terms + 2 * (t * (KT / SCALE_KEYS) + 2 * u));
                x.kc[u] = (f32x2){y.x, y.z};
                x.lv[u] = (f32x2){y.y, y.w};
                x.iv[u] = *(const f32x2 *)(inverses + t * (KT / SCALE_KEYS) + 2 * u);
            }
        }
        if (t0 + KT > lo || (seen[0] & seen[SUB - 1]) != ~0u) {
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const uint32_t mine = seen[u] >> (4 * h);
                const int left = lim - t0 - u * 32 - 4 * h;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int kk = 8 * (j / 4) + j % 4;
                    // (a hidden key's terms may be anything)
                    const float v = BLOCKS ? __builtin_fmaf(s[u][j], x.kc[u][j / 8], x.lv[u][j / 8]) : s[u][j];
                    s[u][j] = kk < left && ((mine >> kk) & 1) ? v : -INFINITY;
                }
                if constexpr (BLOCKS) {
                    x.kc[u] = (f32x2){1.f, 1.f};
                    x.lv[u] = (f32x2){0.f, 0.f};
                }
            }
        }
        float mx = BLOCKS ? -INFINITY : s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
            if constexpr (BLOCKS) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float b = s[u][8 * y];
#pragma unroll
                    for (int j = 1; j < 8; ++j) b = fmaxf(b, s[u][8 * y + j]);
                    mx = fmaxf(mx, __builtin_fmaf(b, x.kc[u][y], x.lv[u][y]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[u][j]);
            }
        mx = fmaxf(m, BLOCKS ? half_max(mx) : half_max(mx) * sc);
        // weights are taken from the base m.  With bf16 weights it follows the maximum only when that has grown by more than
        // 2^8, and the outputs need no rescaling up to there; with fp16 weights it is the maximum, whose weight is then
        // exactly 1 (outputs 2.4e-4 from the 64-bit result, 3.3e-4 by the other rule).  (A row that has seen nothing stays empty.)
        if (__any(mx > m + M::LAZY)) {
            const float keep = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mx);
            l *= keep;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[d][j] *= keep;
            m = mx;
        }
        return m == -INFINITY ? 0.f : m;
    };
    auto weights = [&](const f32x16 &s, float base, const Terms &x, int u, frag (&pf)[2], int j0, int n) {
#pragma unroll
        for (int j = j0; j < j0 + n; ++j) {
            const float p = __builtin_amdgcn_exp2f(BLOCKS ? __builtin_fmaf(s[j], x.kc[u][j / 8], x.lv[u][j / 8]) : s[j] * sc - base);
            if constexpr (BLOCKS) l = __builtin_fmaf(p, x.iv[u][j / 8], l);
            else l += p;
            pf[j / 8][j % 8] = (T)p;
        }
    };
    // The tile's weights and outputs; v0: the values of its first 16 keys.  Operands are read a group of products ahead, and the
    // second half's exponentials stand between the first half's products: left to itself the compiler reads each product's
    // operands right before it and waits for them.
    auto tile_outputs = [&](int vb, raw (&v0)[ND], const f32x16 (&s)[SUB], float base, Terms &x) {
        raw v1[ND];
        frag pf[SUB][2];
        if constexpr (BLOCKS) {
#pragma unroll
            for (int u = 0; u < SUB; ++u) x.lv[u] = (f32x2){x.lv[u].x - base, x.lv[u].y - base};
        }
        read_values(vb, 1, v1);
        __builtin_amdgcn_sched_barrier(0);
        weights(s[0], base, x, 0, pf[0], 0, 16);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (SUB == 2) {
            constexpr int PER = 16 / (2 * ND);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    raw &v = y ? v1[d] : v0[d];
                    o[d] = M::run(cooked(v), pf[0][y], o[d]);
                    v = value_raw(vb + 32 * ORB, y, d);
                    weights(s[1], base, x, 1, pf[1], (y * ND + d) * PER, PER);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = M::run(cooked(y ? v1[d] : v0[d]), pf[SUB - 1][y], o[d]);
    };

    for (int c0 = k0; c0 < w.k1; c0 += TABLE_KEYS) {
        // the pool rows of the next positions (row 0 where there is none), and which exist
        const bool first = c0 == k0;
        if (!first) lds_barrier();
        const int tid = opaque(threadIdx.x);
#pragma unroll 1
        for (int j = tid; j < TABLE_KEYS && c0 + j - tid < w.k1 + 64; j += 256) {  // (a tile past the end reads up to 63 rows past it)
            const int key = c0 + j, page = first && j == tid ? page0 : page_of(key);
            const int e = first && j == tid ? entry0 : entry_of(key, page);
            const bool in_pool = e >= 0 && e < a.n_pages, ok = in_pool && (!BLOCKS || key >= w.k0);
            if constexpr (BLOCKS) {                                    // lanes 0 .. 3: of the wave's 64 positions
                const int ln = tid & 63, b = ln < 64 / SCALE_KEYS ? ln : 0, eb = __shfl(in_pool ? e : -1, b * SCALE_KEYS);
                const int kb = key - ln + b * SCALE_KEYS, pb = page_of(kb);
                const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(size_t)((__attribute__((address_space(3))) float *)(raw_scales + j / SCALE_KEYS)));
                if (ln < 64 / SCALE_KEYS && eb >= 0) {
                    const int64_t at = ((int64_t)eb * (a.NH / a.G) + w.kvh) * a.per_page + (kb - pb * a.page_size) / a.by_block;
                    copy_dword_to_lds(a.ks + at, to);
                    copy_dword_to_lds(a.vs + at, to + BLOCKS_OF * 4);
                }
            }
            sh.rows[j] = ok ? (uint32_t)e * a.page_rows + (uint32_t)w.kvh * a.head_rows + (uint32_t)(key - page * a.page_size) * a.slot_rows : 0u;
            const uint64_t b = __ballot(ok);
            if ((tid & 63) == 0) *(uint64_t *)&sh.seen[j / 32] = b;
        }
        lds_barrier();
        // the queries have landed: inside the loops the compiler must not wait for them, which would wait for the copies too
#pragma unroll
        for (int p = 0; p < NS; ++p) asm volatile("" : "+v"(qf[p]));
        const int nt = (min(w.k1 - c0, TABLE_KEYS) + KT - 1) / KT;     // tiles; this key wave's are kw, kw + WK ..
        if constexpr (WM == 1) {
            // a wave of its own: one tile, keys and values copied apart, so that the next keys are on their way while the
            // values are awaited and used
            constexpr int kb = 0, vb = TL::TILE;
            const int n = min(nt, (max(hi - c0, 0) + KT - 1) / KT);    // tiles behind the last seen position are skipped
            if (kw < n) {
                copy_tile(a.k, kw, lds0);
                copy_tile(a.v, kw, lds0 + TL::TILE);
            }
            for (int t = kw; t < n; t += WK) {
                const bool more = t + WK < n;
                uint32_t seen[SUB];
#pragma unroll
                for (int u = 0; u < SUB; ++u) seen[u] = seen_of(t * SUB + u);
                copies_wait<TL::COPIES>();
                f32x16 s[SUB];
                raw k[SUB][NS], v0[ND];
#pragma unroll
                for (int u = 0; u < SUB; ++u) read_keys(kb + u * 32 * ORB, k[u]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < SUB; ++u) scores(k[u], s[u]);
                if constexpr (BLOCKS) {                                // (a wave's tiles are the positions whose scales it copied, before them)
                    static_assert(!BLOCKS || (KT == 64 && WK == 4), "tiles of a wave");
                    if (t == kw) make_terms();
                }
                lds_wait();
                if (more) copy_tile(a.k, t + WK, lds0);
                Terms x;
                const float base = maxima(s, t, c0 + t * KT, seen, x);
                if (more) copies_wait<TL::COPIES>();
                else copies_wait<0>();
                clear_values(vb, t, c0 + t * KT, seen[0] & seen[SUB - 1]);
                read_values(vb, 0, v0);
                tile_outputs(vb, v0, s, base, x);
                lds_wait();
                if (more) copy_tile(a.v, t + WK, lds0 + TL::TILE);
            }
        } else {
            // the row waves share a tile; the next one is copied meanwhile
            const int rounds = (nt + WK - 1) / WK;
            // WIDE: codes go through registers, a tile ahead of the one that is brought to 16 bits and written behind matrix products
            u32x4 codes[2][WIDE ? TL::COPIES : 1];
            auto fetch_codes = [&](int t) {
                uint32_t r[TL::COPIES];
                rows_of(t, r);
#pragma unroll
                for (int c = 0; c < TL::COPIES; ++c) {
                    const uint64_t at = offset_of(r[c], c);
                    codes[0][c] = *(const u32x4 *)(a.k + at);
                    codes[1][c] = *(const u32x4 *)(a.v + at);
                }
            };
            // (the place of the lane's first codes in a tile; the others' differ by constants, as piece_swap of a sum of such rows is
            // the xor of the rows' own)
            const int wide_piece = (lane % NCH) ^ piece_swap<NCH>(copy0);
            const uint32_t wide0 = copy0 * ORB + (((2 * wide_piece) ^ piece_swap<ONCH>(copy0)) << 4);
            auto put_codes = [&](uint32_t to, int v) {
#pragma unroll
                for (int c = 0; c < TL::COPIES; ++c) {
                    const uint32_t swap = ((2 * piece_swap<NCH>(c * RPC)) ^ piece_swap<ONCH>(c * RPC)) << 4;
                    const uint32_t at = to + v * TL::TILE + c * RPC * ORB;
                    const u32x4 x = codes[v][c];
                    *lds_at<frag>(at + (wide0 ^ swap)) = widened((u32x2){x.x, x.y});
                    *lds_at<frag>(at + (wide0 ^ swap ^ 16)) = widened((u32x2){x.z, x.w});
                }
            };
            if constexpr (WIDE) {
                fetch_codes(kw);
                copies_wait<0>();
                make_terms();
                put_codes(lds0, 0);
                put_codes(lds0, 1);
                if (rounds > 1) fetch_codes(kw + WK);
            } else {
                copy_tile(a.k, kw, lds0);
                copy_tile(a.v, kw, lds0 + TL::TILE);
                if constexpr (BLOCKS) {
                    copies_wait<0>();
                    make_terms();
                }
            }
            uint32_t seen_next[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) seen_next[u] = seen_of(kw * SUB + u);
            auto step = [&](int i, auto stage_of) {
                constexpr int ST = decltype(stage_of)::value * 2 * TL::TILE;
                const int t = i * WK + kw;
                const bool more = i + 1 < rounds;
                constexpr int kb = ST, vb = ST + TL::TILE;
                const uint32_t to = lds0 + (2 * TL::TILE - ST);
                uint32_t seen[SUB], r[TL::COPIES];
#pragma unroll
                for (int u = 0; u < SUB; ++u) seen[u] = seen_next[u];
                if (more) {                                            // (read ahead of the barrier)
                    if constexpr (!WIDE) rows_of(t + WK, r);
#pragma unroll
                    for (int u = 0; u < SUB; ++u) seen_next[u] = seen_of((t + WK) * SUB + u);
                }
                if constexpr (!WIDE) {
                    copies_wait<0>();
                    clear_values(vb, t, c0 + t * KT, seen[0] & seen[SUB - 1]);
                }
                lds_barrier();
                // the next tile's copies are issued behind matrix products: a CU takes one in 16 cycles, and four waves that
                // issue theirs together wait for each other
                auto copies = [&](int part) {
                    if (!more) return;
                    if constexpr (WIDE) {
#pragma unroll
                        for (int v = part; v < 2; v += SUB) put_codes(to, v);
                        if (part == SUB - 1 && i + 2 < rounds) fetch_codes(t + 2 * WK);
                    } else {
#pragma unroll
                        for (int c = part; c < TL::COPIES; c += SUB) {
                            const uint64_t at = offset_of(r[c], c);
                            copy_row(a.k, at, to, c);
                            copy_row(a.v, at, to + TL::TILE, c);
                        }
                    }
                };
                if (c0 + t * KT >= hi) {
#pragma unroll
                    for (int u = 0; u < SUB; ++u) copies(u);
                    return;
                }
                f32x16 s[SUB];
                raw k[SUB][NS], v0[ND];
#pragma unroll
                for (int u = 0; u < SUB; ++u) read_keys(kb + u * 32 * ORB, k[u]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    scores(k[u], s[u]);
                    copies(u);
                }
                read_values(vb, 0, v0);
                Terms x;
                const float base = maxima(s, t, c0 + t * KT, seen, x);
                tile_outputs(vb, v0, s, base, x);
            };
            for (int i = 0; i < rounds; i += 2) {
                step(i, std::integral_constant<int, 0>{});
                if (i + 1 < rounds) step(i + 1, std::integral_constant<int, 1>{});
            }
        }
    }
    if constexpr (BLOCKS) copies_wait<0>();                            // (scales of a wave without tiles)
    l = half_sum(l);
    if (w.ntok > 1) lds_barrier();
    const bool nonfinite = w.ntok > 1 && __builtin_amdgcn_readfirstlane(sh.nonfinite);

    // The key waves of a row group joined in LDS: each takes a share of the values (4-value pieces q0 ..) of all of them
    constexpr int SHARE = TL::QUADS / WK;
    const int q0 = WK > 1 ? kw * SHARE : 0;
    f32x4 out[SHARE];
    if constexpr (WK > 1) {
        lds_barrier();
        f32x4 *const area = (f32x4 *)smem;                             // [key wave][piece][row wave][lane]
        if (h == 0) sh.ml[wv][col] = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                area[((kw * TL::QUADS + d * 4 + j) * WM + rw) * 64 + lane] =
                    (f32x4){o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
        lds_barrier();
        float mm = -INFINITY, f[WK];
#pragma unroll
        for (int k = 0; k < WK; ++k) mm = fmaxf(mm, sh.ml[k * WM + rw][col].x);
        const float base = mm == -INFINITY ? 0.f : mm;
        l = 0.f;
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            const float2 x = sh.ml[k * WM + rw][col];
            f[k] = __builtin_amdgcn_exp2f(x.x - base);
            l += x.y * f[k];
        }
        m = mm;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
            out[i] = area[((q0 + i) * WM + rw) * 64 + lane] * f[0];
#pragma unroll
            for (int k = 1; k < WK; ++k) out[i] += area[((k * TL::QUADS + q0 + i) * WM + rw) * 64 + lane] * f[k];
        }
    } else {
#pragma unroll
        for (int i = 0; i < SHARE; ++i)
            out[i] = (f32x4){o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
    }
    if (nonfinite) {
#pragma unroll 1
        for (int key = max(border, w.k0); key < w.k1; ++key) {
            const int page = page_of(key), e = entry_of(key, page);
            if (e < 0 || e >= a.n_pages || key >= lim) continue;
            const uint8_t *v = a.v + (uint64_t)((uint32_t)e * a.page_rows + (uint32_t)w.kvh * a.head_rows + (uint32_t)(key - page * a.page_size) * a.slot_rows) * RB +
                               (4 * h + 8 * q0) * (KV8 ? 1 : 2);
#pragma unroll
            for (int i = 0; i < SHARE; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if constexpr (KV8) {
                        if ((v[8 * i + c] & 0x7f) == 0x7f) out[i][c] = NAN;
                    } else {
                        const float x = (float)((const T *)v)[8 * i + c];
                        if (!(fabsf(x) < INFINITY)) out[i][c] += x;
                    }
                }
        }
    }
    const int row2 = rw * 32 + (opaque(lane) & 31), tok2 = row2 / a.by_g;
    if (row2 < w.ntok * a.G && (w.rec >= 0 || w.tok0 + tok2 < a.rows)) {       // (records have room for every row of the plan)
        const int hh2 = row2 - tok2 * a.G;
        const float vs = KV == KV_E4M3 ? a.vs[w.kvh] : 1.f;
        if (w.rec < 0) {
            const float il = l > 0.f ? vs / l : 0.f;                   // a row that sees nothing: zeros
            const int64_t head = w.kvh * a.G + hh2;
            T *d0 = (T *)a.out + (int64_t)(w.tok0 + tok2) * a.out_row + head * a.out_head + 4 * h + 8 * q0;
#pragma unroll
            for (int i = 0; i < SHARE; ++i) {
                typedef T T4 __attribute__((ext_vector_type(4)));
                *(T4 *)(d0 + 8 * i) = (T4){(T)(out[i][0] * il), (T)(out[i][1] * il), (T)(out[i][2] * il), (T)(out[i][3] * il)};
            }
            if (a.lse && h == 0 && kw == 0)
                a.lse[(int64_t)(w.tok0 + tok2) * a.NH + head] = l == 0.f ? -INFINITY : LN2 * (m + log2f(l));
        } else {
            const int64_t rec = w.rec + row2;
            float *d0 = a.po + rec * HD + 4 * h + 8 * q0;
#pragma unroll
            for (int i = 0; i < SHARE; ++i) *(f32x4 *)(d0 + 8 * i) = out[i];
            if (h == 0 && kw == 0) a.ml[rec] = (f32x4){m, l, vs, 0.f};
        }
    }
}

template <class T, int KV, int HD>
__global__ void __launch_bounds__(256, 2) k_paged_attn(ArgsOf<KV> a) {
    extern __shared__ __align__(1024) unsigned char smem[];            // attn_smem<KV>
    __shared__ __align__(16) AttnShared sh;
    const int n = a.n_items ? *a.n_items : gridDim.x;
    for (int it = blockIdx.x; it < n; it += gridDim.x) {
        const Item w = a.items[it];
        if (it != (int)blockIdx.x) lds_barrier();                      // LDS is free of the item before
        if (w.kind == 0) run_item<T, KV, HD, 1>(a, w, smem, sh);
        else if (w.kind == 1) run_item<T, KV, HD, 2>(a, w, smem, sh);
        else run_item<T, KV, HD, 4>(a, w, smem, sh);
    }
}

// The records of a token joined.  Tokens whose item wrote the output itself are left alone; a token without any key gets zeros
// (and lse -inf).  WAVES waves of a block share a (token, query head): each takes every WAVES-th batch of records, four
// (HD 128) or eight (64) records per load and UNROLL loads in flight, and wave 0 adds the waves' sums in order.
struct JoinArgs {
    const TokenRecs *toks;
    const int *n_toks;                // and behind it the most records of a token
    const float *po;
    const f32x4 *ml;
    void *out;
    float *lse;
    int64_t out_row, out_head;
    int rows, NH, G;
};
constexpr int JOIN_UNROLL = 4;
template <int HD> constexpr int JOIN_BATCH = 64 / (HD / 8) * JOIN_UNROLL;      // records that a wave has in flight
template <class T, int HD, int WAVES>
__device__ __forceinline__ void join_heads(const JoinArgs &a) {
    constexpr int LPR = HD / 8, RPL = 64 / LPR, UNROLL = JOIN_UNROLL;  // lanes per record, records per load
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    __shared__ f32x8 sum_s[4][LPR];
    const int tok = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int head = blockIdx.y * (4 / WAVES) + wv / WAVES, part = wv % WAVES;
    if (tok >= min(*a.n_toks, a.rows)) return;
    const TokenRecs t = a.toks[tok];
    if (t.parts[0] < 0 || t.parts[1] < 0) return;
    const bool live = head < a.NH;
    const int kvh = (live ? head : 0) / a.G, hh = (live ? head : 0) - kvh * a.G, n = t.parts[0] + t.parts[1];
    auto rec_of = [&](int j) {
        const int w = j < t.parts[0] ? 0 : 1, p = w ? j - t.parts[0] : j;
        return ((int64_t)t.base[w] + (int64_t)(kvh * t.parts[w] + p) * t.tile[w] + t.i[w]) * a.G + hh;
    };
    const int sub = lane / LPR, li = lane % LPR;
    float M = -INFINITY, L = 0.f;
    f32x8 acc = {};
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int cnt = min(64, n - j0);
        f32x8 v[UNROLL];
        auto fetch = [&](int b) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int j = (b + u * WAVES) * RPL + sub;             // (past the last record: the last again, unused)
                v[u] = *(const f32x8 *)(a.po + rec_of(j0 + min(j, cnt - 1)) * HD + li * 8);
            }
        };
        fetch(part);
        const f32x4 x = lane < cnt ? a.ml[rec_of(j0 + lane)] : (f32x4){-INFINITY, 0.f, 0.f, 0.f};
        const float top = fmaxf(M, wave_max_dpp(x.x));
        const float base = top == -INFINITY ? 0.f : top;
        const float keep = __builtin_amdgcn_exp2f(M - base), f = __builtin_amdgcn_exp2f(x.x - base);
        L = L * keep + wave_sum_dpp(x.y * f);
        acc *= keep;
        M = top;
        const float share = lane < cnt ? x.z * f : 0.f;
        for (int b = part; b * RPL < cnt; b += UNROLL * WAVES) {
            if (b != part) fetch(b);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int j = (b + u * WAVES) * RPL + sub;
                const float fj = __shfl(share, min(j, 63));
                const f32x8 x = j < cnt ? v[u] : (f32x8){};
#pragma unroll
                for (int c = 0; c < 8; ++c) acc[c] += x[c] * fj;
            }
        }
    }
    // the records of one load side by side, then the waves
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] += __shfl_xor(acc[c], o);
    if constexpr (WAVES > 1) {
        if (sub == 0) sum_s[wv][li] = acc;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) acc += sum_s[wv + k][li];
    }
    if (!live || sub != 0) return;
    const float il = L > 0.f ? 1.f / L : 0.f;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T *o = (T *)a.out + (int64_t)tok * a.out_row + (int64_t)head * a.out_head + li * 8;
    *(T4 *)o = (T4){(T)(acc[0] * il), (T)(acc[1] * il), (T)(acc[2] * il), (T)(acc[3] * il)};
    *(T4 *)(o + 4) = (T4){(T)(acc[4] * il), (T)(acc[5] * il), (T)(acc[6] * il), (T)(acc[7] * il)};
    if (a.lse && lane == 0) a.lse[(int64_t)tok * a.NH + head] = L == 0.f ? -INFINITY : LN2 * (M + log2f(L));
}
// WAVES 0: a captured launch, a block per (token, query head), which takes the form that the tables of each replay ask for, so that
// its sums have the eager call's order; the blocks that the one-wave form has too many end at once.
template <class T, int HD, int WAVES>
__global__ void __launch_bounds__(256) k_paged_join(JoinArgs a) {
    if constexpr (WAVES > 0) {
        join_heads<T, HD, WAVES>(a);
    } else if (a.n_toks[1] > JOIN_BATCH<HD>) {
        join_heads<T, HD, 4>(a);
    } else if ((int)blockIdx.y < (a.NH + 3) / 4) {
        join_heads<T, HD, 1>(a);
    }
}

}  // namespace paged
