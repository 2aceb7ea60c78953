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
// many.  Scores, maxima, sums and outputs are fp32; P is rounded to the queries' type for its product with V.
#pragma once
#include "sp_paged_plan.h"
#include "sp_rotate.h"

namespace paged {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct AttnArgs {
    const void *q;
    void *out;
    float *lse;                       // [rows][NH] or NULL
    int64_t q_row, q_head, out_row, out_head;
    const uint8_t *k, *v;
    const float *ks, *vs;             // e4m3: scale per K/V head
    const int *table;                 // [n_seq][max_pages]
    int rows, n_seq, max_pages, n_pages, page_size;      // rows of q and out, of the table; its width; the pool
    uint32_t page_rows;               // page stride in rows of head_dim values
    int NH, G;
    float scale;                      // of the scores, times log2(e)
    const Item *items;
    const int *n_items;
    float *po;                        // records: [rows][HD] unnormalised outputs
    float2 *ml;                       // [rows] (m in log2 units, l)
};

template <class T> struct Mma;
template <> struct Mma<f16> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pair(uint32_t codes, bool hi) {          // two e4m3 codes of a dword's half
        return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true))
                  : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false));
    }
};
template <> struct Mma<bf16> {
    typedef bf16x8 frag;
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

// Piece (16 bytes) c of row k lies at piece c ^ piece_swap<NCH>(k).  Reads of one piece of 16 rows and transpose reads of a
// pair of pieces of 4 rows each fall on distinct banks (rows of 256, 128 and 64 bytes).
template <int NCH>
__device__ __forceinline__ int piece_swap(int k) {
    if constexpr (NCH == 16) return ((k & 3) << 2) | ((k >> 1) & 2) | ((k >> 3) & 1);
    else if constexpr (NCH == 8) return ((k & 2) << 1) | ((k >> 1) & 2) | ((k >> 3) & 1);
    else return ((k >> 1) & 2) | ((k >> 3) & 1);
}

// One 16-byte global-to-LDS copy per lane: lane i's 16 bytes at g land at LDS byte address lds + 16 i.  Inline asm so that the
// compiler does not make every LDS read wait for the copies in flight; copies_landed waits for them.  The hardware needs one
// wait state between the scalar write of M0 (the LDS address) and the copy.
__device__ __forceinline__ void copy_to_lds(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds) : "memory");
}
__device__ __forceinline__ void copies_landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
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

template <bool KV8, int HD, int WM>
struct AttnTile {
    static constexpr int WK = 4 / WM;                                  // waves over keys
    static constexpr int KT = WM == 4 ? 64 : 32;                       // keys of a tile (of one group of WM waves)
    static constexpr int RB = HD * (KV8 ? 1 : 2), NCH = RB / 16;       // bytes and pieces of a row
    static constexpr int TILE = KT * RB;                               // bytes of a tile's keys (and of its values)
    static constexpr int COPIES = KT * NCH / 64 / WM;                  // copies per wave, of keys and of values
    static constexpr int JOIN = (WK - 1) * WM * 32 * HD * 4;           // LDS of the join over the key waves
    static constexpr int SMEM = WK * 2 * 2 * TILE > JOIN ? WK * 2 * 2 * TILE : JOIN;
    static_assert(COPIES >= 1 && COPIES * 64 * WM == KT * NCH, "whole copies");
};

template <class T, bool KV8, int HD, int WM>
__global__ void __launch_bounds__(256, WM == 1 ? 1 : 2) k_paged_attn(AttnArgs a) {
    typedef AttnTile<KV8, HD, WM> TL;
    typedef Mma<T> M;
    typedef typename M::frag frag;
    constexpr int KT = TL::KT, RB = TL::RB, NCH = TL::NCH, WK = TL::WK, NS = HD / 16, ND = HD / 32, SUB = KT / 32;
    constexpr int RPC = 64 / NCH;                                      // rows of one copy
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float2 ml_s[4][32];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;                          // the lane's query row; its half of every 8 keys
    const int rw = wv % WM, kw = wv / WM;
    unsigned char *const buf0 = smem + kw * (4 * TL::TILE);            // [2 stages][keys, values] of this key wave
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
        (uint32_t)(size_t)((__attribute__((address_space(3))) unsigned char *)buf0));

    // reads of a tile: key row `col`, its piece for head-dim step s at kbase ^ (step bytes); values by transpose reads
    const int swz = piece_swap<NCH>(col);
    const int krow = col * RB;
    const int kbase = KV8 ? (swz << 4) | (h << 3) : ((h ^ swz) << 4);
    const int tg = (lane >> 4) & 1, ti = lane & 15;                    // which 16 of 32 dims; lane within them

    for (int it = blockIdx.x; it < *a.n_items; it += gridDim.x) {
        const Item w = a.items[it];
        const int nt = (w.k1 - w.k0 + KT - 1) / KT, ni = (nt + WK - 1) / WK;
        const int row = rw * 32 + col;
        // (a captured call may meet tables set later: its own sizes bound every access)
        const bool live = row < w.ntok * a.G && w.tok0 + row / a.G < a.rows;
        const int tok = live ? row / a.G : 0, hh = live ? row - tok * a.G : 0;
        // the row sees positions < lim; rows behind the tile's last compute along and are never stored
        const int lim = live ? min(w.k1, w.pos0 + tok + 1) : w.k1;
        int lo = lim, hi = live ? lim : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { lo = min(lo, __shfl_xor(lo, o)); hi = max(hi, __shfl_xor(hi, o)); }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);

        frag qf[NS];
        {
            const T *q = (const T *)a.q + (int64_t)min(w.tok0 + tok, a.rows - 1) * a.q_row + (int64_t)(w.kvh * a.G + hh) * a.q_head + 8 * h;
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[s] = *(const frag *)(q + 16 * s);
        }
        const float sc = KV8 ? a.scale * a.ks[w.kvh] : a.scale;

        // the page of key `lane` of tile i of this key wave: entry loaded one tile ahead
        const int *table = a.table + (int64_t)w.seq * a.max_pages;
        auto key_of = [&](int i) { return w.k0 + (kw + i * WK) * KT + (lane & (KT - 1)); };
        auto entry_of = [&](int i) {
            const int key = key_of(i), page = key / a.page_size;
            return key < w.k1 && w.seq < a.n_seq && page < a.max_pages ? table[page] : -1;
        };
        // copies tile i to stage st; returns which of its positions exist
        auto stage = [&](int i, int entry, int st) -> uint64_t {
            const int key = key_of(i);
            const bool ok = key < w.k1 && entry >= 0 && entry < a.n_pages;
            const uint32_t r = ok ? (uint32_t)entry * a.page_rows + (uint32_t)(w.kvh * a.page_size + key % a.page_size) : 0u;
#pragma unroll
            for (int c = 0; c < TL::COPIES; ++c) {
                const int n = rw * TL::COPIES + c, kr = n * RPC + lane / NCH;      // row of the tile
                const uint32_t src = __shfl(r, kr);
                const uint64_t off = (uint64_t)src * RB + (((lane % NCH) ^ piece_swap<NCH>(kr)) << 4);
                const uint32_t to = lds0 + st * (2 * TL::TILE) + n * 1024;
                copy_to_lds(a.k + off, to);
                copy_to_lds(a.v + off, to + TL::TILE);
            }
            return KT == 64 ? __ballot(ok) : __ballot(ok) | 0xffffffff00000000ull;
        };
        // rows without a position hold row 0 of the pool: zeros instead, so that 0 x value stays 0
        auto clear = [&](int st, uint64_t seen) {
            if (seen == ~0ull) return;
#pragma unroll
            for (int c = 0; c < TL::COPIES; ++c) {
                const int n = rw * TL::COPIES + c, kr = n * RPC + lane / NCH;
                if (!((seen >> kr) & 1)) {
                    unsigned char *d = buf0 + st * (2 * TL::TILE) + n * 1024 + lane * 16;
                    *(u32x4 *)d = (u32x4){0, 0, 0, 0};
                    *(u32x4 *)(d + TL::TILE) = (u32x4){0, 0, 0, 0};
                }
            }
        };

        f32x16 o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[d][j] = 0.f;
        float m = -INFINITY, l = 0.f;                                  // m in raw scores; l of the lane's own keys

        int entry = entry_of(0);
        uint64_t next = stage(0, entry, 0);
        entry = entry_of(1);
        for (int i = 0; i < ni; ++i) {
            const int st = i & 1;
            const uint64_t seen = next;
            copies_landed();
            clear(st, seen);
            if constexpr (WM > 1) lds_barrier();
            else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (i + 1 < ni) {
                const int e = entry;
                entry = entry_of(i + 2);
                next = stage(i + 1, e, st ^ 1);
            }
            const int t0 = w.k0 + (kw + i * WK) * KT;                  // the tile's first position
            if (t0 >= hi) continue;
            const unsigned char *kb = buf0 + st * (2 * TL::TILE), *vb = kb + TL::TILE;
            f32x16 s[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
#pragma unroll
                for (int j = 0; j < 16; ++j) s[u][j] = 0.f;
#pragma unroll
                for (int p = 0; p < NS; ++p) {
                    frag kf;
                    if constexpr (KV8) kf = from_e4m3<T>(*(const u32x2 *)(kb + u * 32 * RB + krow + (kbase ^ (p << 4))));
                    else kf = *(const frag *)(kb + u * 32 * RB + krow + (kbase ^ (p << 5)));
                    s[u] = M::run(kf, qf[p], s[u]);
                }
            }
            if (t0 + KT > lo || seen != ~0ull) {
                const uint64_t mine = seen >> (4 * h);
                const int left = lim - t0 - 4 * h;
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int kk = u * 32 + 8 * (j / 4) + j % 4;
                        s[u][j] = kk < left && ((mine >> kk) & 1) ? s[u][j] : -INFINITY;
                    }
            }
            float mx = s[0][0];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[u][j]);
            mx = fmaxf(m, half_max(mx));
            const float base = mx == -INFINITY ? 0.f : mx * sc;        // a row that has seen nothing stays empty
            if (__any(mx > m)) {
                const float keep = __builtin_amdgcn_exp2f(m * sc - base);
                l *= keep;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[d][j] *= keep;
                m = mx;
            }
            frag pf[SUB * 2];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float p = __builtin_amdgcn_exp2f(s[u][j] * sc - base);
                    l += p;
                    pf[u * 2 + j / 8][j % 8] = (T)p;
                }
#pragma unroll
            for (int y = 0; y < SUB * 2; ++y)                          // 16 keys
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    frag vf;
                    if constexpr (KV8) {
                        const int rr = ti >> 1, key = 16 * y + 8 * (rr >> 2) + 4 * h + (rr & 3);
                        const int at = key * RB + (((2 * d + tg) ^ piece_swap<NCH>(key)) << 4) + ((ti & 1) << 3);
                        vf = from_e4m3<T>(__builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                            (__attribute__((address_space(3))) i32x2 *)(vb + at))));
                    } else {
                        const int key = 16 * y + 4 * h + (ti >> 2), c = 4 * d + 2 * tg + ((ti >> 1) & 1);
                        const int a0 = key * RB + ((c ^ piece_swap<NCH>(key)) << 4) + ((ti & 1) << 3);
                        const int a1 = (key + 8) * RB + ((c ^ piece_swap<NCH>(key + 8)) << 4) + ((ti & 1) << 3);
                        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(vb + a0));
                        const s16x4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(vb + a1));
                        const u32x2 xx = __builtin_bit_cast(u32x2, x), zz = __builtin_bit_cast(u32x2, z);
                        vf = __builtin_bit_cast(frag, (u32x4){xx.x, xx.y, zz.x, zz.y});
                    }
                    o[d] = M::run(vf, pf[y], o[d]);
                }
        }
        l = half_sum(l);
        m = m == -INFINITY ? -INFINITY : m * sc;                       // log2 units

        if constexpr (WK > 1) {
            // the key waves of a row group joined in LDS: waves kw > 0 leave theirs, wave kw = 0 adds them in order
            lds_barrier();
            f32x4 *const area = (f32x4 *)smem;
            if (h == 0) ml_s[wv][col] = make_float2(m, l);
            if (kw > 0) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        area[(((kw - 1) * WM + rw) * (4 * ND) + d * 4 + j) * 64 + lane] =
                            (f32x4){o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
            }
            lds_barrier();
            if (kw == 0) {
                float mm = m;
#pragma unroll
                for (int k = 1; k < WK; ++k) mm = fmaxf(mm, ml_s[k * WM + rw][col].x);
                const float base = mm == -INFINITY ? 0.f : mm;
                float f = __builtin_amdgcn_exp2f(m - base);
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[d][j] *= f;
#pragma unroll
                for (int k = 1; k < WK; ++k) {
                    const float2 x = ml_s[k * WM + rw][col];
                    f = __builtin_amdgcn_exp2f(x.x - base);
                    l += x.y * f;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const f32x4 y = area[(((k - 1) * WM + rw) * (4 * ND) + d * 4 + j) * 64 + lane];
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[d][4 * j + c] += y[c] * f;
                        }
                }
                m = mm;
            }
        }
        if (kw == 0 && live) {
            const float vs = KV8 ? a.vs[w.kvh] : 1.f;
            if (w.rec < 0) {
                const float il = l > 0.f ? vs / l : 0.f;               // a row that sees nothing: zeros
                const int64_t head = w.kvh * a.G + hh;
                T *d0 = (T *)a.out + (int64_t)(w.tok0 + tok) * a.out_row + head * a.out_head + 4 * h;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        typedef T T4 __attribute__((ext_vector_type(4)));
                        *(T4 *)(d0 + d * 32 + 8 * j) = (T4){(T)(o[d][4 * j] * il), (T)(o[d][4 * j + 1] * il),
                                                            (T)(o[d][4 * j + 2] * il), (T)(o[d][4 * j + 3] * il)};
                    }
                if (a.lse && h == 0)
                    a.lse[(int64_t)(w.tok0 + tok) * a.NH + head] = l > 0.f ? LN2 * (m + log2f(l)) : -INFINITY;
            } else {
                const int64_t rec = w.rec + row;
                float *d0 = a.po + rec * HD + 4 * h;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *(f32x4 *)(d0 + d * 32 + 8 * j) = (f32x4){o[d][4 * j] * vs, o[d][4 * j + 1] * vs, o[d][4 * j + 2] * vs,
                                                                  o[d][4 * j + 3] * vs};
                if (h == 0) a.ml[rec] = make_float2(m, l);
            }
        }
        lds_barrier();                                                 // LDS is free for the next item
    }
}

// The records of a token joined: one wave per (token, query head), lane i on values HD/64 i ...  Tokens whose item wrote the
// output itself are left alone; a token without any key gets zeros (and lse -inf).
struct JoinArgs {
    const TokenRecs *toks;
    const int *n_toks;
    const float *po;
    const float2 *ml;
    void *out;
    float *lse;
    int64_t out_row, out_head;
    int rows, NH, G;
};
template <class T, int HD>
__global__ void __launch_bounds__(256) k_paged_join(JoinArgs a) {
    const int tok = blockIdx.x, lane = threadIdx.x & 63;
    const int head = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (tok >= min(*a.n_toks, a.rows) || head >= a.NH) return;
    const TokenRecs t = a.toks[tok];
    if (t.parts[0] < 0 || t.parts[1] < 0) return;
    const int kvh = head / a.G, hh = head - kvh * a.G, n = t.parts[0] + t.parts[1];
    auto rec_of = [&](int j) {
        const int w = j < t.parts[0] ? 0 : 1, p = w ? j - t.parts[0] : j;
        return ((int64_t)t.base[w] + (int64_t)(kvh * t.parts[w] + p) * t.tile[w] + t.i[w]) * a.G + hh;
    };
    constexpr int D = HD / 64;
    float M = -INFINITY, L = 0.f, acc[D] = {};
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int cnt = min(64, n - j0);
        const float2 x = lane < cnt ? a.ml[rec_of(j0 + lane)] : make_float2(-INFINITY, 0.f);
        const float top = fmaxf(M, wave_max_dpp(x.x));
        const float base = top == -INFINITY ? 0.f : top;
        const float keep = __builtin_amdgcn_exp2f(M - base), f = __builtin_amdgcn_exp2f(x.x - base);
        L = L * keep + wave_sum_dpp(x.y * f);
#pragma unroll
        for (int d = 0; d < D; ++d) acc[d] *= keep;
        M = top;
#pragma unroll 4
        for (int j = 0; j < cnt; ++j) {
            const float fj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), j));
            const float *p = a.po + rec_of(j0 + j) * HD + lane * D;
#pragma unroll
            for (int d = 0; d < D; ++d) acc[d] += p[d] * fj;
        }
    }
    const float il = L > 0.f ? 1.f / L : 0.f;
    T *o = (T *)a.out + (int64_t)tok * a.out_row + (int64_t)head * a.out_head + lane * D;
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = (T)(acc[d] * il);
    if (a.lse && lane == 0) a.lse[(int64_t)tok * a.NH + head] = L > 0.f ? LN2 * (M + log2f(L)) : -INFINITY;
}

}  // namespace paged
