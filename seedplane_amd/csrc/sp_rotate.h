// Rotary embedding and its fused form, the append of keys and values to a paged cache.
//
// A pair (x1, x2) of a head at position p turns by the angle a = p * inv_freq[j]: f (x1 cos a - x2 sin a),
// f (x2 cos a + x1 sin a).  Pairs are (j, j + rot / 2) (half layout) or (2 j, 2 j + 1) (interleaved) of the head's first
// `rot` values; the rest passes through.
//
// The angle is formed and reduced to one turn in 64 bits: at position 1e6 a 32-bit product is off by 0.03 rad.  Its cosine
// and sine come from sincospif of the reduced turn (32 bits), the rotation runs in 32 bits and rounds once, on the store.
//
// Both kernels are bound by memory for long inputs and by the chain position -> angle -> store for short ones: 2048 rows x 32
// heads of 128 in bf16 rotate in 8.3 us (33.6 MB, 4.0 TB/s), 2048 rows of 28 + 4 + 4 heads are appended in 11.0 us (37.7 MB, 3.4 TB/s),
// and steps of 16 rows take 2.7 and 3.9 us, where an empty launch takes 2.3 (a copy of 1 GiB: 5.1 TB/s).  A row of more units than a
// block has threads (the 320 of 28 + 4 + 4 heads of 128) takes a second round, whose loads are issued behind the first's stores, for
// few threads' work; blocks of up to 512 threads in equal rounds took 11.9 us a call instead of 11.1.  A block
// takes whole rows: its threads load their values, then form the rows' (cos, sin) table in LDS, each pair once for all heads
// (a thread per pair and head would spend more on angles than on memory), then rotate and store.
#pragma once
#include <algorithm>

#include "sp_device.h"
#include "../../include/seedplane_hip.h"

namespace paged {

typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------------------------------------ values <-> fp32
template <class T, int N>
__device__ __forceinline__ void load_values(const T *p, float *v) {
    if constexpr (N == 1) {
        v[0] = (float)p[0];
    } else if constexpr (sizeof(T) == 4) {
        *(f32x4 *)v = *(const f32x4 *)p;
        *(f32x4 *)(v + 4) = *(const f32x4 *)(p + 4);
    } else {
        typedef T T8 __attribute__((ext_vector_type(8)));
        const T8 x = *(const T8 *)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    }
}

// fp32 -> OCP e4m3, nearest even, saturated at 448 (the conversion itself turns larger values into NaN); NaN stays NaN.
__device__ __forceinline__ float e4m3_clamp(float x) { return x > 448.f ? 448.f : x < -448.f ? -448.f : x; }
__device__ __forceinline__ uint32_t e4m3_pack4(const float *v) {
    uint32_t p = 0;
    p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(v[0]), e4m3_clamp(v[1]), p, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(v[2]), e4m3_clamp(v[3]), p, true);
}

// N fp32 values to element `at` of an array of type dt (SP_DT_*).
template <int N>
__device__ __forceinline__ void store_values(void *p, int64_t at, int dt, const float *v) {
    if (dt == SP_DT_F32) {
        float *d = (float *)p + at;
        if constexpr (N == 1) d[0] = v[0];
        else { *(f32x4 *)d = *(const f32x4 *)v; *(f32x4 *)(d + 4) = *(const f32x4 *)(v + 4); }
    } else if (dt == SP_DT_F16) {
        f16 *d = (f16 *)p + at;
        if constexpr (N == 1) d[0] = (f16)v[0];
        else {
            f16x8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (f16)v[i];
            *(f16x8 *)d = x;
        }
    } else if (dt == SP_DT_BF16) {
        bf16 *d = (bf16 *)p + at;
        if constexpr (N == 1) d[0] = (bf16)v[0];
        else {
            bf16x8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (bf16)v[i];
            *(bf16x8 *)d = x;
        }
    } else {
        uint8_t *d = (uint8_t *)p + at;
        if constexpr (N == 1) {
            d[0] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(v[0]), 0.f, 0u, false);
        } else {
            *(u32x2 *)d = (u32x2){e4m3_pack4(v), e4m3_pack4(v + 4)};
        }
    }
}

// ------------------------------------------------------------------------------------------------ rotation
struct Rotation {
    const double *inv;      // [rot / 2] radians per position
    int rot, pairs;         // rotated values of a head; 1: interleaved pairs
    float factor;           // on cosines and sines
};

// (cos, sin) of pair j at position p
__device__ __forceinline__ float2 turn_of(const Rotation &r, int p, int j) {
    const double t = (double)p * r.inv[j] * 0.15915494309189533577;          // in turns
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    return make_float2(c * r.factor, s * r.factor);
}

// A unit is VEC pairs of one head: two vectors of VEC values, at at1 and at2 of the head.
template <int VEC>
__device__ __forceinline__ void unit_offsets(const Rotation &r, int u, int &at1, int &at2) {
    at1 = r.pairs ? 2 * u * VEC : u * VEC;
    at2 = r.pairs ? at1 + VEC : (r.rot >> 1) + at1;
}
template <int VEC>
__device__ __forceinline__ void turn_unit(const Rotation &r, const float2 *cs, float *a, float *b) {
    if (!r.pairs || VEC == 1) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float2 t = cs[i];
            const float x = a[i], y = b[i];
            a[i] = x * t.x - y * t.y;
            b[i] = y * t.x + x * t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 t = cs[i / 2], w = cs[(VEC + i) / 2];
            const float x = a[i], y = a[i + 1], z = b[i], q = b[i + 1];
            a[i] = x * t.x - y * t.y;
            a[i + 1] = y * t.x + x * t.y;
            b[i] = z * w.x - q * w.y;
            b[i + 1] = q * w.x + z * w.y;
        }
    }
}

constexpr int ROT_THREADS = 256;

// n / d for n, d < 2^16 by a multiplication: the rounded-up reciprocal is off by less than 2^-32 d, so n times it is off by
// less than one part of d.
struct Divisor {
    uint32_t inverse, d;
    Divisor() = default;
    explicit Divisor(int v) : inverse((uint32_t)((((uint64_t)1 << 32) + v - 1) / std::max(v, 1))), d(v) {}
};
__device__ __forceinline__ int operator/(int n, Divisor v) { return v.d == 1 ? n : (int)__umulhi((uint32_t)n, v.inverse); }

struct RotateArgs {
    Rotation rot;
    const void *x;
    void *out;
    int64_t x_row, x_head, out_row, out_head;    // elements
    const int *pos;
    int rows, heads, per_block;                  // rows per block
    int units, per_head, per_row;                // units of a head's rotated part; with the vectors of its rest (none in place)
    Divisor by_row, by_head, by_half;
};

// Angles of the block's rows: cs [n][rot / 2]
__device__ __forceinline__ void turn_rows(const Rotation &rot, const int *pos, int n, Divisor by_half, float2 *cs) {
    const int half = rot.rot >> 1;
    for (int k = threadIdx.x; k < n * half; k += blockDim.x) {
        const int r = k / by_half;
        cs[k] = turn_of(rot, pos[r], k - r * half);
    }
}

template <class T> constexpr int dtype_of() { return sizeof(T) == 4 ? SP_DT_F32 : std::is_same<T, f16>::value ? SP_DT_F16 : SP_DT_BF16; }

template <class T, int VEC>
__global__ void __launch_bounds__(ROT_THREADS) k_rotate(RotateArgs a) {
    extern __shared__ __align__(16) unsigned char rot_smem[];
    float2 *cs = (float2 *)rot_smem;
    const int row0 = blockIdx.x * a.per_block, n = min(a.per_block, a.rows - row0), half = a.rot.rot >> 1;
    const int total = n * a.per_row;
    float v1[VEC], v2[VEC];
    int at1 = 0, at2 = 0, r = 0, head = 0, u = 0;
    // (the unrotated rest has one vector: v2 repeats it and is not stored; a load under a condition would put the vectors into
    // scratch memory: 20.1 us instead of 8.3 for 2048 rows x 32 heads)
    auto fetch = [&](int i) {
        r = i / a.by_row;
        const int k = i - r * a.per_row;
        head = k / a.by_head;
        u = k - head * a.per_head;
        unit_offsets<VEC>(a.rot, u, at1, at2);
        if (u >= a.units) at1 = at2 = a.rot.rot + (u - a.units) * VEC;
        const T *src = (const T *)a.x + (int64_t)(row0 + r) * a.x_row + (int64_t)head * a.x_head;
        load_values<T, VEC>(src + at1, v1);
        load_values<T, VEC>(src + at2, v2);
    };
    int i = threadIdx.x;
    if (i < total) fetch(i);
    turn_rows(a.rot, a.pos + row0, n, a.by_half, cs);
    __syncthreads();
    while (i < total) {
        const int64_t to = (int64_t)(row0 + r) * a.out_row + (int64_t)head * a.out_head;
        if (u < a.units) {
            turn_unit<VEC>(a.rot, cs + r * half + u * VEC, v1, v2);
            store_values<VEC>(a.out, to + at2, dtype_of<T>(), v2);
        }
        store_values<VEC>(a.out, to + at1, dtype_of<T>(), v1);
        i += blockDim.x;
        if (i < total) fetch(i);
    }
}

// ------------------------------------------------------------------------------------------------ append
struct AppendArgs {
    Rotation rot;                                // rot.rot 0: none
    const void *q, *k, *v;                       // q may be NULL (nq 0)
    void *q_out, *kc, *vc;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head;
    const float *ks, *vs;                        // e4m3: scale per K/V head
    const int *pos, *seq, *at, *table;           // rotation position, sequence, cached position of a row; [n_seq][max_pages]
    int rows, nq, nkv, hd, qo_dt, kv_dt, per_block;
    int n_seq, max_pages, n_pages, page_size;
    int64_t page_stride, head_stride, row_stride;
    int units, tail, vecs;                       // of a head: rotated units, vectors of the rest, vectors of a value
    int turned, rest, per_row;                   // units of a row: rotated, unrotated rests of queries and keys, all
    Divisor by_row, by_units, by_tail, by_vecs, by_half;
};

// Units of a row: the rotated parts of the query and key heads, their unrotated rests, the value heads.  A row whose
// sequence, position or page is out of range writes nothing.
template <class T, int VEC>
__global__ void __launch_bounds__(ROT_THREADS) k_append(AppendArgs a) {
    extern __shared__ __align__(16) unsigned char rot_smem[];
    int64_t *dst = (int64_t *)rot_smem;                                // [rows of the block]: element offset in the pools, or -1
    float2 *cs = (float2 *)(dst + a.per_block);                        // [rows of the block][rot / 2]
    const int row0 = blockIdx.x * a.per_block, n = min(a.per_block, a.rows - row0), half = a.rot.rot >> 1;
    const int total = n * a.per_row;
    float v1[VEC], v2[VEC];
    int at1 = 0, at2 = 0, r = 0, head = 0, u = 0;
    bool two = false;                                                  // a rotated unit (else v2 repeats v1 and is not stored)
    auto fetch = [&](int i) {
        r = i / a.by_row;
        int k = i - r * a.per_row;
        const int64_t row = row0 + r;
        const T *src;
        two = k < a.turned;
        if (k < a.turned + a.rest) {
            if (two) {
                head = k / a.by_units;
                u = k - head * a.units;
                unit_offsets<VEC>(a.rot, u, at1, at2);
            } else {
                k -= a.turned;
                head = k / a.by_tail;
                at1 = at2 = a.rot.rot + (k - head * a.tail) * VEC;
            }
            src = head < a.nq ? (const T *)a.q + row * a.q_row + (int64_t)head * a.q_head
                              : (const T *)a.k + row * a.k_row + (int64_t)(head - a.nq) * a.k_head;
        } else {
            k -= a.turned + a.rest;
            head = k / a.by_vecs;
            at1 = at2 = (k - head * a.vecs) * VEC;
            src = (const T *)a.v + row * a.v_row + (int64_t)head * a.v_head;
            head += a.nq + a.nkv;
        }
        load_values<T, VEC>(src + at1, v1);
        load_values<T, VEC>(src + at2, v2);
    };
    int i = threadIdx.x;
    if (i < total) fetch(i);
    // (the places are looked up by the last threads, the angles formed by the first)
    for (int k = blockDim.x - 1 - threadIdx.x; k < n; k += blockDim.x) {
        const int s = a.seq[row0 + k], p = a.at[row0 + k];
        int64_t to = -1;
        if (s >= 0 && s < a.n_seq && p >= 0 && p / a.page_size < a.max_pages) {
            const int e = a.table[(int64_t)s * a.max_pages + p / a.page_size];
            if (e >= 0 && e < a.n_pages) to = e * a.page_stride + (p % a.page_size) * a.row_stride;
        }
        dst[k] = to;
    }
    turn_rows(a.rot, a.pos + row0, n, a.by_half, cs);
    __syncthreads();
    while (i < total) {
        const int64_t to = dst[r];
        if (to >= 0) {
            if (two) turn_unit<VEC>(a.rot, cs + r * half + u * VEC, v1, v2);
            if (head < a.nq) {
                const int64_t o = (int64_t)(row0 + r) * a.qo_row + (int64_t)head * a.qo_head;
                store_values<VEC>(a.q_out, o + at1, a.qo_dt, v1);
                if (two) store_values<VEC>(a.q_out, o + at2, a.qo_dt, v2);
            } else {
                const bool key = head < a.nq + a.nkv;
                const int h = head - a.nq - (key ? 0 : a.nkv);
                if (a.kv_dt == SP_DT_E4M3) {
                    const float scale = (key ? a.ks : a.vs)[h];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) { v1[j] /= scale; v2[j] /= scale; }
                }
                const int64_t o = to + h * a.head_stride;
                store_values<VEC>(key ? a.kc : a.vc, o + at1, a.kv_dt, v1);
                if (two) store_values<VEC>(key ? a.kc : a.vc, o + at2, a.kv_dt, v2);
            }
        }
        i += blockDim.x;
        if (i < total) fetch(i);
    }
}

}  // namespace paged
