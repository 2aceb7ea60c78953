// Beam search's selection: of each request's beams, the n best continuations by score + log softmax(logits).
//
// A beam's order of continuations is its logits' order, so the softmax's sum is needed only to compare beams: one pass over the logits
// takes the maximum, the sum of exponentials and the n best of a part of a row together (k_beam_rows), and a second, small launch
// forms the sums' logarithms, compares totals in 64 bits and writes the results in order (k_beam_merge).  Ties go to the lowest beam,
// then token.
//
// The n best of a part: a block's waves take 8 values a thread at a time.  From the first chunk a border that at least n of its
// values reach is known (each of 8 waves has ceil(n / 8) threads whose largest value does); values on the good side of it go to a
// buffer in LDS, and when the buffer fills, its exact n best stay and the n-th becomes the border.  Later chunks bring few: a value
// reaches the n best of what came before it n / (position) of the time.
#pragma once
#include "sp_device.h"
#include "sp_rotate.h"

namespace beam {

using paged::bf16;

constexpr int THREADS = 512, WAVES = THREADS / 64, VALUES = 8, CHUNK = THREADS * VALUES;
constexpr int MOST_N = 64, MOST_BEAMS = 64, MOST_EOS = 8, MOST_SPLITS = 64, LEAST_SPLITS = 4;
constexpr int KEPT = 256;                  // entries of the buffer from which it is cut back to n
constexpr int CAPACITY = KEPT + THREADS;   // one value of every thread fits behind them
constexpr int LISTS = 512;                 // parts of a request's rows at most (splits are chosen so)

struct Entry { float v; int i; };          // value, token
struct Args {
    const void *logits;
    int64_t ld;
    const float *scores;                   // [B][K]
    int B, K, V, n, splits, len;           // len: values of a part
    Entry *best;                           // [B K][splits][n], best first; i -1: none
    float2 *sums;                          // [B K][splits]: maximum, sum of exponentials
    float *out_score, *next_score;
    int *out_beam, *out_token, *next_row, *next_token;
    int eos[MOST_EOS], n_eos;
};

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }
__device__ __forceinline__ bool alive(float score) { return score > -INFINITY; }       // (NaN: no)

struct RowShared {
    Entry buf[CAPACITY], top[MOST_N];
    int count, overflow;
    float border[WAVES];
    float2 sum[WAVES];
};

// The exact n best of the buffer's count entries, in order, to its front.  Every thread calls; ends with a barrier.
__device__ __forceinline__ int cut(RowShared &sh, int count, int n, float &bv, int &bi) {
    for (int e = threadIdx.x; e < count; e += THREADS) {
        const Entry x = sh.buf[e];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += better(sh.buf[j].v, sh.buf[j].i, x.v, x.i);
        if (rank < n) sh.top[rank] = x;
    }
    __syncthreads();
    const int left = min(count, n);
    if ((int)threadIdx.x < left) sh.buf[threadIdx.x] = sh.top[threadIdx.x];
    if (threadIdx.x == 0) sh.count = left;
    if (count >= n) { bv = sh.top[n - 1].v; bi = sh.top[n - 1].i; }
    __syncthreads();
    return left;
}

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) k_beam_rows(Args a) {
    __shared__ RowShared sh;
    const int split = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int lo = split * a.len, hi = min(a.V, lo + a.len);
    Entry *const best = a.best + ((int64_t)row * a.splits + split) * a.n;
    if (!alive(a.scores[row]) || lo >= hi) {
        if (tid < a.n) best[tid] = {-INFINITY, -1};
        if (tid == 0) a.sums[(int64_t)row * a.splits + split] = make_float2(-INFINITY, 0.f);
        return;
    }
    const T *const x = (const T *)a.logits + row * a.ld;
    auto fetch = [&](int at, float (&v)[VALUES]) {
        if (ALIGNED && at + VALUES <= hi) {
            paged::load_values<T, VALUES>(x + at, v);
        } else {
#pragma unroll
            for (int j = 0; j < VALUES; ++j) v[j] = at + j < hi ? (float)x[at + j] : -INFINITY;
        }
    };
    if (tid == 0) { sh.count = 0; sh.overflow = 0; }
    float next[VALUES], v[VALUES];
    fetch(lo + tid * VALUES, next);
    float m = -INFINITY, s = 0.f;
    float bv = -INFINITY;                                              // a value is taken if it is better than (bv, bi)
    int bi = -1, kept = 0;
    for (int c = lo; c < hi; c += CHUNK) {
        const int at = c + tid * VALUES;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) v[j] = next[j];
        if (c + CHUNK < hi) fetch(at + CHUNK, next);
        float top = v[0];
#pragma unroll
        for (int j = 1; j < VALUES; ++j) top = fmaxf(top, v[j]);
        if (top > m) {
            s *= __builtin_amdgcn_exp2f((m - top) * 1.4426950408889634f);
            m = top;
        }
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) s += __builtin_amdgcn_exp2f((v[j] - base) * 1.4426950408889634f);
        if (c == lo) {
            // each wave's ceil(n / WAVES)-th largest of its threads' largest values; the least of the waves'
            float mine = top, w = -INFINITY;
            for (int k = 0; k < a.n; k += WAVES) {
                w = wave_max_dpp(mine);
                const uint64_t who = __ballot(mine == w);
                if (who && lane == __builtin_ctzll(who)) mine = -INFINITY;
            }
            if (lane == 0) sh.border[wv] = w;
            __syncthreads();
            bv = sh.border[0];
#pragma unroll
            for (int k = 1; k < WAVES; ++k) bv = fminf(bv, sh.border[k]);
            bi = bv == -INFINITY ? -1 : 0x7fffffff;
        }
        int mine = 0;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) mine += better(v[j], at + j, bv, bi);
        if (mine) {
            int to = atomicAdd(&sh.count, mine);
            if (to + mine > CAPACITY) {
                sh.overflow = 1;
            } else {
#pragma unroll
                for (int j = 0; j < VALUES; ++j)
                    if (better(v[j], at + j, bv, bi)) sh.buf[to++] = {v[j], at + j};
            }
        }
        __syncthreads();
        const bool over = sh.overflow;
        int count = sh.count;
        __syncthreads();
        if (over) {                                                    // the chunk again, one value of each thread at a time
            if (tid == 0) { sh.count = kept; sh.overflow = 0; }
            __syncthreads();
#pragma unroll 1
            for (int j = 0; j < VALUES; ++j) {
                float mine = v[0];
#pragma unroll
                for (int k = 1; k < VALUES; ++k) mine = j == k ? v[k] : mine;
                if (better(mine, at + j, bv, bi)) sh.buf[atomicAdd(&sh.count, 1)] = {mine, at + j};
                __syncthreads();
                count = sh.count;
                __syncthreads();
                if (count > KEPT) count = cut(sh, count, a.n, bv, bi);
            }
        } else if (count > KEPT) {
            count = cut(sh, count, a.n, bv, bi);
        }
        kept = count;
    }
    kept = cut(sh, kept, a.n, bv, bi);
    if (tid < a.n) best[tid] = tid < kept ? sh.buf[tid] : Entry{-INFINITY, -1};
    // the part's maximum and sum
    const float wm = wave_max_dpp(m), wbase = wm == -INFINITY ? 0.f : wm;
    const float ws = wave_sum_dpp(s * __builtin_amdgcn_exp2f((m - wbase) * 1.4426950408889634f));
    if (lane == 0) sh.sum[wv] = make_float2(wm, ws);
    __syncthreads();
    if (tid == 0) {
        float M = sh.sum[0].x, S = 0.f;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) M = fmaxf(M, sh.sum[k].x);
        const float b = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) S += sh.sum[k].y * __builtin_amdgcn_exp2f((sh.sum[k].x - b) * 1.4426950408889634f);
        a.sums[(int64_t)row * a.splits + split] = make_float2(M, S);
    }
}

// ------------------------------------------------------------------------------------------------ merge
struct Total { double v; int64_t i; };     // score, beam V + token
__device__ __forceinline__ bool better(const Total &x, const Total &y) { return x.v > y.v || (x.v == y.v && x.i < y.i); }

struct MergeShared {
    // a continuation's total is (logit - top) + shift: 64 bits would lose the shift beside a type's lowest values
    double top[MOST_BEAMS], shift[MOST_BEAMS];      // largest logit; score - log of the sum, NaN: a beam without continuations
    Total head[LISTS], border, out[MOST_N];
    int good[MOST_N];
    int count;
    Total buf[MOST_N * MOST_N];            // at most n lists have a head at or before the border, of n entries each
};

__global__ void __launch_bounds__(THREADS) k_beam_merge(Args a) {
    extern __shared__ __align__(16) unsigned char merge_smem[];
    MergeShared &sh = *(MergeShared *)merge_smem;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t row0 = (int64_t)b * a.K;
    for (int k = wv; k < a.K; k += WAVES) {
        // (splits are at most a wave's lanes)
        const float2 p = lane < a.splits ? a.sums[(row0 + k) * a.splits + lane] : make_float2(-INFINITY, 0.f);
        float bad = p.x != p.x || !(p.y < INFINITY) || p.x == INFINITY ? 1.f : 0.f;
        bad = wave_max_dpp(bad);
        const float M = wave_max_dpp(p.x);
        double s = M > -INFINITY ? (double)p.y * exp((double)p.x - (double)M) : 0.0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) {
            const float score = a.scores[row0 + k];
            sh.top[k] = (double)M;
            sh.shift[k] = bad > 0.f || !(s > 0.0) || !alive(score) ? (double)NAN : (double)score - log(s);
        }
    }
    if (tid == 0) { sh.count = 0; sh.border = {-INFINITY, -1}; }
    __syncthreads();
    const int lists = a.K * a.splits;
    const Entry *const best = a.best + row0 * a.splits * a.n;
    auto total_of = [&](int list, int j) -> Total {
        const int k = list / a.splits;
        const Entry e = best[(int64_t)list * a.n + j];
        const double v = ((double)e.v - sh.top[k]) + sh.shift[k];
        return e.i < 0 || v != v ? Total{-INFINITY, -1} : Total{v, (int64_t)k * a.V + e.i};
    };
    for (int l = tid; l < lists; l += THREADS) {
        Total h = total_of(l, 0);
        if (h.i < 0) h.i = ((int64_t)1 << 62) + l;                     // lists without entries come last, in a definite order
        sh.head[l] = h;
    }
    __syncthreads();
    for (int l = tid; l < lists; l += THREADS) {
        const Total h = sh.head[l];
        int rank = 0;
        for (int j = 0; j < lists; ++j) rank += better(sh.head[j], h);
        if (rank < a.n) sh.good[rank] = l;
        if (rank == a.n - 1 && h.v > -INFINITY) sh.border = h;
    }
    __syncthreads();
    const int lists_in = min(lists, a.n);
    const Total border = sh.border;
    for (int e = tid; e < lists_in * a.n; e += THREADS) {
        const int g = e / a.n;
        const Total t = total_of(sh.good[g], e - g * a.n);
        if (t.v > -INFINITY && !better(border, t)) sh.buf[atomicAdd(&sh.count, 1)] = t;
    }
    __syncthreads();
    const int count = sh.count, found = min(count, a.n);
    for (int e = tid; e < count; e += THREADS) {
        const Total t = sh.buf[e];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += better(sh.buf[j], t);
        if (rank < a.n) sh.out[rank] = t;
    }
    __syncthreads();
    if (wv != 0) return;
    // one wave: place i of the n best, and those among them that go on
    const bool have = lane < found;
    const Total t = have ? sh.out[lane] : Total{-INFINITY, -1};
    const int beam = have ? (int)(t.i / a.V) : -1, token = have ? (int)(t.i - (int64_t)beam * a.V) : -1;
    if (lane < a.n) {
        const int64_t o = (int64_t)b * a.n + lane;
        a.out_score[o] = (float)t.v;
        a.out_beam[o] = beam;
        a.out_token[o] = token;
    }
    bool on = have;
    for (int k = 0; k < a.n_eos; ++k) on &= token != a.eos[k];
    const uint64_t going = __ballot(on);
    const int at = __popcll(going & (((uint64_t)1 << lane) - 1)), n = min(__popcll(going), a.K);
    if (on && at < a.K) {
        const int64_t o = row0 + at;
        a.next_score[o] = (float)t.v;
        a.next_row[o] = (int)(row0 + beam);
        a.next_token[o] = token;
    }
    if (lane >= n && lane < a.K) {
        const int64_t o = row0 + lane;
        a.next_score[o] = -INFINITY;
        a.next_row[o] = -1;
        a.next_token[o] = -1;
    }
}

}  // namespace beam
