// Beam search's selection: of each request's beams, the n best continuations by score + log softmax(logits).
//
// A beam's order of continuations is its logits' order, so the softmax's sum is needed only to compare beams: one pass over the logits
// takes the maximum, the sum of exponentials and the n best of a part of a row together (k_beam_rows), and a second, small launch
// forms the sums' logarithms, compares totals in 64 bits and writes the results in order (k_beam_merge).  Ties go to the lowest beam,
// then token.  The sums of a part are held in 32 bits, at most V / 1024 + 40 terms after each other, off by 2^-24 of the sum each at most: the
// same for all continuations of a beam, so that only beams whose totals lie closer than that may change places (64 bits would be a conversion and
// a 64-bit sum more for each logit).
//
// The n best of a part: each thread streams its values, keeping their largest beside the sum.  The largest of all threads give a border
// that at least n values reach and few others (each of 4 waves has ceil(n / 4) threads at or above it: about 2 n values of a part);
// the few threads that have such values are listed, their values read once more by the whole block, and what reaches the border is put in order.
// The stream has no barrier, no LDS and nothing but a maximum and an exponential for each value.  Where more values reach the border than
// the buffer holds (masks of a type's lowest value, padded vocabularies, ordered rows), borders with a token follow until they fit.
//
// What bounds it: few rows, the two launches' chains (4 beams x 151936 in fp32: 6.5 + 4.8 us); many, the stream: 256 rows in bf16, 78 MB, take
// 22.4 us of which 15.3 are the bytes at a large copy's rate, 43 to 54 if masked to the lowest value, padded or ordered (by single values
// past a border, in order, 546 to 666); the blocks all run at once, and what each does behind its stream (border, the
// few values again, their order) has no other's stream beside it, but more blocks cost more than that (4096 33.9, 8192 42.8 us a call
// against 29.8 by 2048; 1024 blocks of 512 threads 33.7).  With a buffer in LDS that took every value past a running border, chunk by chunk
// between barriers, the call took 51 us.
#pragma once
#include "sp_device.h"
#include "sp_rotate.h"

namespace beam {

using paged::bf16;

constexpr int THREADS = 256, WAVES = THREADS / 64, VALUES = 8, CHUNK = THREADS * VALUES;
constexpr int MERGE_THREADS = 512, MERGE_WAVES = MERGE_THREADS / 64;
constexpr int MOST_N = 64, MOST_BEAMS = 64, MOST_EOS = 8, MOST_SPLITS = 64, LEAST_SPLITS = 4;
constexpr int AHEAD = 2;                   // vectors of a thread in flight
constexpr int CAPACITY = THREADS;          // entries of the buffer
constexpr int LISTS = MERGE_THREADS;       // parts of a request's rows at most (splits are chosen so)
constexpr int MERGED = 512;                // entries that the merge puts in order at once

struct Entry { float v; int i; };          // value, token
struct Args {
    const void *logits;
    int64_t ld;
    const float *scores;                   // [B][K]
    int B, K, V, n, splits, len;           // len: values of a part
    Entry *best;                           // [B K][splits][n], best first; i -1: none
    float2 *sums;                          // [B K][splits]: m, the largest value, and sum e^(v - m)
    float *out_score, *next_score;
    int *out_beam, *out_token, *next_row, *next_token;
    int eos[MOST_EOS], n_eos;
    paged::Divisor by_splits, by_n;
};

// A value and its token as one number that grows with the value, then with lower tokens (v + 0: zeros are equal).
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    const uint32_t u = __float_as_uint(v + 0.f);
    return (uint64_t)(u ^ (uint32_t)((int)u >> 31 | 0x80000000)) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ Entry entry_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return {__uint_as_float(u ^ (u >> 31 ? 0x80000000u : ~0u)), (int)~(uint32_t)key};
}
__device__ __forceinline__ bool alive(float score) { return score > -INFINITY; }       // (NaN: no)

constexpr float LOG2E = 1.4426950408889634f;

// The n-th largest of a wave's values (-infinity: there are fewer).  A border for more than the wave has only to be reached by n values,
// so NaNs, which fmaxf leaves out, do not matter.
// (A turn for each takes 0.12 us, comparing every lane's value with all others' 0.5.)
__device__ __forceinline__ float nth_of_wave(float mine, int n) {
    if (n <= 4) {
        float w = -INFINITY;
        for (int k = 0; k < n; ++k) {
            w = wave_max_dpp(mine);
            const uint64_t who = __ballot(mine == w);
            if (who && (int)(threadIdx.x & 63) == __builtin_ctzll(who)) mine = -INFINITY;
        }
        return w;
    }
    int above = 0;
#pragma unroll
    for (int k = 0; k < 64; ++k) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), k)) > mine;
    return -wave_max_dpp(above < n ? -mine : -INFINITY);
}

struct RowShared {
    __align__(16) uint64_t buf[CAPACITY], own[THREADS];
    uint64_t top[MOST_N];
    int count, threads, who[THREADS];
    float border[WAVES];
    float2 sum[WAVES];
};

// The n best of count keys (room for THREADS of them) in order to top.  Every thread calls; begins and ends with a barrier.
__device__ __forceinline__ void put_in_order(uint64_t *keys, int count, uint64_t *top, int n) {
    const int tid = threadIdx.x;
    if (count <= THREADS / 4) {                                        // 4 threads a key
        __syncthreads();
        if (tid / 4 < count) {
            const uint64_t x = keys[tid / 4];
            int rank = 0;
#pragma unroll 4
            for (int j = tid & 3; j < count; j += 4) rank += keys[j] > x;
            rank += __shfl_xor(rank, 1);
            rank += __shfl_xor(rank, 2);
            if ((tid & 3) == 0 && rank < n) top[rank] = x;
        }
    } else {
        if (tid == 0 && count % 2) keys[count] = 0;
        __syncthreads();
        const uint64_t x = keys[tid];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; j += 2) {
            const ulonglong2 y = *(const ulonglong2 *)(keys + j);
            rank += (y.x > x) + (y.y > x);
        }
        if (tid < count && rank < n) top[rank] = x;
    }
    __syncthreads();
}

// SHORT: rows of fewer values than a vector.
template <class T, bool SHORT>
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
    // A vector past the part's end is read from its last 8 values, and those before its own first are hidden: one load without a
    // branch, wherever rows begin.
    typedef T Vector __attribute__((ext_vector_type(VALUES), aligned(sizeof(T))));
    auto place = [&](int own) { return SHORT ? own : min(own, hi - VALUES); };
    auto fetch = [&](int own) -> Vector {
        if constexpr (!SHORT) return *(const Vector *)(x + place(own));
        Vector v;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) v[j] = own + j < hi ? x[own + j] : (T)-INFINITY;
        return v;
    };
    auto values = [&](const Vector &raw, int own, float (&v)[VALUES]) {
        const int hidden = own - place(own);
#pragma unroll
        for (int j = 0; j < VALUES; ++j) v[j] = (float)raw[j];
        if (hidden > 0) {
#pragma unroll
            for (int j = 0; j < VALUES; ++j) v[j] = j < hidden ? -INFINITY : v[j];
        }
    };
    if (tid == 0) { sh.count = 0; sh.threads = 0; }
    // the thread's values: the largest, sum e^(v - m); AHEAD vectors at a time
    float m = -INFINITY, s = 0.f;
    for (int c = lo + tid * VALUES; c < hi; c += AHEAD * CHUNK) {
        Vector raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) raw[u] = fetch(c + u * CHUNK);
        float v[AHEAD][VALUES], top = m;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            values(raw[u], c + u * CHUNK, v[u]);
#pragma unroll
            for (int j = 0; j < VALUES; ++j) top = fmaxf(top, v[u][j]);
        }
        const float base = top == -INFINITY ? 0.f : top;
        s *= __builtin_amdgcn_exp2f((m - base) * LOG2E);
        m = top;
        // (a fused v LOG2E - m would save an instruction, but leave fp32's range for a type's lowest values)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int j = 0; j < VALUES; ++j) s += __builtin_amdgcn_exp2f((v[u][j] - base) * LOG2E);
    }
    // A border that at least n values reach: ceil(n / waves) threads of every wave whose lanes all have a value, or, where some wave has
    // too few, n threads of one wave.
    const int waves = min(hi - lo, CHUNK) / (64 * VALUES);
    float bv = -INFINITY;
    if (waves > 0) {                                                   // (a part of fewer, 511 values at most, is listed whole: past 256 see below)
        float w = nth_of_wave(m, (a.n + waves - 1) / waves);
        if (lane == 0) sh.border[wv] = w;
        __syncthreads();
        bv = sh.border[0];
        for (int k = 1; k < waves; ++k) bv = fminf(bv, sh.border[k]);
        if (bv == -INFINITY) {
            __syncthreads();
            w = nth_of_wave(m, a.n);
            if (lane == 0) sh.border[wv] = w;
            __syncthreads();
            for (int k = 0; k < waves; ++k) bv = fmaxf(bv, sh.border[k]);
        }
    } else {
        __syncthreads();
    }
    // (past the buffer's end only that there are more matters)
    auto full = [&]() { return __hip_atomic_load(&sh.count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) > CAPACITY; };
    // a vector's values from the border (its token: the last one of equal values) to the buffer
    auto collect = [&](const Vector &raw, int own, float border, int token) {
        float v[VALUES];
        values(raw, own, v);
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < VALUES; ++j)
            mine |= (uint32_t)(v[j] > -INFINITY && (v[j] > border || (v[j] == border && place(own) + j <= token))) << j;
        if (!mine || full()) return;
        int to = atomicAdd(&sh.count, __popc(mine));
#pragma unroll
        for (int j = 0; j < VALUES; ++j)
            if ((mine >> j & 1) && to < CAPACITY) sh.buf[to++] = key_of(v[j], place(own) + j);
    };
    // the threads that have such values, and their vectors again, one a thread
    if (m >= bv && m > -INFINITY) sh.who[atomicAdd(&sh.threads, 1)] = tid;
    __syncthreads();
    const int listed = sh.threads, vectors = listed * ((hi - lo + CHUNK - 1) / CHUNK);
    for (int e = tid; e < vectors && !full(); e += THREADS) {
        const int c = e / listed, own = lo + c * CHUNK + sh.who[e - c * listed] * VALUES;
        if (own < hi) collect(fetch(own), own, bv, a.V);
    }
    __syncthreads();
    // Equal values, or the best side by side, may be more than that.  The n-th best of the threads' best (values, then tokens) leaves those of
    // n threads at most, few of each; if that is not few enough, or not n threads have a value, the n-th best of those in the buffer leaves
    // fewer every time.
    int kept = sh.count;
    for (bool first = true; kept > CAPACITY; first = false) {
        uint64_t last = 0;
        if (first) {
            int token = -1;
            for (int c = lo + tid * VALUES; m > -INFINITY && token < 0 && c < hi; c += CHUNK) {
                float v[VALUES];
                values(fetch(c), c, v);
#pragma unroll
                for (int j = VALUES - 1; j >= 0; --j) token = v[j] == m ? place(c) + j : token;
            }
            sh.own[tid] = token < 0 ? 0 : key_of(m, token);
            if (tid < a.n) sh.top[tid] = 0;
            put_in_order(sh.own, THREADS, sh.top, a.n);
            last = sh.top[a.n - 1];
        }
        if (last == 0) {
            __syncthreads();
            put_in_order(sh.buf, CAPACITY, sh.top, a.n);
            last = sh.top[a.n - 1];
        }
        const Entry border = entry_of(last);
        if (tid == 0) sh.count = 0;
        __syncthreads();
        if (m >= border.v)
            for (int c = lo + tid * VALUES; c < hi && !full(); c += AHEAD * CHUNK) {
                Vector raw[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) raw[u] = fetch(c + u * CHUNK);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) collect(raw[u], c + u * CHUNK, border.v, border.i);
            }
        __syncthreads();
        kept = sh.count;
    }
    put_in_order(sh.buf, kept, sh.top, a.n);
    if (tid < a.n) best[tid] = tid < kept ? entry_of(sh.top[tid]) : Entry{-INFINITY, -1};
    // the part's maximum and sum
    const float wm = wave_max_dpp(m);
    const float ws = wave_sum_dpp(s * __builtin_amdgcn_exp2f((m - (wm == -INFINITY ? 0.f : wm)) * LOG2E));
    if (lane == 0) sh.sum[wv] = make_float2(wm, ws);
    __syncthreads();
    if (tid == 0) {
        float M = sh.sum[0].x, S = 0.f;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) M = fmaxf(M, sh.sum[k].x);
        const float b = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) S += sh.sum[k].y * __builtin_amdgcn_exp2f((sh.sum[k].x - b) * LOG2E);
        a.sums[(int64_t)row * a.splits + split] = make_float2(M, S);
    }
}

// ------------------------------------------------------------------------------------------------ merge
struct Total {
    double v;
    uint64_t at;                           // beam, token
    __device__ int beam() const { return (int)(at >> 32); }
    __device__ int token() const { return (int)(uint32_t)at; }
};
__device__ __forceinline__ bool better(const Total &x, const Total &y) { return (x.v > y.v) | ((x.v == y.v) & (x.at < y.at)); }
constexpr Total NONE = {-INFINITY, ~0ull};

struct MergeShared {
    // a continuation's total is (logit - top) + shift: 64 bits would lose the shift beside a type's lowest values
    double top[MOST_BEAMS], shift[MOST_BEAMS];      // largest logit; score - log of the sum, NaN: a beam without continuations
    float border[MERGE_WAVES];
    int lists, count, good[LISTS];
    Total out[MOST_N], buf[MERGED];
};

// One block a request.  The parts' lists are in order, so a list whose first entry is behind the border has nothing to give.  For the border
// wave w takes totals number d = 2^w of all lists, rounded to fp32 (which keeps their order): where ceil(n / d) lists have theirs at
// or above a value, n totals are.  The largest such value is the border, and few more than n pass it, whether all beams are about as good or one
// has nearly all of the best (by the lists' first totals alone: 32 x 16 beams, n 32, 146 us instead of 9; 64 beams, n 64, 173 instead of 23).
// Rows of many parts spread their best over many lists: then the first totals are enough, of which each wave has an eighth (1 x 8 beams,
// n 16, 64 parts: 6.2 us instead of 8.1).  The least of the waves' borders counts, so lists of other waves may pass beyond the n best; where a
// wave's parts are all masked every list does, with n totals each, which come to the buffer by turns (1 beam of 64 parts, n 16, every eighth
// masked: 11.9 us, none 5.5), hence not for large n.
__global__ void __launch_bounds__(MERGE_THREADS) k_beam_merge(Args a) {
    __shared__ MergeShared sh;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t row0 = (int64_t)b * a.K;
    const int lists = a.K * a.splits;                                  // at most LISTS: one a thread
    const Entry *const best = a.best + row0 * a.splits * a.n;
    const int list = lane * MERGE_WAVES + wv, beam = list / a.by_splits;       // (every wave has some of them)
    const Entry head = list < lists ? best[(int64_t)list * a.n] : Entry{-INFINITY, -1};
    // entry `depth` of all lists, LISTS / 64 a lane
    const bool spread = a.splits >= 2 * a.n && a.n <= 16;
    const int depth = 1 << wv;
    Entry deep[LISTS / 64];
    if (!spread) {
#pragma unroll
        for (int i = 0; i < LISTS / 64; ++i) {
            deep[i] = {-INFINITY, -1};
            if (depth <= a.n && i * 64 < lists && i * 64 + lane < lists) deep[i] = best[(int64_t)(i * 64 + lane) * a.n + depth - 1];
        }
    }
    if (tid == 0) { sh.lists = 0; sh.count = 0; }
    for (int k = wv; k < a.K; k += MERGE_WAVES) {
        // (splits are at most a wave's lanes)
        const float score = a.scores[row0 + k];
        const float2 p = lane < a.splits ? a.sums[(row0 + k) * a.splits + lane] : make_float2(-INFINITY, 0.f);
        const bool bad = __any(p.x != p.x || !(p.y < INFINITY) || p.x == INFINITY);
        const float M = wave_max_dpp(p.x);
        double s = M > -INFINITY ? (double)(p.y * __builtin_amdgcn_exp2f((p.x - M) * LOG2E)) : 0.0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) {
            sh.top[k] = (double)M;
            sh.shift[k] = bad || !(s > 0.0) || !alive(score) ? (double)NAN : (double)score - log(s);
        }
    }
    __syncthreads();
    auto total_of = [&](const Entry &e, int k) -> Total {
        if (e.i < 0) return NONE;
        const double v = ((double)e.v - sh.top[k]) + sh.shift[k];
        return v > -INFINITY ? Total{v, (uint64_t)k << 32 | (uint32_t)e.i} : NONE;
    };
    Total mine = list < lists ? total_of(head, beam) : NONE;
    float at_depth = (float)mine.v;
    int wanted = (a.n + MERGE_WAVES - 1) / MERGE_WAVES;
    if (!spread) {
        at_depth = -INFINITY;
        wanted = (a.n + depth - 1) / depth;
#pragma unroll
        for (int i = 0; i < LISTS / 64; ++i)
            if (i * 64 < lists) at_depth = fmaxf(at_depth, (float)total_of(deep[i], min(i * 64 + lane, lists - 1) / a.by_splits).v);
    }
    const float w = nth_of_wave(at_depth, wanted);
    if (lane == 0) sh.border[wv] = w;
    __syncthreads();
    float border = sh.border[0];
#pragma unroll
    for (int k = 1; k < MERGE_WAVES; ++k) border = spread ? fminf(border, sh.border[k]) : fmaxf(border, sh.border[k]);
    if ((float)mine.v >= border && mine.v > -INFINITY) sh.good[atomicAdd(&sh.lists, 1)] = list;
    __syncthreads();
    // totals from the border on; where equal ones are more than the buffer holds, those from the n-th best of the first MERGED / 2 on, again
    const int entries = sh.lists * a.n;
    Total last = NONE;
    int count;
    for (bool again = false;; again = true) {
        for (int e0 = tid; e0 < entries; e0 += MERGE_THREADS * 4) {
            Entry x[4];
            int g[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int e = min(e0 + u * MERGE_THREADS, entries - 1), o = e / a.by_n;
                g[u] = sh.good[o];
                x[u] = best[(int64_t)g[u] * a.n + (e - o * a.n)];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (e0 + u * MERGE_THREADS >= entries) break;
                const Total t = total_of(x[u], g[u] / a.by_splits);
                if (t.v > -INFINITY && (again ? !better(last, t) : (float)t.v >= border)) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < MERGED) sh.buf[at] = t;
                }
            }
        }
        __syncthreads();
        count = sh.count;
        const int some = count <= MERGED ? count : MERGED / 2;
        for (int e = tid / 8; e < some; e += MERGE_THREADS / 8) {      // 8 threads an entry
            const Total t = sh.buf[e];
            int rank = 0;
#pragma unroll 4
            for (int j = tid & 7; j < some; j += 8) rank += better(sh.buf[j], t);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor(rank, o);
            if ((tid & 7) == 0 && rank < a.n) sh.out[rank] = t;
        }
        __syncthreads();
        if (count <= MERGED) break;
        last = sh.out[a.n - 1];
        if (tid == 0) sh.count = 0;
        __syncthreads();
    }
    const int found = min(count, a.n);
    if (wv != 0) return;
    // one wave: place i of the n best, and those among them that go on
    const bool have = lane < found;
    const Total t = have ? sh.out[lane] : NONE;
    if (lane < a.n) {
        const int64_t o = (int64_t)b * a.n + lane;
        a.out_score[o] = (float)t.v;
        a.out_beam[o] = t.beam();
        a.out_token[o] = t.token();
    }
    bool on = have;
    for (int k = 0; k < a.n_eos; ++k) on &= t.token() != a.eos[k];
    const uint64_t going = __ballot(on);
    const int at = __popcll(going & (((uint64_t)1 << lane) - 1)), n = min(__popcll(going), a.K);
    if (on && at < a.K) {
        const int64_t o = row0 + at;
        a.next_score[o] = (float)t.v;
        a.next_row[o] = (int)(row0 + t.beam());
        a.next_token[o] = t.token();
    }
    if (lane >= n && lane < a.K) {
        const int64_t o = row0 + lane;
        a.next_score[o] = -INFINITY;
        a.next_row[o] = -1;
        a.next_token[o] = -1;
    }
}

}  // namespace beam
