// Host-side plan of the paged attention: which block reads which keys for which query rows.
//
// Query rows of a K/V head: row r of a range of tokens is (token r / G, query head r % G of the head's group).  A segment is a
// range of tokens, the sequence whose page table gives the keys, and a range of its positions:
//   - the shared positions of a group of sequences, for all tokens of the group but those of sequences that fill row tiles by
//     themselves (every token sees all of them: a group's shared range ends at the earliest of these queries at the latest, so
//     that no mask is needed).  Where filling sequences stand between them the tokens are no range, and a list names them;
//   - a sequence's remaining positions, for its own tokens (causal).
// Segments are cut into row tiles of whole tokens: 32, 64 or 128 rows (1, 2 or 4 of a block's four waves side by side over
// the rows, the others over the keys).  Where the tiles of one size are too few to fill the chip, their keys are cut
// into parts of one common length, and every part leaves an (m, l, o) record per row; a token's records are the parts of its
// prefix tile and of its own tile.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <vector>

namespace paged {

struct Item {                        // one block's work
    int32_t tok0, ntok, kvh, seq;    // tokens, K/V head, row of the page table
    int32_t k0, k1;                  // positions read
    int32_t pos0;                    // token tok0 + i sees positions <= pos0 + i (ALL_SEEN: every one)
    int32_t rec;                     // first record (row r of the tile leaves record rec + r), -1: the output itself
    int32_t kind;                    // row tile of 32 << kind rows
    int32_t list;                    // the tokens are list[list ..] (tok0 the first), -1: tok0 ..
    int32_t reserved[2];
};
struct TokenRecs {                   // the records of a token: record (kvh * parts + j) * tile + i, times G, from base
    int32_t base[2], parts[2], tile[2], i[2];     // of the shared positions, of its own
};
constexpr int32_t ALL_SEEN = 1 << 30;
constexpr int KINDS = 3;                                       // row tiles of 32 << kind rows
constexpr int TILE_ROWS_OF[KINDS] = {32, 64, 128};
constexpr int KEY_STEP = 64;                                   // parts are whole steps of keys
// Cost of a step by kind: a tile of many rows is bound by its products and exponentials, one of few by memory, and how much
// they take of each other depends on the batch.  Decode of 32 / 96 requests over 8192 / 16384 shared positions, bf16 / e4m3, costs of
// 32 rows : more: 1 : 1 24.0 / 68.7 us, 2 : 3 23.7 / 62.2, 1 : 2 24.0 / 59.1, 2 : 5 25.3 / 61.3, 1 : 3 26.2 / 63.8.
constexpr int STEP_COST[KINDS] = {1, 2, 2};
// The fewest steps of a part: shorter ones cost more in records and latency than they spread.  Two (9 drafted tokens of 12 sequences
// over 1531 positions: 16.4 us, by one 18.5, by three 17.0); three where two would leave a row more than 32 records and the tile
// has rows enough for their traffic to count (4, 8, 16 requests of 7 heads on 8192: 12.8, 15.2, 20.1 -> 11.5, 14.1, 18.1 us; 16 on 6000
// 17.4 -> 16.6, on 4032 15.4 -> 15.3, on 3000 14.4 -> 14.8; a lone token's 7 rows on 8000 9.3 -> 10.3).
inline int64_t least_steps(int64_t steps, int64_t rows) { return steps > 64 && rows > 16 ? 3 : 2; }
constexpr int MAX_GROUP = 32;                                  // query heads per K/V head

// Tiles without shared positions up to this many values a row (positions x head_dim) are not cut: their items write the outputs, and
// the join's launch is saved (a pass over 1 to 16 sequences of head_dim 128, 256 / 512 / 640 / 768 positions: 7.2 / 9.1 / 10.2 / 11.6 us
// uncut, 10.7 cut and joined; head_dim 64, 512 / 1024: 7.3 / 9.3 against 10.6).
constexpr int64_t UNCUT_VALUES = 640 * 128;
struct Segment {
    int32_t tok0, ntok, seq, k0, k1, pos0, which, kind, list;  // which: 0 shared, 1 own; list: as an item's
};

struct PlanTables {
    std::vector<Item> items;         // the costliest first
    std::vector<TokenRecs> toks;
    std::vector<int32_t> list;       // tokens of shared items whose tokens are no range, each at most once
    bool joined = false;             // some token needs the join
    int32_t most_parts = 0;          // most records of a token that does
    int64_t records = 0;             // rows of records
    int32_t max_kv = 0;
};

// A part has the ITEM_TARGET-th of the whole cost: two blocks on each of 256 CUs get about the same; shorter tiles fill in (the
// two batches above: 448 23.9 / 64.8 us, 512 24.0 / 59.1, 576 26.8 / 63.8, 1024 34.8 / 68.0).
constexpr int ITEM_TARGET = 512;
// Most rows of records: a tile that is not cut leaves one record per row and range; the parts of those that are, each of more
// than one part's cost, are fewer than 2 ITEM_TARGET.
inline int64_t records_bound(int64_t rows, int n_heads) { return 2 * rows * n_heads + (int64_t)2 * ITEM_TARGET * 128; }
inline int64_t items_bound(int64_t rows, int n_kv) { return 2 * rows * n_kv + ITEM_TARGET; }

inline int kind_of(int64_t rows) { return rows <= 32 ? 0 : rows <= 64 ? 1 : 2; }

// The tables for the given lengths (checked by the caller: 0 <= q_len, 0 <= kv_len, group sizes sum to n_seq, shared <= kv_len
// of the group's sequences with queries).
inline void make_plan(int n_heads, int n_kv, int head_dim, int n_seq, const int32_t *q_len, const int32_t *kv_len, int n_groups,
                      const int32_t *group_size, const int32_t *group_shared, PlanTables &out) {
    const int G = n_heads / n_kv;
    std::vector<Segment> segs;
    std::vector<int32_t> sharing;                                            // the tokens that share, of a group
    int32_t n_tok = 0;
    out = PlanTables{};
    // a sequence whose own queries fill their row tiles (an eighth empty at most) gains nothing from rows of others beside
    // them: it reads the shared positions with its own, in one range, and needs no join
    const int per_tile = TILE_ROWS_OF[KINDS - 1] / G;
    auto fills_tiles = [&](int32_t q) { return (int64_t)(q + per_tile - 1) / per_tile * per_tile * 8 <= (int64_t)q * 9; };
    auto shares = [&](int s) { return q_len[s] > 0 && !fills_tiles(q_len[s]); };
    auto tiles_of = [&](int32_t ntok, auto &&tile) {
        const int kind = kind_of((int64_t)ntok * G), per = TILE_ROWS_OF[kind] / G;
        for (int32_t t = 0; t < ntok; t += per) tile(t, std::min(per, ntok - t), kind);
    };
    int s0 = 0;
    for (int g = 0; g < n_groups; ++g) {
        const int s1 = s0 + group_size[g];
        int32_t shared = group_shared[g], first = -1, members = 0, at = n_tok;
        sharing.clear();
        for (int s = s0; s < s1; ++s) {
            if (shares(s)) {
                if (first < 0) first = s;
                ++members;
                shared = std::min(shared, std::max(0, kv_len[s] - q_len[s]));
                for (int32_t i = 0; i < q_len[s]; ++i) sharing.push_back(at + i);
            }
            at += q_len[s];
        }
        if (members < 2) shared = 0;                                         // nothing to share
        if (shared > 0) {
            const int32_t n = (int32_t)sharing.size();
            const bool range = sharing[n - 1] - sharing[0] == n - 1;
            const int32_t base = (int32_t)out.list.size();
            if (!range) out.list.insert(out.list.end(), sharing.begin(), sharing.end());
            tiles_of(n, [&](int32_t t, int32_t len, int kind) {
                const bool run = sharing[t + len - 1] - sharing[t] == len - 1;
                segs.push_back({sharing[t], len, first, 0, shared, ALL_SEEN, 0, kind, run ? -1 : base + t});
            });
        }
        for (int s = s0; s < s1; ++s) {
            const int32_t k0 = shares(s) ? shared : 0, pos0 = kv_len[s] - q_len[s];
            tiles_of(q_len[s], [&](int32_t t, int32_t len, int kind) {
                const int32_t end = std::min(kv_len[s], pos0 + t + len);     // the tile's last token sees positions < end
                if (end > k0) segs.push_back({n_tok + t, len, s, k0, end, pos0 + t, 1, kind, -1});
            });
            if (q_len[s]) out.max_kv = std::max(out.max_kv, kv_len[s]);
            n_tok += q_len[s];
        }
        s0 = s1;
    }
    auto token = [&](const Segment &s, int i) { return s.list < 0 ? s.tok0 + i : out.list[s.list + i]; };
    out.toks.assign(n_tok, TokenRecs{});
    auto steps_of = [](const Segment &s) { return (int64_t)(s.k1 - s.k0 + KEY_STEP - 1) / KEY_STEP; };
    int64_t total = 0;
    for (const Segment &s : segs) total += steps_of(s) * STEP_COST[s.kind] * n_kv;
    const int64_t share = (total + ITEM_TARGET - 1) / ITEM_TARGET;
    bool whole = true;
    for (const Segment &s : segs) whole &= s.which == 1 && steps_of(s) * KEY_STEP * head_dim <= UNCUT_VALUES;
    auto parts_of = [&](const Segment &s) {
        if (whole) return (int64_t)1;
        const int64_t len = std::max<int64_t>(least_steps(steps_of(s), (int64_t)s.ntok * G), (share + STEP_COST[s.kind] - 1) / STEP_COST[s.kind]);
        return std::max<int64_t>(1, (steps_of(s) + len / 2) / len);        // (half a part more costs less than a cut)
    };
    for (const Segment &s : segs)
        for (int i = 0; i < s.ntok; ++i) {
            TokenRecs &t = out.toks[token(s, i)];
            t.parts[s.which] = (int32_t)parts_of(s);
            t.tile[s.which] = s.ntok;
            t.i[s.which] = i;
        }
    // records: a tile's block of (K/V head, part, token) rows, unless the tile's tokens have no other range or part
    for (const Segment &s : segs) {
        const int32_t parts = out.toks[s.tok0].parts[s.which];
        bool alone = parts == 1;
        for (int i = 0; i < s.ntok && alone; ++i) alone = out.toks[token(s, i)].parts[1 - s.which] == 0;
        const int64_t base = out.records;
        for (int i = 0; i < s.ntok; ++i) {
            TokenRecs &t = out.toks[token(s, i)];
            if (alone) t.parts[s.which] = -1;                                // written by its item
            else t.base[s.which] = (int32_t)(base / G);
        }
        if (!alone) out.records += (int64_t)n_kv * parts * s.ntok * G;
        const int64_t steps = steps_of(s);
        for (int h = 0; h < n_kv; ++h)
            for (int j = 0; j < parts; ++j) {                                // parts of nearly equal length
                const int32_t a = s.k0 + (int32_t)(steps * j / parts) * KEY_STEP;
                const int32_t b = j + 1 == parts ? s.k1 : s.k0 + (int32_t)(steps * (j + 1) / parts) * KEY_STEP;
                out.items.push_back({s.tok0, s.ntok, h, s.seq, a, b, s.pos0,
                                     alone ? -1 : (int32_t)(base + ((int64_t)h * parts + j) * s.ntok * G), s.kind, s.list, {0, 0}});
            }
    }
    std::stable_sort(out.items.begin(), out.items.end(), [](const Item &x, const Item &y) {
        return (int64_t)(x.k1 - x.k0) * STEP_COST[x.kind] > (int64_t)(y.k1 - y.k0) * STEP_COST[y.kind];
    });
    for (const TokenRecs &t : out.toks)
        if (t.parts[0] >= 0 && t.parts[1] >= 0) {                            // records to join, or no key at all (zeros)
            out.joined = true;
            out.most_parts = std::max(out.most_parts, t.parts[0] + t.parts[1]);
        }
}

}  // namespace paged
