// A call of sequences that share a prefix: which way its rows go, and what the ways are estimated to take.  Host arithmetic without a device,
// so that it can be run over any shape anywhere.
#pragma once

#include <algorithm>
#include <cmath>

#include "splitk_plan.h"

namespace tt {

constexpr int kFrontRows = 128;      // rows of a tile that packs the rows of all sequences (attn_splitk.hip)
constexpr int kSharedTokens = 1024;  // rows of all sequences together that are served at a time, so that the partial results stay small
// Sequences that are served at a time: 1 where there is nobody to share with.
inline int shared_seqs_at_once(int n_seq, int rows) { return std::max(std::min({n_seq, kMaxSeqPerLaunch, kSharedTokens / rows}), 1); }

struct SharedCall {
    int n_cus, split_override;
    int n_seq;          // at most shared_seqs_at_once
    const int *totals;  // keys up to each sequence's last row
    int rows, front;    // rows of a sequence; the shared keys, whole blocks
    int n_q_heads, n_kv_heads, head_dim, bits;
    bool chunk_kernel;  // serves these rows
};

// What the ways of a shared-prefix call are estimated to take, in us: fitted to calls of 2 .. 64 sequences of 1 and 4 rows behind 700 .. 20,000
// keys, of 16/4 heads of 64, 32/8 of 128, 16/2 and 24/2 of 256 over 16, 8 and 4 bits, where what they choose takes 3 % more than the best way.
// 128 keys of a tile's walk (a block for each of its workgroup's wavefronts): their way out of L2, mostly, whatever their
// bits, and over fewer of them the 32-row tiles' widening.
inline double turn_us(int D, int nt, int bits) {
    return (0.2 + 0.0057 * D) * (bits == 16 || nt == 16 ? 1.0 : D == 256 ? 1.6 : 1.15);
}
// A workgroup beside its walk, and how many of them a CU holds.
inline double start_us(int D, int nt) { return nt == 32 ? 1.5 + 0.0215 * D : 2.0 + 0.0098 * D; }
inline int groups_per_cu(int D, int nt) { return nt == 32 ? 256 / D : D == 256 ? 2 : 4; }
// Partial results that are written and read back.
inline double partials_us(double rows, int D) { return rows * D * 8.0 / 2.5e6; }

// Two passes in one launch: the tokens of all sequences over the keys [0, front) of prefix_slot, every sequence over its own from there on.
// The shared keys in the split-K tiles of 16 or 32 rows or in tiles of 128 packed ones, the own keys in split-K tiles, both in splits of at
// most the same length, the one that makes the launch the cheapest (64 rows of 16/2 heads of 256 over 30,011 keys and 50 .. 2,000 of their
// own, packed, in splits of 256 / 512 / 960 / 1,536 / 2,048 113 / 84 / 79 / 67 / 74 us, with the join; 20 of 32/8 of 128 over 6,000 over 8 bits, not
// packed, in 128 / 512 / 1,024 / 2,048 26 / 17.6 / 17.4 / 23.6).
struct PairPlan {
    LaunchPlan tiles;
    bool packed_rows;  // the shared keys by tiles of kFrontRows packed rows (attn_splitk.hip); tiles.nt and .tt are those of the own keys' tiles
    int own_tok_tiles, own_tiles, len;
    double us;  // with the join behind it
};
inline int splits_in(int keys, int len) { return std::max((keys + len - 1) / len, 1); }
inline int plan_pieces(const SharedCall &c, bool packed_rows, PairPlan *p) {
    const int n_seq = c.n_seq, rows = c.rows, front = c.front, n_q_heads = c.n_q_heads, *totals = c.totals;
    const int D = c.head_dim, tokens = n_seq * rows;
    long long own_keys = 0, own_turns = 0;
    int longest_own = 0;
    for (int i = 0; i < n_seq; ++i) {
        const int own = totals[i] - front;
        longest_own = std::max(longest_own, own);
        own_keys += own;
        own_turns += (own + 127) / 128;
    }
    // (tiles of 16 or 32 rows: by the shared keys, which both passes then take in the same ones, or by the own keys alone)
    const int st = packed_rows ? plan_splitk(c.n_cus, c.split_override, 0, n_seq, n_q_heads, c.n_kv_heads, D, rows, own_keys, 0, longest_own, &p->tiles,
                                             c.bits, true)
                               : plan_splitk(c.n_cus, c.split_override, 0, 1, n_q_heads, c.n_kv_heads, D, tokens, front, front, front, &p->tiles,
                                             c.bits, true);
    if (st != TT_HIP_OK) return st;
    LaunchPlan &plan = p->tiles;
    p->packed_rows = packed_rows;
    p->own_tok_tiles = (rows + plan.tt - 1) / plan.tt;
    p->own_tiles = plan.n_tiles / plan.tok_tiles * p->own_tok_tiles;
    if (packed_rows) {
        plan.tok_tiles = (tokens * (n_q_heads / c.n_kv_heads) + kFrontRows - 1) / kFrontRows;
        plan.n_tiles = plan.tok_tiles * c.n_kv_heads;
    }
    const int slots_on_chip = c.n_cus * groups_per_cu(D, packed_rows ? 32 : plan.nt);
    const double fixed = start_us(D, packed_rows ? 32 : plan.nt), turn = turn_us(D, plan.nt, c.bits);
    // (packed rows: a block of keys a step; the workgroups of a CU hide some of each other's)
    const int per_cu = groups_per_cu(D, 32);
    const double step = (0.3 + 0.0021 * D) * (c.bits == 16 ? 1.0 : 1.0 + 0.0013 * D);
    const double shared_step = step * (per_cu == 1 ? 1.0 : per_cu == 2 ? 1.2 : 1.8);
    const double walk_us = 1.36 * ((double)plan.n_tiles * ((front + 127) / 128) + (double)own_turns * p->own_tiles) * turn / c.n_cus;
    const double turn_alone = 0.36 + 0.005 * D;
    const int longest = std::max(front, longest_own);
    auto us_of = [&](int len) {
        const double own = n_seq + (longest_own > len ? (double)(own_keys / len) : 0.0);  // (splits of own keys, or a few more)
        const double front_groups = (double)plan.n_tiles * splits_in(front, len), groups = front_groups + own * p->own_tiles;
        const double rounds = std::ceil(groups / slots_on_chip), part_rows = ((double)tokens * splits_in(front, len) + rows * own) * n_q_heads;
        if (packed_rows) {
            // The workgroups over shared keys start first, those over own keys take the places that they leave.
            const int steps = std::min(len, front) / 32;
            const double own_group = 0.35 * fixed + (0.13 + 0.0023 * D) * std::ceil(std::min<double>(len, own_keys / own) / 128.0);
            const double busy = (front_groups * (0.57 * fixed + steps * shared_step) + own * p->own_tiles * own_group) / slots_on_chip;
            const double walk = std::max(std::ceil(front_groups / slots_on_chip) * (0.57 * fixed + steps * step), busy + 1.8 * own_group);
            return 7.5 + 0.0016 * tokens * n_q_heads + walk + 0.48 * partials_us(part_rows, D);
        }
        return 6.6 + fixed * (0.16 + 0.84 * rounds) + std::max(walk_us, (std::min(len, longest) + 127) / 128 * turn_alone) +
               0.2 * partials_us(part_rows, D);
    };
    if (c.split_override > 0) {
        p->len = (c.split_override + 31) / 32 * 32;
        p->us = us_of(p->len);
        return TT_HIP_OK;
    }
    p->len = 0;
    const int finest = packed_rows ? 32 : 128;
    for (int len = 128; p->len == 0 || len < longest + finest; len += std::max(finest, len / 8 / finest * finest)) {
        const double us = us_of(len);
        if (p->len == 0 || us < p->us) {
            p->us = us;
            p->len = len;
        }
    }
    return TT_HIP_OK;
}

// The ways:
//  * one pass: every sequence walks the shared keys like its own, out of the other slot's page; they are read once per sequence, mostly from L2;
//  * two passes in one launch and a join, the shared keys by split-K tiles, which the tokens of ALL sequences fill that one
//    sequence's rows leave mostly empty;
//  * the same, the shared keys by tiles of 128 packed rows: for more rows than a split-K tile has;
//  * the chunk kernel over ranges of the shared keys, its scores and values on wavefronts of their own, a pass over the own keys, and the join.
// One pass / two / two with packed rows / ranges, us, 100 own keys: one row a sequence of 16/2 heads of 256, 2 behind 2,000 9.1 / 11.0 / 13.3 / 24, 20 behind 6,000 18.3 / 16.3 / 23.5 / 29.5, 64 behind 20,000 92.8 / 44.9 / 44.0 / 47.7; 24/2 heads over 4
// bits, 20 behind 20,000 60 / 80 / 39 / 51; 32/8 of 128 over 8 bits, 20 behind 6,000 56 / 18.9 / 20.1 / 32.6, behind 20,000 177 / 44.5 / 33.2 / 57.7; four
// rows a sequence, 64 of 24/2 of 256 behind 2,000 39.4 / 91.6 / 50.4 / 56.6, behind 20,000 267 / 290 / 160 / 153.
// Between ranges and the rest the estimates are the coarsest.  Ranges / what the call takes without them, of calls that are sent to ranges: heads of
// 256, 16/2, 64 x 16 rows behind 4,096 140 / 166, 5 x 200 158 / 224, over 8 bits 64 x 4 behind 20,011 121 / 134; 24/2, 3 x 100 behind 4,100 78 / 185, over
// 8 bits 8 x 100 behind 1,055 204 / 363, over 4 bits 64 x 2 behind 32,768 142 / 166, but 5 x 200 behind 2,080 over 16 bits 260 / 186; heads of 128, 32/8,
// 64 x 4 rows behind 4,096 57.8 / 51.8, over 8 bits 64 x 16 168 / 147, 32/4, 32 x 32 161 / 127.
enum class SharedWay { one_pass, tiles, packed_rows, ranges };
struct SharedPlan {
    SharedWay way;
    SharedWay without_ranges;  // where the ranges' results or the dequantised pages find no room
    PairPlan pair;             // of the two passes in one launch that is the cheaper one
    KeyRanges ranges;
};
inline int plan_shared(const SharedCall &c, SharedPlan *p) {
    *p = SharedPlan{};
    const int D = c.head_dim, n_seq = c.n_seq;
    long long keys = 0;
    int longest = 0;
    for (int i = 0; i < n_seq; ++i) {
        keys += c.totals[i];
        longest = std::max(longest, c.totals[i]);
    }
    if (n_seq == 1 || longest <= 384) return TT_HIP_OK;  // (nobody to share with; one launch that ends in the final rows)
    LaunchPlan alone{};
    int st = plan_splitk(c.n_cus, c.split_override, 0, n_seq, c.n_q_heads, c.n_kv_heads, D, c.rows, keys, longest, longest, &alone, c.bits, true);
    if (st != TT_HIP_OK) return st;
    PairPlan packed{};
    st = plan_pieces(c, false, &p->pair);
    if (st == TT_HIP_OK) st = plan_pieces(c, true, &packed);
    if (st != TT_HIP_OK) return st;
    if (packed.us < p->pair.us) p->pair = packed;
    const double turn = turn_us(D, alone.nt, c.bits), key_us = 0.9 * turn / c.n_cus / 128.0;  // of a tile
    long long splits = 0;
    for (int i = 0; i < n_seq; ++i) splits += splits_in(c.totals[i], alone.split_len);
    const bool joined = longest > alone.split_len;
    const double rounds = std::ceil((double)splits * alone.n_tiles / (c.n_cus * groups_per_cu(D, alone.nt)));
    const double alone_us = 2.9 + start_us(D, alone.nt) * (0.45 + 0.5 * rounds) +
                            std::max(key_us * alone.n_tiles * (double)keys, (std::min(alone.split_len, longest) + 127) / 128 * 0.8 * turn) +
                            (joined ? 1.6 + 0.75 * partials_us((double)splits * c.rows * c.n_q_heads, D) : 0.0);
    double ranges_us = 0.0;
    if (c.chunk_kernel) {
        p->ranges = plan_key_ranges(c.n_cus, D, c.n_q_heads, c.n_kv_heads, n_seq * c.rows, c.front / 32);
        ranges_us = p->ranges.us + 4.0 + 4.0 + key_us * alone.n_tiles * (double)(keys - (long long)n_seq * c.front) + 7.0;
        // (quantised pages are dequantised once per call in front of the chunk kernel)
        if (c.bits != 16) ranges_us += 4.0 + (double)c.front * c.n_kv_heads * D * (2.0 + c.bits / 8.0) * 2.0 / 6.0e6;
    }
    p->without_ranges = alone_us <= p->pair.us ? SharedWay::one_pass : p->pair.packed_rows ? SharedWay::packed_rows : SharedWay::tiles;
    p->way = c.chunk_kernel && p->ranges.n_splits >= 2 && ranges_us < std::min(alone_us, p->pair.us) ? SharedWay::ranges : p->without_ranges;
    return TT_HIP_OK;
}

}  // namespace tt
