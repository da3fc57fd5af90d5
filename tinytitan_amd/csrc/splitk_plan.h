// How the split-K kernel is launched: its tiles, and how keys are cut into splits.  Host arithmetic without a device, so that it can be
// run over any shape anywhere.
#pragma once

#include <cstddef>

#include "../../include/ctinytitan_hip.h"
#include "chunk_plan.h"

namespace tt {

constexpr int kMaxSeqPerLaunch = 64;

struct LaunchPlan {
    int nt;  // 16 or 32 query rows per tile
    int gh, tt, hsubs, tok_tiles, n_tiles;
    int waves;
    int split_len, n_splits_max;
    long long workgroups;
    std::size_t lds_bytes;  // (the kernel's to say)
    bool stream;  // every K/V byte is read once by the launch, and there are many of them: non-temporal loads
    bool paired;  // ... and V operands in pairs, over heads of 256 in tiles of 32 rows
    bool xcd_grid;  // launch with kHotXcdGrid
    int slots_per_cu;  // workgroups that the planner's rule for unlike lengths counts on
    int packed_splits;  // > 0: launch with kHotPackedSplits over this many splits
    bool partials_only;  // the partial results are somebody else's to combine (PassParts)
};

inline int plan_splitk(int n_cus, int split_override, int kind, int n_seq, int n_q_heads, int n_kv_heads, int head_dim, int rows,
                       long long total_keys, int min_keys, int max_keys, LaunchPlan *plan, int kv_bits, bool small_tiles_ok) {
    if (n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads != 0) return TT_HIP_ERR_SHAPE;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return TT_HIP_ERR_SHAPE;
    if (rows <= 0 || n_seq <= 0) return TT_HIP_ERR_INVALID_ARGUMENT;
    const int group = n_q_heads / n_kv_heads;
    LaunchPlan p{};
    if (kind == 1) {  // prefill: 32 tokens of one q head per tile
        p.nt = 32;
        p.gh = 1;
    } else {
        // GQA-packed rows: all q heads of a KV head (times the tile's tokens) share one pass over K/V.
        p.gh = packed_heads(group);
        p.nt = (rows * p.gh <= 16) ? 16 : 32;
        // Tiles of 16 rows although the rows would fill tiles of 32, while the launch reads little: the 32-row
        // kernel's fixed costs (one workgroup per CU, 32 rows x D floats per wavefront merged through LDS and left as
        // the partial result) then outweigh reading the cache once per tile of 16.  "Little" is counted in keys walked
        // by tiles of 16 over the whole launch, keys x tiles of 16 x KV heads (figures for 2 KV heads of 256, fp16):
        //  * A few verify rows (up to four tiles of 16 per KV head, whose reads all come from HBM): 4 rows at 8k keys
        //    16.4 -> 13.8 us, at 2k keys 13.5 -> 9.8, 4 sequences x 4 rows at 4k keys 19.5 -> 16.7, 8 rows at 8k keys
        //    18.6 -> 16.0; at 36k keys 24.1 against 24.3, at 64k keys 32.6 against 35.5 the other way.  Over quantised
        //    pages the 32-row tile is dearer still (4 rows at 64k keys over 8 bits 28.6 -> 24.6 us).
        //  * A short chunk behind a short context (more tiles, which re-read the same keys from L2), as long as the
        //    tiles are one round of workgroups: 32 rows from position 0 11.0 -> 6.5 us, 128 rows behind 1024 keys
        //    18.7 -> 15.0, 256 rows behind 1024 keys 22.8 -> 17.4; 128 rows behind 3k keys 26.4 against 29.2 the
        //    other way, and 512 rows from position 0 were 17.0 against 19.7.
        // With 8 KV heads of 128 the same counts hold per KV head four times earlier (4 sequences x 16 rows at 4k keys:
        // 22.2 us in tiles of 32, 27.2 in tiles of 16; 8 rows at 8k keys 15.1 against 13.9), with 4 of 64 twice.
        if (small_tiles_ok && p.nt == 32 && p.gh <= 16) {
            const long long tiles16 = (rows + 16 / p.gh - 1) / (16 / p.gh);
            const long long launch_tiles16 = tiles16 * n_kv_heads * (group / p.gh);  // per sequence
            long long limit;  // of keys x tiles of 16 over the launch (the rows' own keys included)
            if (tiles16 <= 4) limit = kv_bits == 16 ? 144 * 1024 : 288 * 1024;
            else if (launch_tiles16 * n_seq <= n_cus) limit = kv_bits == 16 ? 320 * 1024 : 384 * 1024;
            else limit = 0;
            if (total_keys * launch_tiles16 <= limit) p.nt = 16;
        }
    }
    p.tt = p.nt / p.gh;
    p.hsubs = group / p.gh;
    p.tok_tiles = (rows + p.tt - 1) / p.tt;
    p.n_tiles = n_kv_heads * p.hsubs * p.tok_tiles;
    p.waves = 4;
    const int min_split = 32 * p.waves;  // one key block per wave
    // Workgroup slots of the chip: the 16-row kernel fits two workgroups per CU, the 32-row one.
    p.slots_per_cu = p.nt == 16 ? 2 : 1;
    const long long slots = (long long)n_cus * p.slots_per_cu;
    int split_len;
    if (split_override > 0) {
        split_len = ((split_override + 31) / 32) * 32;
    } else if (kind == 1) {
        split_len = ((max_keys + 31) / 32) * 32;  // prefill tiles are plentiful: no split
    } else if (min_keys == max_keys) {
        // Equal lengths: give every (sequence, tile) the same whole number of splits so that the
        // launch is exactly one round of at most n_cus workgroups -- a 257th workgroup would wait
        // for a CU and double the kernel's time.
        const long long pairs = (long long)n_seq * p.n_tiles;
        long long per_pair = n_cus / pairs;
        // Two rounds, side by side on a CU, where a workgroup's loads are few bytes and its walk is long (131k keys over 8 bits
        // with 16/4 heads of 64 23.4 -> 18.0 us, over 4 bits with 32/8 heads of 128 43.0 -> 35.6; with 16/2 of 256 27.4 -> 30.1).
        // Twice the partial results have to be worth it, which is a walk the longer the more rows and dims they have (before the
        // line / at it: 16 rows of 64, 920 keys a workgroup 12.8 -> 13.0 us, 1080 15.2 -> 13.0; 16 of 128 or 32 of 64, 860 keys
        // 14.9 -> 15.8, 1300 19.0 -> 16.2; 32 of 128, 1400 keys 26.3 -> 28.3, 1730 39.2 -> 30.3), and where there was one
        // workgroup a tile, and no combine, a longer one still (1613 keys 21.0 -> 27.0, 3416 25.9 -> 29.2, 8486 87 -> 61).
        const long long walk = per_pair <= 1 ? 4096 : p.nt * head_dim <= 1024 ? 1024 : p.nt * head_dim <= 2048 ? 1280 : 1536;
        if (head_dim * kv_bits <= 512 && pairs <= n_cus && max_keys >= walk * per_pair) per_pair = 2 * n_cus / pairs;
        if (per_pair < 1) per_pair = 1;
        split_len = (int)((max_keys + per_pair - 1) / per_pair);
        split_len = ((split_len + min_split - 1) / min_split) * min_split;
    } else {
        // Ragged lengths: about two workgroups per slot evens out the unequal last splits.
        const long long target_wgs = 2 * slots;
        const long long key_work = total_keys * p.n_tiles;
        long long per_wg = (key_work + target_wgs - 1) / target_wgs;
        // ... and at most 256 splits for the longest sequence: the grid is (splits of the longest, tiles,
        // sequences), and one long sequence beside many short ones would otherwise launch a grid of
        // workgroups that find nothing to do.
        if (per_wg < (max_keys + 255) / 256) per_wg = (max_keys + 255) / 256;
        split_len = (int)(((per_wg + min_split - 1) / min_split) * min_split);
    }
    // Up to 384 keys: one split, whose workgroup writes the final rows itself -- a wavefront's three blocks cost less
    // than the second launch (one decode row at 128 keys 8.6 -> 6.3 us a step, at 256 keys 8.7 -> 7.4; at 512 keys
    // 10.3 against 8.7 the other way).
    if (split_override <= 0 && kind == 0 && max_keys <= 384) split_len = ((max_keys + 31) / 32) * 32;
    if (split_len < 32) split_len = 32;
    p.split_len = split_len;
    p.n_splits_max = max_keys > 0 ? (max_keys + split_len - 1) / split_len : 1;
    if (p.n_splits_max < 1) p.n_splits_max = 1;
    p.workgroups = (long long)p.n_splits_max * p.n_tiles * n_seq;
    p.xcd_grid = false;
    *plan = p;
    return TT_HIP_OK;
}

}  // namespace tt
