// kv_attn_plan.h -- how the attention of a batch is launched: which kernel, in how
// many tiles and parts.  Shared by the launchers (kv_attn.hip), the C ABI and the
// CPU tests (tests/native).
#pragma once

#include <algorithm>
#include <stddef.h>

#include "kv_common.h"

namespace ihip {

// k_attn_rows
constexpr int AR_ROWS = 16;   // rows of a tile
constexpr int AR_KEYS = 32;   // keys of a wave's step
constexpr int AR_WAVES = 4;
constexpr int AR_SPLITS = 128; // parts of a tile's keys at most

// k_attn_chunk
constexpr int AC_ROWS = 128; // rows of a workgroup's tile, 32 a wave
constexpr int AC_KEYS = 128; // keys of a step at most
// Splits that one thread joins alone; more are shared among a workgroup's.  us,
// 256 tokens of 32 heads over 8000 keys in 8 splits 40 alone, 53 shared; 64 tokens
// of 4 heads over 60000 keys in 128 splits 44, 27.
constexpr int AC_FEW_SPLITS = 16;

// Keys that a wave multiplies in a step: as many as leave its registers room
// beside O^T and q (256 wide: 128 registers of O^T, 64 a part of q).  us, 32 keys
// against 64, a prompt of 4096 tokens of 32 heads, 256 wide: 3 parts 990, 2273; 2
// parts 830, 769.
constexpr int ac_half_keys(int parts, int dp) { return dp == 256 && parts == 3 ? 32 : 64; }
// Waves a SIMD: two, where a wave's operands fit 256 registers.
constexpr int ac_waves(int parts, int dp) { return dp <= 64 || (dp <= 128 && parts <= 2) ? 2 : 1; }

// Counts in front of the workspace, for calls of all sizes: its place does not
// depend on a call's.
constexpr int kAttnCounts = 4096;
// How a batch of these sizes is launched: it depends on nothing else, so that
// the workspace can be sized before the lengths are known.
struct AttnPlan {
    int rows;    // rows (tokens x heads of a group) of a tile
    int tiles;   // tiles at most, over all sequences
    int splits;  // parts of a tile's keys at most
    int least;   // keys of a part at least
    bool halves; // whether two halves of a workgroup share a tile's keys
    size_t bytes; // workspace: the counts, then the parts
};

// window: the window where there is one and no prefix reaches behind it, else 0
// (which never needs less workspace).
inline AttnPlan attn_plan(int act, int kv_type, int q_heads, int kv_heads, int dim, int sequences, int tokens,
                          int64_t capacity, int window)
{
    AttnPlan p;
    const int group = q_heads / kv_heads, parts = act != kF32 ? 1 : kv_type == kF16 ? 2 : 3;
    // p.tiles: the sum of ceil(rows of a sequence / p.rows) at most
    const int64_t rows = (int64_t)tokens * group, some = std::min(sequences, tokens);
    // Two tiles of few rows a sequence on average, or short caches whose tiles of few
    // rows all have room at once, take the kernel of few rows; more rows read the keys
    // too often there.  us, few rows against many (fp16, 128 wide, 8 KV heads): 8
    // sequences of 20 rows over 4000 keys 42, 48; of 48 rows 59, 54; of 96 rows 86,
    // 53; of 96 rows over 300 keys 15, 20; 32 of 48 rows over 300 keys 24, 18.
    auto tiles_of = [&](int n) { return (rows - some) / n + some; };
    const bool fits = capacity <= 512 && tiles_of(AR_ROWS) * kv_heads <= 512;
    p.rows = rows <= 2 * (int64_t)AR_ROWS * some || fits ? AR_ROWS : AC_ROWS;
    p.tiles = (int)tiles_of(p.rows);
    const int64_t units = (int64_t)p.tiles * kv_heads;
    int64_t want;
    if (p.rows == AR_ROWS) {
        // a sequence alone fills the chip once; of many, of which some are longer
        // than others, the parts stay short enough to even out
        p.least = units <= 32 ? 128 : units <= 128 ? 256 : 512;
        want = units >= kAttnCounts ? 1 : (256 * std::min<int64_t>(some, 16) + units - 1) / units;
    } else {
        // tiles that fill the chip are not split: joining would cost more.  Fewer are
        // split as far as their workgroups all have room at once (twice as far where
        // sequences differ)
        const int64_t room = ac_waves(parts, dim <= 64 ? 64 : dim <= 128 ? 128 : 256) == 2 ? 512 : 256;
        p.least = 256;
        want = units >= 256 ? 1 : room * std::min<int64_t>(some, 2) / units;
    }
    // (a window, where there is one, ends a tile's keys: no part would lie behind)
    const int64_t reach = window ? std::min(capacity, (int64_t)window + p.rows + AC_KEYS) : capacity;
    const int64_t most = (reach + p.least - 1) / p.least;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(most, want), AR_SPLITS));
    // Few tiles: two halves of a workgroup each, which end a long tile sooner (us,
    // halves against none, 128 wide, 512 tiles of a 2048-token prompt: fp16 43.5, 52,
    // fp32 rows over fp16 96, 100; but 512 tiles of one length, 2048 tokens over 8192
    // keys, 297, 279, which the sizes do not tell apart); of many, two workgroups a CU
    // come further (4096 tokens, fp16: 132, 108).
    p.halves = p.splits == 1 && units <= 512;
    // (with 4096 tiles and heads or more nothing is split: their counts are enough)
    p.bytes = p.splits > 1 ? 4 * (size_t)kAttnCounts + (size_t)p.splits * tokens * q_heads * (dim + 2) * 4 : 0;
    return p;
}

} // namespace ihip
