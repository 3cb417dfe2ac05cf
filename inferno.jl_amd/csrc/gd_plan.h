// gd_plan.h -- which kernels a call of the gated delta rule takes, and where the
// chunks' operands lie in its workspace.  Host code only (no device types), so that
// the CPU tests can walk through it.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ihip {

constexpr int kDeltaShift = 6;  // a chunk is 64 tokens
constexpr int kDeltaTri = 6 * 2 * 1024; // a 64 x 64 lower triangle: 6 tiles of 16 x 32 fp32 values
constexpr int kDeltaRows = 256;  // floats of a chunk's row factors

// Numbers of tiles of 2^shift rows that sequences of `tokens` rows in all can have.
constexpr int64_t gd_tiles(int64_t tokens, int64_t sequences, int shift)
{
    return (tokens > 0 ? (tokens - 1) >> shift : 0) + sequences;
}

// New tokens up to which a batch goes a token at a time, all of it.  A token costs the step
// kernel 1.4 us whatever the batch, until that fills the chip; a chunk costs its
// kernels the same with few tokens as with 64, and every chunk of the batch adds to it.
// Measured on sequences of equally many tokens, 32 heads of 128 x 128 in bf16 with norm and gate, us by
// steps | chunks: one of 8 18.3 | 23.4, of 12 24.5 | 24.6; two of 16 28.8 | 32.4, of 20 35.1 | 33.4; four of 24
// 44.8 | 43.7, of 32 58.8 | 44.8 (the rule is late there); eight of 32 60.9 | 68.0, of 48 85.6 | 72.1.
constexpr int delta_few(int v_heads, int64_t sequences)
{
    const int64_t few = sequences * v_heads / 4;
    return few < 10 ? 10 : few > 32 ? 32 : (int)few;
}

// Beside longer sequences, the step kernel comes before the chunks' and lasts as long as
// its longest sequence, and chunks that do not fill the chip are next to free: there
// only a few tokens go by steps (sequences of 22, 8, 135, 5 and 72 tokens, 24 heads of
// 64 x 64: 27.1 us with up to 4, 35.8 with up to 10, 49.5 with up to 30).
constexpr int delta_few_beside(int v_heads, int64_t sequences)
{
    return sequences * v_heads < 256 ? 4 : 10;
}

// Tokens of a tile of the short convolution, as a power of two: 32, or 16 where those are
// fewer than 4 workgroups to a CU (1024 channels each).  Measured, us with 16 | 32: 2146 tokens of
// 2560 channels 14.3 | 17.7, 8192 of 8192 100.9 | 94.8 (a tile reads width - 1 rows twice).
constexpr int conv_shift(int64_t tokens, int64_t sequences, int channels)
{
    return gd_tiles(tokens, sequences, 5) * ((channels + 1023) / 1024) < 1024 ? 4 : 5;
}

struct DeltaPlan {
    int few;         // new tokens up to which a sequence goes a token at a time, where others take chunks
    bool chunks;     // some sequence may have more new tokens than delta_few
    bool steps;      // some may have fewer beside it
    int64_t tiles;   // numbers of chunks
    int frag;        // bytes of a chunk's K or Q of one head
    size_t tri, rows, raw, bytes; // offsets (K and Q first; P and M, factors, raw outputs) and the size
};

// The longest sequence that a batch may have
constexpr int64_t delta_longest(int64_t tokens, int most)
{
    return most > 0 && most < tokens ? most : tokens;
}

// The areas of chunks in the workspace.  parts: fp16 values that a value of K or Q is held in (2
// for fp32, else 1)
inline void delta_areas(DeltaPlan &p, int parts, int k_heads, int v_heads, int k_dim, int v_dim, int64_t tokens, int64_t sequences)
{
    p.tiles = gd_tiles(tokens, sequences, kDeltaShift);
    const int padded = k_dim <= 64 ? 64 : 128;
    p.frag = padded * 128 * parts;
    p.tri = (size_t)p.tiles * (size_t)k_heads * 2 * (size_t)p.frag;
    p.rows = p.tri + (size_t)p.tiles * (size_t)v_heads * (size_t)(kDeltaTri + padded * 256);
    p.raw = p.rows + (size_t)p.tiles * (size_t)v_heads * kDeltaRows * 4;
    p.bytes = p.raw + (parts == 1 ? (size_t)tokens * (size_t)v_heads * (size_t)v_dim * 4 : 0);
}

inline DeltaPlan delta_plan(int parts, int k_heads, int v_heads, int k_dim, int v_dim, int64_t tokens, int64_t sequences,
                            int most)
{
    DeltaPlan p{};
    p.chunks = delta_longest(tokens, most) > delta_few(v_heads, sequences);
    p.steps = !p.chunks || sequences > 1;
    p.few = p.steps ? delta_few_beside(v_heads, sequences) : 0;
    if (p.chunks)
        delta_areas(p, parts, k_heads, v_heads, k_dim, v_dim, tokens, sequences);
    return p;
}

// Bytes that do for a batch of these sizes and for every one of no more tokens, sequences and
// `most`: fewer sequences go in chunks at lengths at which more of them go by steps.
inline size_t delta_scratch(int parts, int k_heads, int v_heads, int k_dim, int v_dim, int64_t tokens, int64_t sequences,
                            int most)
{
    DeltaPlan p{};
    if (delta_longest(tokens, most) > delta_few(v_heads, 1))
        delta_areas(p, parts, k_heads, v_heads, k_dim, v_dim, tokens, sequences);
    return p.bytes;
}

} // namespace ihip
