// gd_plan.h -- which kernels a call of the gated delta rule takes, and where the
// chunks' operands lie in its workspace.  Host code only (no device types), so that
// the CPU tests can walk through it.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ihip {

constexpr int kDeltaChunk = 64;  // tokens of a chunk
constexpr int kDeltaShift = 6;
constexpr int kDeltaStepMost = 16; // new tokens up to which a sequence goes a token at a time
constexpr int kDeltaTri = 6 * 2 * 1024; // a 64 x 64 lower triangle: 6 tiles of 16 x 32 in two fp16 parts
constexpr int kDeltaRows = 192;  // floats of a chunk's row factors

// Numbers of tiles of 2^shift rows that sequences of `tokens` rows in all can have.
constexpr int64_t gd_tiles(int64_t tokens, int64_t sequences, int shift)
{
    return (tokens > 0 ? (tokens - 1) >> shift : 0) + sequences;
}

struct DeltaPlan {
    bool chunks;     // some sequence may have more new tokens than kDeltaStepMost
    bool steps;      // some may have fewer beside it
    int64_t tiles;   // numbers of chunks
    int frag;        // bytes of a chunk's K or Q of one head
    size_t tri, rows, raw, bytes; // offsets (K and Q first; P and M, factors, raw outputs) and the size
};

// parts: fp16 values that a value of K or Q is held in (2 for fp32, else 1)
inline DeltaPlan delta_plan(int parts, int k_heads, int v_heads, int k_dim, int v_dim, int64_t tokens, int64_t sequences,
                            int most)
{
    DeltaPlan p{};
    const int64_t longest = most > 0 && most < tokens ? most : tokens;
    p.chunks = longest > kDeltaStepMost;
    p.steps = !p.chunks || sequences > 1;
    if (!p.chunks)
        return p;
    p.tiles = gd_tiles(tokens, sequences, kDeltaShift);
    const int padded = k_dim <= 64 ? 64 : 128;
    p.frag = padded * 128 * parts;
    p.tri = (size_t)p.tiles * (size_t)k_heads * 2 * (size_t)p.frag;
    p.rows = p.tri + (size_t)p.tiles * (size_t)v_heads * (size_t)(kDeltaTri + padded * 256);
    p.raw = p.rows + (size_t)p.tiles * (size_t)v_heads * kDeltaRows * 4;
    p.bytes = p.raw + (parts == 1 ? (size_t)tokens * (size_t)v_heads * (size_t)v_dim * 4 : 0);
    return p;
}

} // namespace ihip
