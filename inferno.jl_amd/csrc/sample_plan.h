// sample_plan.h -- how the rows of a sampling call are cut into slices, and where what
// passes between its launches lies in the workspace.  Host code only (no device
// types), so that the CPU tests can walk through it.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ihip {

constexpr int kSampleThreads = 512;
constexpr int kSampleBins = 1024;
constexpr int kSampleList = 4096;   // tokens at a boundary that are resolved in LDS
constexpr int kSampleRows = 256;    // rows of a launch
constexpr int kSampleRecord = 64;   // bytes of a row's bounds
constexpr int kSamplePart = 24;     // bytes of a slice's values
constexpr int kSampleSlices = 512;  // of a row, at most
constexpr int kSampleWide = 8192;   // logits of a slice (a thread's are in registers),
constexpr int kSampleNarrow = 4096; // and where those are fewer than two to a CU
constexpr int64_t kSampleVocab = (int64_t)kSampleWide * kSampleSlices;

struct SamplePlan {
    int per, slices; // logits of a slice; slices of a row
    int rows;        // of a launch
    // offsets of the rows' bounds (behind the slices' values), the slices' and the
    // rows' bins (weights, then counts) and the tokens at the rows' boundaries
    size_t bounds, bins, merged, list, bytes;
};

// The areas of `all` slices in p.rows rows
inline void sample_areas(SamplePlan &p, size_t all)
{
    const size_t n = (size_t)p.rows;
    p.bounds = (all * kSamplePart + 63) / 64 * 64;
    p.bins = p.bounds + n * kSampleRecord;
    p.merged = p.bins + all * kSampleBins * 12;
    p.list = p.merged + n * kSampleBins * 12;
    p.bytes = p.list + n * kSampleList * 8;
}

inline SamplePlan sample_plan(int rows, int vocab)
{
    SamplePlan p{};
    const int64_t wide = (vocab + kSampleWide - 1) / kSampleWide, narrow = (vocab + kSampleNarrow - 1) / kSampleNarrow;
    // Measured with top-k and top-p, us for slices of 8192 | 4096: rows of 151936, one 38.9 |
    // 34.2, 16 46.2 | 45.2, 32 55.1 | 56.4, 61 68.8 | 75.8; of 32000, 61 43.9 | 41.9.
    p.per = rows * wide >= 512 || narrow > kSampleSlices ? kSampleWide : kSampleNarrow;
    p.slices = (int)(p.per == kSampleWide ? wide : narrow);
    p.rows = rows < kSampleRows ? rows : kSampleRows;
    sample_areas(p, (size_t)p.rows * (size_t)p.slices);
    return p;
}

// Bytes that do for these rows and logits and for every call of no more of either.  Fewer rows, or
// logits, may have more slices, as theirs are narrow: rows * wide < 512 then, and narrow <= 2
// wide, so that there are at most 1022 of those.
inline size_t sample_scratch(int rows, int vocab)
{
    const int64_t wide = (vocab + kSampleWide - 1) / kSampleWide, narrow = (vocab + kSampleNarrow - 1) / kSampleNarrow;
    SamplePlan p{};
    p.rows = rows < kSampleRows ? rows : kSampleRows;
    const int64_t narrows = p.rows * narrow < 1022 ? p.rows * narrow : 1022;
    sample_areas(p, (size_t)(p.rows * wide > narrows ? p.rows * wide : narrows));
    return p.bytes;
}

} // namespace ihip
