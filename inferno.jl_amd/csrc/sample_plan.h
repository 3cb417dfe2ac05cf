// sample_plan.h -- how the rows of a sampling call are cut into slices, and where what
// passes between its launches lies in the workspace.  Host code only (no device
// types), so that the CPU tests can walk through it.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ihip {

constexpr int kSampleThreads = 512;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 2048;  // tokens at a boundary that are resolved in LDS
constexpr int kSampleRows = 512;   // rows of a launch
constexpr int kSampleRecord = 32;  // bytes of a row that are zero between calls
constexpr int kSampleSlices = 512; // of a row, at most

struct SamplePlan {
    int per, slices; // logits of a slice; slices of a row
    int rows;        // of a launch
    // offsets of the slices' values, the rows' bounds, their bins (weights, then
    // counts) and the tokens at their boundaries
    size_t parts, bounds, bins, list, bytes;
};

inline SamplePlan sample_plan(int rows, int vocab)
{
    SamplePlan p{};
    // Slices of 16384 logits, or of 4096 where those would leave CUs idle (151936
    // logits: from 26 rows on; us, either side of it to be measured beside the kernels)
    const int64_t wide = 16384, narrow = 4096;
    int64_t per = rows * ((vocab + wide - 1) / wide) >= 256 ? wide : narrow;
    while ((vocab + per - 1) / per > kSampleSlices)
        per *= 2;
    p.per = (int)per;
    p.slices = (int)((vocab + per - 1) / per);
    p.rows = rows < kSampleRows ? rows : kSampleRows;
    const size_t n = (size_t)p.rows;
    p.parts = (size_t)kSampleRows * kSampleRecord;
    p.bounds = p.parts + n * (size_t)p.slices * 16;
    p.bins = p.bounds + n * 64;
    p.list = p.bins + n * kSampleBins * 12;
    p.bytes = p.list + n * kSampleList * 8;
    return p;
}

} // namespace ihip
