// kv_common.h -- the paged cache of keys and values and the batch that reads
// and extends it, shared by the kernels of kv_rope.hip, kv_attn.hip and
// kv_pages.hip.
//
// A page holds page_size tokens of every KV head: element (page, head, slot,
// i) of K or V is at page * page_stride + (head * page_size + slot) * dim + i,
// so that the tokens of one head in one page are one contiguous run, which is
// what a workgroup of the attention reads.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ihip {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30; // GGML type ids (src/GGUF.jl:25-60)
constexpr int kMaxHeadDim = 256;
constexpr int kMinPage = 16;

// bits of *flags (IHIP_FLAG_KV_*)
constexpr uint32_t kFlagKvPage = 8, kFlagKvLength = 16, kFlagKvFull = 32;

struct KvCache {
    void *k, *v;
    int type, pages, page_shift, heads, dim;
    int64_t page_stride; // elements
};

struct KvBatch {
    const int32_t *starts, *lens, *table;
    int sequences, stride, tokens;
};

// A sequence of the batch as the kernels see it: its rows start .. start + n - 1
// of q and its length in the cache.  Values that do not fit the batch's sizes
// are cut to them, so that no index formed from them leaves the buffers.
struct KvSeq {
    int start, n, len;
};

__device__ __forceinline__ int kv_clamp(int v, int lo, int hi)
{
    return min(max(v, lo), hi);
}

__device__ __forceinline__ KvSeq kv_seq(const KvBatch &b, int page_shift, int s)
{
    KvSeq q;
    q.start = kv_clamp(b.starts[s], 0, b.tokens);
    q.n = kv_clamp(b.starts[s + 1], q.start, b.tokens) - q.start;
    const int64_t cap = (int64_t)b.stride << page_shift;
    q.len = (int)min((int64_t)max(b.lens[s], 0), cap);
    return q;
}

// Reports the sequences whose values had to be cut, or have more new tokens
// than tokens.  One workgroup of a launch calls it.
__device__ __forceinline__ void kv_report(const KvBatch &b, int page_shift, uint32_t *flags)
{
    for (int s = threadIdx.x; s < b.sequences; s += blockDim.x) {
        const KvSeq q = kv_seq(b, page_shift, s);
        if (q.len != b.lens[s] || q.n > q.len || q.start != b.starts[s] || q.start + q.n != b.starts[s + 1])
            atomicOr(flags, kFlagKvLength);
    }
}

// The sequence that unit `want` lies in, where a sequence of n rows has
// units(n) of them (its rows, or tiles of them): the lanes of a wave look at 64
// sequences at a time, so that a batch of up to 64 costs one round of loads.
// Returns its index (-1: the batch has no such unit), the units of those before
// it in `first` and the sequence itself in `q`.  All lanes must be active.
// ROW: units are rows, and `want` comes as a row of q and is made the unit that
// it is, counted from the first sequence's first row (which need not be row 0).
template <bool ROW, typename F>
__device__ __forceinline__ int kv_find(const KvBatch &b, int page_shift, int &want, int &first, KvSeq &q, F units)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < b.sequences; s0 += 64) {
        const int s = s0 + lane;
        KvSeq mine{0, 0, 0};
        if (s < b.sequences)
            mine = kv_seq(b, page_shift, s);
        if (ROW && s0 == 0) {
            want -= __builtin_amdgcn_readlane(mine.start, 0);
            if (want < 0)
                return -1;
        }
        const int own = units(mine.n);
        int sum = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int up = __shfl_up(sum, d);
            sum += lane >= d ? up : 0;
        }
        const uint64_t past = __ballot(before + sum > want);
        if (past) {
            const int at = __builtin_ctzll(past);
            first = before + __builtin_amdgcn_readlane(sum - own, at);
            q.start = __builtin_amdgcn_readlane(mine.start, at);
            q.n = __builtin_amdgcn_readlane(mine.n, at);
            q.len = __builtin_amdgcn_readlane(mine.len, at);
            return s0 + at;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

} // namespace ihip
