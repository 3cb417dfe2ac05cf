// kv_launch.h -- internal launchers of the paged-cache kernels, shared by the
// kernel files and the C ABI.
#pragma once

#include "kq_launch.h"
#include "kv_attn_plan.h"
#include "kv_common.h"

namespace ihip {

// kv_rope.hip
struct RopeArgs {
    const float *q, *k, *v;
    int64_t q_step, k_step, v_step; // floats from one token to the next
    int q_heads, kv_heads, dim;     // kv_heads 0: q alone
    const float *q_norm, *k_norm;
    float eps;
    const double *turns;
    int rot, interleaved;
    float mscale;
    const int32_t *positions;
    void *out;
    int out_type;
    KvCache cache;
    KvBatch batch;
    uint32_t *flags;
    int hb, blocks; // heads a workgroup, workgroups a token (set by the launcher)
};
hipError_t launch_rope_kv(RopeArgs a, hipStream_t s);

// kv_attn.hip
struct AttnArgs {
    const void *q;
    void *out;
    int act, q_heads, group;
    float scale, cap;
    // set by the launcher: the scale's power of two, and without that a score's
    // factor to a power of two (with a cap: the cap's, and the score's to the cap)
    int scale_exp;
    float by, to_cap;
    int window;
    const int32_t *prefix;
    const float *slopes;
    KvCache cache;
    KvBatch batch;
    uint32_t *flags;
    uint32_t *count; // parts of each tile that have ended (0 between calls)
    float *part; // partial rows, then their maxima and sums, of every split
};
hipError_t launch_attn(AttnArgs a, const AttnPlan &p, hipStream_t s);

// kv_pages.hip
struct ForkArgs {
    const int32_t *table, *lens, *parents;
    int sequences, children, stride, page_size, room, pages;
    int32_t *refs, *table_out, *lens_out, *copies;
    int32_t *fresh; // 2 x children ints of scratch: pages each child is missing, and from where
    uint32_t *flags;
};
hipError_t launch_kv_fork(const ForkArgs &a, hipStream_t s);
struct CompactArgs {
    int32_t *table;
    int64_t entries;
    int32_t *refs;
    int pages;
    int32_t *copies, *moved;
    int32_t *to; // pages ints of scratch: each page's new index
    uint32_t *flags;
};
hipError_t launch_kv_compact(const CompactArgs &a, hipStream_t s);
// page_bytes: of one page of K (or V) in one layer; strides in bytes
hipError_t launch_kv_copy(void *k, void *v, int64_t page_bytes, int64_t page_stride, int64_t layer_stride,
                          int layers, int pages, const int32_t *copies, int n, const int32_t *count,
                          uint32_t *flags, hipStream_t s);

} // namespace ihip
