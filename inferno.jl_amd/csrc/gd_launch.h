// gd_launch.h -- internal launchers of the layers that keep a state, shared by the
// kernel files and the C ABI.
#pragma once

#include "gd_common.h"
#include "kq_launch.h"

namespace ihip {

// gd_conv.hip
struct ConvArgs {
    const void *x;
    int x_type;
    int64_t x_step; // elements from one token to the next
    const float *w, *bias;
    int channels, width, silu;
    int shift; // a tile has 2^shift tokens
    float *state;
    int64_t slot_step; // floats from one slot to the next
    int pool;
    void *out;
    int out_type;
    StateBatch batch;
    uint32_t *flags;
};
hipError_t launch_short_conv(const ConvArgs &a, hipStream_t s);

// gd_step.hip, gd_chunk.hip
struct DeltaArgs {
    const void *q, *k, *v;
    int type;
    int64_t q_step, k_step, v_step; // elements from one token to the next
    const float *a, *b;
    int64_t a_step, b_step;
    const float *gate;
    int64_t gate_step;
    void *out;
    int out_type;
    float *state;
    int64_t slot_step; // floats from one slot to the next
    int pool;
    int k_heads, v_heads, group, k_dim, v_dim;
    const float *decay, *dt_bias, *norm_w;
    float norm_eps, l2_eps, scale;
    StateBatch batch;
    uint32_t *flags;
    // sequences that the chunks' kernels leave to the other one: with so many new
    // tokens, or fewer (the step kernel takes those; all of them where it is negative)
    int few;
    uint8_t *work;
    DeltaPlan plan;
    float *raw; // outputs before their norm (out itself where that is fp32)
};
hipError_t launch_delta_step(const DeltaArgs &a, hipStream_t s);
hipError_t launch_delta_chunks(const DeltaArgs &a, hipStream_t s);

} // namespace ihip
