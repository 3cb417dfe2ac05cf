// gd_conv.hip -- the short causal convolution of a recurrent layer:
//
//   y[t, c] = act(bias[c] + sum_{j < W} w[c, j] x[t - W + 1 + j, c])
//
// where the inputs before a sequence's first new token are the W - 1 that its slot
// keeps (zeros where the sequence begins), and the slot then keeps the last W - 1.
#include "gd_launch.h"

namespace ihip {

namespace {

constexpr int CONV_THREADS = 256;
constexpr int CONV_AHEAD = 8; // tokens whose values are on their way at once

// A thread owns 4 channels of a tile and walks down its tokens with the last W - 1
// inputs in registers, so that a tile reads W - 1 rows twice and everything else
// once.  A sequence's first tile alone reads and writes its state (the new one is
// read from x, wherever its tile is), and in one thread, so no tile waits for another.
// Bound by bytes: 8192 tokens of 8192 channels, fp32 in and bf16 out, 93 to 96 us (4.2 to 4.3 TB/s;
// 103 with the type looked at beside every load, which then wait for each other); one
// token of 6144 channels 4.1, its launch and two rounds of loads.
template <int TYPE, int W>
__global__ void __launch_bounds__(CONV_THREADS) k_short_conv(ConvArgs a)
{
    if (a.flags && blockIdx.x == 0 && blockIdx.y == 0)
        gd_report(a.batch, a.flags);
    int c = 0;
    const int s = gd_find(a.batch, a.shift, (int)blockIdx.x, c);
    if (s < 0)
        return;
    const GdSeq q = gd_seq(a.batch, a.pool, s, c == 0 && blockIdx.y == 0 ? a.flags : nullptr);
    const int ch = 4 * (int)(blockIdx.y * CONV_THREADS + threadIdx.x);
    if (q.slot < 0 || ch >= a.channels)
        return;
    float *state = a.state + q.slot * a.slot_step + ch;
    gd_f4 win[W]; // the last W - 1 inputs, then the token's own
    const int t0 = c << a.shift, t1 = min(t0 + (1 << a.shift), q.n);
    const int64_t row0 = (int64_t)q.start * a.x_step + ch;
    if (c > 0) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            win[j] = gd_wide(gd_raw4<TYPE>(a.x, row0 + (t0 - (W - 1) + j) * a.x_step));
    } else {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            win[j] = gd_f4{};
        if (!q.begins)
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
                win[j] = *(const gd_f4 *)(state + (int64_t)j * a.channels);
    }
    float w[4][W];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j)
            w[i][j] = a.w[(int64_t)(ch + i) * W + j];
    const gd_f4 bias = a.bias ? *(const gd_f4 *)(a.bias + ch) : gd_f4{};

    if (c == 0) {
        // the last W - 1 inputs: new ones, behind old ones where there are fewer
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const int t = q.n - (W - 1) + j;
            gd_f4 v{};
            if (t >= 0)
                v = gd_wide(gd_raw4<TYPE>(a.x, row0 + t * a.x_step));
            else
#pragma unroll
                for (int i = 0; i < W - 1; ++i)
                    if (i == j + q.n)
                        v = win[i];
            *(gd_f4 *)(state + (int64_t)j * a.channels) = v;
        }
    }
    for (int t = t0; t < t1; t += CONV_AHEAD) {
        typename GdType<TYPE>::T4 x[CONV_AHEAD]; // (behind the last token: it again)
#pragma unroll
        for (int i = 0; i < CONV_AHEAD; ++i)
            x[i] = gd_raw4<TYPE>(a.x, row0 + min(t + i, t1 - 1) * a.x_step);
#pragma unroll
        for (int i = 0; i < CONV_AHEAD; ++i) {
            if (t + i >= t1)
                break;
            win[W - 1] = gd_wide(x[i]);
            gd_f4 y = bias;
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y[e] = fmaf(w[e][j], win[j][e], y[e]);
            if (a.silu)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y[e] = gd_silu(y[e]);
            gd_store4(a.out, (int64_t)(q.start + t + i) * a.channels + ch, a.out_type, y);
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
                win[j] = win[j + 1];
        }
    }
}

template <int TYPE>
hipError_t launch(const ConvArgs &a, hipStream_t s)
{
    const dim3 grid((unsigned)gd_tiles(a.batch.tokens, a.batch.sequences, a.shift),
                    (unsigned)((a.channels / 4 + CONV_THREADS - 1) / CONV_THREADS));
    switch (a.width) {
#define IHIP_CONV(W)                                                                           \
    case W:                                                                                    \
        hipLaunchKernelGGL((k_short_conv<TYPE, W>), grid, dim3(CONV_THREADS), 0, s, a);        \
        break;
        IHIP_CONV(2) IHIP_CONV(3) IHIP_CONV(4) IHIP_CONV(5) IHIP_CONV(6) IHIP_CONV(7) IHIP_CONV(8)
#undef IHIP_CONV
    default:
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

} // namespace

hipError_t launch_short_conv(const ConvArgs &a, hipStream_t s)
{
    return a.x_type == kF32 ? launch<kF32>(a, s) : a.x_type == kF16 ? launch<kF16>(a, s) : launch<kBF16>(a, s);
}

} // namespace ihip
