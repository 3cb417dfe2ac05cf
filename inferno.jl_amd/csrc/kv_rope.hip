// kv_rope.hip -- what lies between a layer's wq/wk/wv and its attention: the q
// and k norms, the rotary positions and the append of k and v to the paged
// cache, as one launch.
//
//   y = x / sqrt(mean(x^2) + eps) * w                     (where a norm is given)
//   (y_a, y_b) <- m (y_a cos t - y_b sin t, y_a sin t + y_b cos t),  t = 2 pi turns_i pos
//
// for the pairs (a, b) = (i, i + rot/2) or (2 i, 2 i + 1), i < rot/2; the rest
// of a head is left as it is.  The angle is formed in turns and in 64 bits
// (position 500000 times a 24-bit frequency would be off by up to 0.02 turns);
// whole turns are dropped there, and what is left is exact enough for a sine
// and cosine in 32 bits.
#include "kq_common.h"
#include "kv_launch.h"

namespace ihip {

namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_FLOATS = 4096; // head values a workgroup holds
constexpr int ROPE_HEADS = 16;    // heads a workgroup holds (16 lanes each sum a norm)

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float float8 __attribute__((ext_vector_type(8)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));

// 8 values, rounded once to the type they are kept in (to nearest)
__device__ __forceinline__ void store8(void *base, int64_t at, int type, float8 v)
{
    if (type == kF32)
        *(float8 *)((float *)base + at) = v;
    else if (type == kF16)
        *(half8 *)((_Float16 *)base + at) = __builtin_convertvector(v, half8);
    else
        *(bhalf8 *)((__bf16 *)base + at) = __builtin_convertvector(v, bhalf8);
}

// A workgroup takes `hb` of one token's q_heads + 2 kv heads.  Bound by bytes
// for a prompt (8192 tokens of 32 + 16 heads, 128 wide: 302 MB in 67 us, 4.5 TB/s;
// 113 with the values in indexed arrays), by its launch and three loads that wait
// for each other for a decode step (4.6 us).  The heads go through LDS: the two
// values of a pair lie rot/2 apart or side by side, and either way a thread then
// writes 8 neighbours at once.
__global__ void __launch_bounds__(ROPE_THREADS) k_rope_kv(RopeArgs a)
{
    __shared__ __attribute__((aligned(16))) float x[ROPE_FLOATS];
    __shared__ float2 cs[kMaxHeadDim / 2];
    __shared__ float inv[ROPE_HEADS];
    const int tid = threadIdx.x;
    const int D = a.dim;
    const int token = blockIdx.x / a.blocks, h0 = (blockIdx.x % a.blocks) * a.hb;
    const int heads = min(a.hb, a.q_heads + 2 * a.kv_heads - h0);
    const int knob = a.q_heads, vnob = a.q_heads + a.kv_heads; // first k and first v head

    // the values are on their way while the token's place is looked up
    const int n4 = heads * D / 4;
    f4 val[ROPE_FLOATS / 4 / ROPE_THREADS];
#pragma unroll
    for (int j = 0; j < ROPE_FLOATS / 4 / ROPE_THREADS; ++j) {
        const int i = tid + ROPE_THREADS * j;
        val[j] = f4{};
        if (i < n4) {
            const int h = h0 + 4 * i / D, e = 4 * i % D;
            const float *src = h < knob ? a.q + token * a.q_step + h * D
                             : h < vnob ? a.k + token * a.k_step + (h - knob) * D
                                        : a.v + token * a.v_step + (h - vnob) * D;
            val[j] = *(const f4 *)(src + e);
        }
    }

    if (blockIdx.x == 0 && a.flags)
        kv_report(a.batch, a.cache.page_shift, a.flags);
    int first = 0;
    KvSeq seq;
    int row = token;
    const int s = kv_find<true>(a.batch, a.cache.page_shift, row, first, seq, [](int n) { return n; });
    if (s < 0)
        return; // a row before the first sequence or behind the last
    const int at = seq.len - seq.n + (row - first);
    const int pos = a.positions ? a.positions[token] : at;

    for (int i = tid; i < a.rot / 2; i += ROPE_THREADS) {
        double t = (double)pos * a.turns[i];
        t -= rint(t);
        float sn, c;
        sincospif(2.0f * (float)t, &sn, &c);
        cs[i] = make_float2(a.mscale * c, a.mscale * sn);
    }
#pragma unroll
    for (int j = 0; j < ROPE_FLOATS / 4 / ROPE_THREADS; ++j) {
        const int i = tid + ROPE_THREADS * j;
        if (i < n4)
            *(f4 *)(x + 4 * i) = val[j];
    }
    __syncthreads();
    if (a.q_norm || a.k_norm) {
        // 16 lanes a head; the sum of squares in 32 bits, in a fixed order
        const int h = tid >> 4;
        if (h < heads) {
            float sum = 0.0f;
            for (int e = 4 * (tid & 15); e < D; e += 64) {
                const f4 v = *(const f4 *)(x + h * D + e);
                sum += (v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w);
            }
            sum = dpp_add<0xb1, 0xf>(sum);  // quad_perm [1,0,3,2]
            sum = dpp_add<0x4e, 0xf>(sum);  // quad_perm [2,3,0,1]
            sum = dpp_add<0x141, 0xf>(sum); // row_half_mirror
            sum = dpp_add<0x140, 0xf>(sum); // row_mirror
            if ((tid & 15) == 0)
                inv[h] = 1.0f / sqrtf(sum / (float)D + a.eps);
        }
        __syncthreads();
    }

    // where the token's k and v go
    int64_t slot = -1;
    if (a.kv_heads && at >= 0) {
        const int id = a.batch.table[(int64_t)s * a.batch.stride + (at >> a.cache.page_shift)];
        if ((unsigned)id < (unsigned)a.cache.pages)
            slot = id * a.cache.page_stride + (int64_t)(at & ((1 << a.cache.page_shift) - 1)) * D;
        else if (a.flags && tid == 0)
            atomicOr(a.flags, kFlagKvPage);
    }

    const int R2 = a.rot / 2, n8 = heads * D / 8;
    const bool wide = a.interleaved ? a.rot % 8 == 0 : R2 % 8 == 0; // a thread's 8 partners lie together
    for (int i = tid; i < n8; i += ROPE_THREADS) {
        const int hl = 8 * i / D, h = h0 + hl, e0 = 8 * i % D;
        const float *xh = x + hl * D;
        float8 y = *(const float8 *)(xh + e0);
        if (h < vnob) {
            const float *w = h < knob ? a.q_norm : a.k_norm;
            const float f = w ? inv[hl] : 1.0f;
            if (w)
                y = y * f * *(const float8 *)(w + e0);
            if (e0 < a.rot) {
                if (a.interleaved && wide) {
#pragma unroll
                    for (int u = 0; u < 8; u += 2) {
                        const float2 c = cs[(e0 + u) / 2];
                        const float p = y[u], q = y[u + 1];
                        y[u] = p * c.x - q * c.y;
                        y[u + 1] = p * c.y + q * c.x;
                    }
                } else if (wide) {
                    const int low = e0 < R2 ? e0 : e0 - R2, other = e0 < R2 ? e0 + R2 : low;
                    const float side = e0 < R2 ? -1.0f : 1.0f;
                    float8 z = *(const float8 *)(xh + other);
                    if (w)
                        z = z * f * *(const float8 *)(w + other);
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const float2 c = cs[low + u];
                        y[u] = y[u] * c.x + side * z[u] * c.y;
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        // (behind the rotated part: the first pair's partner, not used)
                        const bool in = e0 + u < a.rot;
                        const int e = in ? e0 + u : 0;
                        const bool left = a.interleaved ? e % 2 == 0 : e < R2;
                        const int other = a.interleaved ? e ^ 1 : left ? e + R2 : e - R2;
                        const float2 c = cs[a.interleaved ? e / 2 : left ? e : e - R2];
                        float z = xh[other];
                        if (w)
                            z = z * f * w[other];
                        y[u] = in ? y[u] * c.x + (left ? -z : z) * c.y : y[u];
                    }
                }
            }
        }
        if (h < knob)
            store8(a.out, ((int64_t)token * a.q_heads + h) * D + e0, a.out_type, y);
        else if (slot >= 0) {
            const int64_t to = slot + ((int64_t)(h < vnob ? h - knob : h - vnob) << a.cache.page_shift) * D + e0;
            store8(h < vnob ? a.cache.k : a.cache.v, to, a.cache.type, y);
        }
    }
}

} // namespace

hipError_t launch_rope_kv(RopeArgs a, hipStream_t s)
{
    const int heads = a.q_heads + 2 * a.kv_heads;
    int hb = ROPE_FLOATS / a.dim < ROPE_HEADS ? ROPE_FLOATS / a.dim : ROPE_HEADS;
    // few tokens: one 16-byte load a thread, spread over more workgroups (us, spread
    // against not: 1 token 4.6, 4.9; 61 5.0, 5.9; 128 4.7, 4.6; 1000 14.7, 11.0)
    const int small = ROPE_THREADS * 4 / a.dim;
    if ((int64_t)a.batch.tokens * ((heads + hb - 1) / hb) < 2 * device_cus())
        hb = small < hb ? small : hb;
    a.hb = hb;
    a.blocks = (heads + hb - 1) / hb;
    hipLaunchKernelGGL(k_rope_kv, dim3((uint32_t)a.batch.tokens * (uint32_t)a.blocks), dim3(ROPE_THREADS), 0, s, a);
    return hipGetLastError();
}

} // namespace ihip
