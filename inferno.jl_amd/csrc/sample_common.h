// sample_common.h -- a row's settings and weights, shared by the kernels of
// sample.hip, and their launcher.
#pragma once

#include "gd_common.h"
#include "sample_plan.h"

namespace ihip {

constexpr uint32_t kSampleNan = 1, kSamplePosInf = 2, kSampleAllNegInf = 4; // IHIP_FLAG_*
constexpr uint32_t kSampleFinite = 8;                                       // (within the kernels)

struct SampleArgs {
    const void *logits;
    int type, rows, vocab;
    int64_t row_step; // elements from one row to the next
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    int32_t *tokens;
    float *logprobs;
    uint32_t *flags;
    uint8_t *work;
    SamplePlan plan;
    int row0; // of the launch's rows
};
hipError_t launch_sample(SampleArgs a, hipStream_t s);

struct SampleRow {
    float t, p, min_p, u;
    int k;
};

__device__ __forceinline__ SampleRow sample_row(const SampleArgs &a, int row)
{
    SampleRow r;
    r.t = a.temperature ? a.temperature[row] : 1.0f;
    r.k = a.top_k ? a.top_k[row] : 0;
    r.p = a.top_p ? a.top_p[row] : 1.0f;
    r.min_p = a.min_p ? a.min_p[row] : 0.0f;
    r.u = a.u[row];
    return r;
}

__device__ __forceinline__ float sample_logit(const void *p, int64_t i, int type)
{
    return type == kF32 ? ((const float *)p)[i]
         : type == kF16 ? (float)((const _Float16 *)p)[i] : (float)((const __bf16 *)p)[i];
}

// A whole number in the order of the logits (-0 and 0 alike), and back.
__device__ __forceinline__ uint32_t sample_key(float l)
{
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sample_value(uint32_t k)
{
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ uint32_t sample_flags(float l)
{
    return l != l ? kSampleNan : l == __builtin_inff() ? kSamplePosInf : l == -__builtin_inff() ? 0 : kSampleFinite;
}

// w = 2^(rate (l - most) / 32), and as a whole number of units of which 2^bits make 1, so
// that a row's sums fit 63 bits.
struct SampleScale {
    double rate, most;
    int bits;
};

__device__ __forceinline__ SampleScale sample_scale(float t, float most, int vocab)
{
    return SampleScale{32 * 1.4426950408889634074 / (double)t, (double)most, min(46, 62 - (32 - __builtin_clz(vocab)))};
}

// 2^(i / 32), in every workgroup's LDS; filled before its first barrier
__device__ __forceinline__ double *sample_table()
{
    __shared__ double table[32];
    return table;
}
__device__ __forceinline__ void sample_fill_table()
{
    if (threadIdx.x < 32)
        sample_table()[threadIdx.x] = exp2((double)threadIdx.x / 32);
}

// 2^(x / 32) for x <= 0: x to the nearest whole number, whose power of two is in the
// table, and the rest, |f| <= 1/2, by the series of 2^(f / 32), whose own rest is below 2^-48.
// 0 from 2^-1075 on.  (Without the table the series takes six operations more, of 20 in 64
// bits: sums of 256 rows of 151936 logits 50 us, 46 with it.)
__device__ __forceinline__ double sample_exp2_32(double x)
{
    x = fmax(x, -1100.0 * 32);
    constexpr double WHOLE = 6755399441055744.0; // 1.5 * 2^52: a sum with it is whole
    const double s = x + WHOLE, f = x - (s - WHOLE);
    const int n = (int)(uint32_t)__double_as_longlong(s);
    constexpr double L = 0.69314718055994530942 / 32;
    // L^i / i!
    constexpr double c[6] = {1.0, L, L * L / 2, L * L * L / 6, L * L * L * L / 24, L * L * L * L * L / 120};
    double y = c[5];
#pragma unroll
    for (int i = 4; i >= 0; --i)
        y = fma(y, f, c[i]);
    return ldexp(y * sample_table()[n & 31], n >> 5);
}

// (-infinity, and a rate of 0 times it, become -1100)
__device__ __forceinline__ double sample_weight(const SampleScale &s, float l)
{
    return sample_exp2_32(s.rate * ((double)l - s.most));
}

__device__ __forceinline__ uint64_t sample_mass(const SampleScale &s, float l)
{
    return (uint64_t)rint(ldexp(sample_weight(s, l), s.bits));
}

// u as it is used: below 0 and NaN as 0, and 1 or more as what no sum passes
__device__ __forceinline__ double sample_u(float u)
{
    return !(u > 0.0f) ? 0.0 : u >= 1.0f ? 2.0 : (double)u;
}

__device__ __forceinline__ void sample_done(const SampleArgs &a, int row, uint32_t fl, int token, double logprob)
{
    const uint32_t bad = fl & (kSampleNan | kSamplePosInf);
    a.tokens[row] = bad ? 0 : token;
    if (a.logprobs)
        a.logprobs[row] = bad ? __builtin_nanf("") : (float)logprob;
    if (a.flags)
        a.flags[row] = bad ? bad : (fl & kSampleFinite) ? 0 : kSampleAllNegInf;
}

} // namespace ihip
