// gd_common.h -- the sequences of a batch whose layers keep a state instead of
// a cache, shared by the kernels of gd_conv.hip, gd_step.hip and gd_chunk.hip.
//
// Every sequence owns a slot of a layer's pool of states.  The batch's arrays lie
// in device memory, so a kernel looks its sequence up itself; values that do not
// fit the batch's sizes are cut to them, or the sequence is left out, so that no
// index formed from them leaves the buffers.
#pragma once

#include "gd_plan.h"
#include "kq_common.h"
#include "kv_common.h"

namespace ihip {

constexpr int kMaxDeltaDim = 128;            // of a head's keys and values
constexpr uint32_t kFlagStateSlot = 64;      // IHIP_FLAG_STATE_SLOT

struct StateBatch {
    const int32_t *starts, *lens, *slots;
    int sequences, tokens;
};

// A sequence as the kernels see it: its rows start .. start + n - 1, its slot
// (-1: it is left out) and whether it begins with this call, so that what its slot
// holds is not read.
struct GdSeq {
    int start, n, slot;
    bool begins;
};

__device__ __forceinline__ int2 gd_rows(const StateBatch &b, int s)
{
    const int start = kv_clamp(b.starts[s], 0, b.tokens);
    return make_int2(start, kv_clamp(b.starts[s + 1], start, b.tokens) - start);
}

// Sequence s.  A slot that an earlier sequence with new tokens holds too is not
// s's: two that wrote one state would race.  The lanes of a wave look at 64 earlier
// sequences at a time, all of them in flight beside s's own values (up to 64
// sequences: one round of loads).  All lanes must be active.
__device__ __forceinline__ GdSeq gd_seq(const StateBatch &b, int pool, int s, uint32_t *flags)
{
    GdSeq q;
    const int2 r = gd_rows(b, s);
    q.start = r.x, q.n = r.y;
    q.slot = b.slots[s];
    const int len = b.lens ? b.lens[s] : q.n + 1;
    q.begins = len <= q.n;
    bool twice = false;
    for (int e = threadIdx.x & 63; e < s; e += 64)
        twice |= b.slots[e] == q.slot && gd_rows(b, e).y > 0;
    const bool bad = (unsigned)q.slot >= (unsigned)pool || __ballot(twice);
    if (flags && threadIdx.x == 0 && bad && q.n > 0)
        atomicOr(flags, kFlagStateSlot);
    if (bad)
        q.slot = -1;
    return q;
}

// Reports the sequences whose rows had to be cut, or that have more new tokens than
// tokens.  One workgroup of a call calls it.
__device__ __forceinline__ void gd_report(const StateBatch &b, uint32_t *flags)
{
    for (int s = threadIdx.x; s < b.sequences; s += blockDim.x) {
        const int2 r = gd_rows(b, s);
        if (b.starts[s] != r.x || b.starts[s + 1] != r.x + r.y || (b.lens && b.lens[s] < r.y))
            atomicOr(flags, kFlagKvLength);
    }
}

// The tiles of 2^shift rows that the sequences' rows are taken in are numbered so
// that a tile's sequence can be found without sums over the sequences before:
// tile c of sequence s is (start >> shift) + s + c.  As start does not decrease,
// no two tiles have one number; some numbers have no tile, and they end below
// gd_tiles(): floor(start / m) + floor((n - 1) / m) <= floor((start + n - 1) / m).
__device__ __forceinline__ int gd_base(const StateBatch &b, int shift, int s)
{
    return (kv_clamp(b.starts[s], 0, b.tokens) >> shift) + s;
}

// The sequence of tile `tile` (-1: none has it) and the tile's place c in it: the
// last sequence that does not start behind it.  All lanes must be active.
__device__ __forceinline__ int gd_find(const StateBatch &b, int shift, int tile, int &c)
{
    int s = -1;
    for (int s0 = 0; s0 < b.sequences; s0 += 64) {
        const int e = s0 + (threadIdx.x & 63);
        const uint64_t not_behind = __ballot(e < b.sequences && gd_base(b, shift, e) <= tile);
        if (!not_behind)
            break;
        s = s0 + 63 - __builtin_clzll(not_behind);
    }
    if (s < 0)
        return -1;
    c = tile - gd_base(b, shift, s);
    return c >= 0 && ((int64_t)c << shift) < gd_rows(b, s).y ? s : -1;
}

// ---- values of fp32, fp16 or bf16 --------------------------------------------
typedef float gd_f4 __attribute__((ext_vector_type(4)));
typedef _Float16 gd_h4 __attribute__((ext_vector_type(4)));
typedef __bf16 gd_b4 __attribute__((ext_vector_type(4)));

// Values of one type, 1 or 4 neighbours, as they lie in memory and as fp32.  The type is
// the kernels' parameter: looked at beside every load, it would have each of them wait
// for the one before.
template <int TYPE>
struct GdType;
template <>
struct GdType<kF32> {
    typedef float T;
    typedef gd_f4 T4;
};
template <>
struct GdType<kF16> {
    typedef _Float16 T;
    typedef gd_h4 T4;
};
template <>
struct GdType<kBF16> {
    typedef __bf16 T;
    typedef gd_b4 T4;
};
template <int TYPE>
__device__ __forceinline__ typename GdType<TYPE>::T4 gd_raw4(const void *base, int64_t at)
{
    return *(const typename GdType<TYPE>::T4 *)((const typename GdType<TYPE>::T *)base + at);
}
template <typename T4>
__device__ __forceinline__ gd_f4 gd_wide(T4 v)
{
    return __builtin_convertvector(v, gd_f4);
}

// 4 neighbours, rounded once to the type they are kept in (to nearest)
__device__ __forceinline__ void gd_store4(void *base, int64_t at, int type, gd_f4 v)
{
    if (type == kF32)
        *(gd_f4 *)((float *)base + at) = v;
    else if (type == kF16)
        *(gd_h4 *)((_Float16 *)base + at) = __builtin_convertvector(v, gd_h4);
    else
        *(gd_b4 *)((__bf16 *)base + at) = __builtin_convertvector(v, gd_b4);
}

__device__ __forceinline__ float gd_silu(float x)
{
    return x / (1.0f + expf(-x));
}

// ---- sums over lanes ------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float gd_add_dpp(float v)
{
    return dpp_add<CTRL, 0xf>(v);
}
// v + the value 16 (32) lanes on or back
__device__ __forceinline__ float gd_add16(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float gd_add32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The larger of v and the value 16 (32) lanes on or back
__device__ __forceinline__ float gd_max16(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float gd_max32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ double gd_wave_sum(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
        v += __shfl_xor(v, d);
    return v;
}

// A head's outputs of a token, LANES (16 or 32) neighbouring lanes with 4 each (zeros behind the
// last column), divided by sqrt(their mean square + eps).  The squares of fp32 values pass its
// range: they are formed of values times a power of two that makes the largest one 1 to 2.
// Smaller ones than 1 stay as they are, where eps is over all that their squares could lose.
template <int LANES>
__device__ __forceinline__ gd_f4 gd_rms(gd_f4 o, int v_dim, float eps)
{
    // (the order of whole numbers is that of their sizes)
    uint32_t most = max(max(__float_as_uint(fabsf(o.x)), __float_as_uint(fabsf(o.y))),
                        max(__float_as_uint(fabsf(o.z)), __float_as_uint(fabsf(o.w))));
    most = dpp_max_u32<0xb1, 0xf>(most);  // quad_perm [1,0,3,2]
    most = dpp_max_u32<0x4e, 0xf>(most);  // quad_perm [2,3,0,1]
    most = dpp_max_u32<0x141, 0xf>(most); // row_half_mirror
    most = dpp_max_u32<0x140, 0xf>(most); // row_mirror
    if (LANES == 32) {
        const auto both = __builtin_amdgcn_permlane16_swap(most, most, false, false);
        most = max(both[0], both[1]);
    }
    const int e = max((int)(most >> 23) - 127, eps > 0x1p-100f ? 0 : -100);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = ldexpf(o[i], -e);
    float sum = (o.x * o.x + o.y * o.y) + (o.z * o.z + o.w * o.w);
    sum = gd_add_dpp<0xb1>(sum);
    sum = gd_add_dpp<0x4e>(sum);
    sum = gd_add_dpp<0x141>(sum);
    sum = gd_add_dpp<0x140>(sum);
    if (LANES == 32)
        sum = gd_add16(sum);
    return o * (1.0f / sqrtf(sum / (float)v_dim + ldexpf(eps, -2 * e)));
}

// A token's decay, in logarithms: decay * softplus(a + dt_bias).  A rate above 0 would
// let the state grow without bound and is taken as 0; below e^-10000 nothing is left
// in any type, and sums of such logarithms still hold their differences in 64 bits.
__device__ __forceinline__ float gd_log_decay(float decay, float a, float dt_bias)
{
    const float x = a + dt_bias;
    const float g = decay * (x > 20.0f ? x : log1pf(expf(x))); // (e^-20 is under half a step of 20)
    return g > 0.0f ? 0.0f : g < -1e4f ? -1e4f : g;
}
__device__ __forceinline__ float gd_beta(float b)
{
    return 1.0f / (1.0f + expf(-b));
}

} // namespace ihip
