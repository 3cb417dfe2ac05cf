// kv_attn.hip -- attention of each sequence's new tokens over its pages of the
// cache.
//
// For a row (a new token at cache position p, a q head) and the keys j of its
// sequence that it sees,
//
//   s_j = scale q.k_j,  s_j <- cap tanh(s_j / cap),  s_j <- s_j - slope |p - j|
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),    m = max_j s_j
//
// in one pass over the keys with the running m and sum (32 bits); a row that
// sees no key gives 0.  The rows of a tile are those of one KV head's group of
// q heads, token by token, so that a key that is read serves all of them.
//
// The weights are powers of two, 2^((s_j - m) by): m is kept in the units of the
// products, and only differences are multiplied, so that scores of any size give
// the weights that their differences say.  (fma(s_j, by, -m by) is one operation a
// score less, but from scores of 2e7 on it rounds m by more than the room that p
// has in fp16, and gives NaN or wrong weights.  us, this against that: 4096 tokens
// over 32768 keys 2440, 2388; 2048 over 8192, 64 wide 200, 193, 128 wide 297, 289,
// with a bias 328, 321; fp32 rows over bf16 730, 714; one token the same.)
//
// Both products run on the matrix cores, transposed: S^T = K Q^T puts a row's
// scores in the lanes of one column, so that maxima and sums stay in a lane but
// for one exchange between lane groups, and leaves P^T in the registers that
// the second product, O^T = V^T P^T, takes it from.  V^T's operand is read from
// LDS through the transposing read (a 4 x 16 block a 16-lane group).
//
// Operands: q of the cache's type is multiplied as it is and p is rounded once
// to that type (off by 2^-11 / 2^-8 of itself at most, like
// the output in its own rounding).  An fp32 q keeps fp32's accuracy: q and p are
// split into 2 fp16 parts (22 bits) or 3 bf16 parts (24 bits), whose products
// with K and V are exact in the fp32 sums.
#include "kq_common.h"
#include "kv_launch.h"

namespace ihip {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The two cache types: vectors, products, the transposing read.
struct Half {
    typedef _Float16 T;
    typedef h2 V2;
    typedef h4 V4;
    typedef h8 V8;
    // p = e^(s - m) is carried times 2^14 by k_attn_rows: what fp16 keeps of small
    // ones reaches down to 2^-38 of the largest (k_attn_chunk: see kUp there)
    static constexpr float kShift = 14.0f;
    static constexpr uint32_t kExp = 0x7c007c00u;
    static __device__ __forceinline__ f4 mfma16(V8 a, V8 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f16v mfma32(V8 a, V8 b, f16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
struct BHalf {
    typedef __bf16 T;
    typedef b2 V2;
    typedef b4 V4;
    typedef b8 V8;
    static constexpr float kShift = 0.0f;
    static constexpr uint32_t kExp = 0x7f807f80u;
    static __device__ __forceinline__ f4 mfma16(V8 a, V8 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f16v mfma32(V8 a, V8 b, f16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

template <typename V4>
__device__ __forceinline__ V4 read_tr(const uint8_t *lds)
{
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)lds));
}

// The same by LDS byte address, and a plain read.
template <typename V>
__device__ __forceinline__ V read_lds(uint32_t at)
{
    return *(const __attribute__((address_space(3))) V *)at;
}
template <typename V4>
__device__ __forceinline__ V4 read_tr_at(uint32_t at)
{
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at));
}

// Whether any of the 16-bit values in a dword is an infinity or a NaN.
template <typename C>
__device__ __forceinline__ bool odd_value(uint32_t w)
{
    constexpr uint32_t lo = C::kExp & 0xffffu, hi = C::kExp & 0xffff0000u;
    return (w & lo) == lo || (w & hi) == hi;
}

// The two 16-bit values of a dword, 0 in the place of an infinity or a NaN.
template <typename C>
__device__ __forceinline__ uint32_t without_odd(uint32_t w)
{
    constexpr uint32_t lo = C::kExp & 0xffffu, hi = C::kExp & 0xffff0000u;
    return ((w & lo) == lo ? 0u : w & 0xffffu) | ((w & hi) == hi ? 0u : w & 0xffff0000u);
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNone = -__builtin_inff();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// max / sum over the four 16-lane groups of a wave (lanes of one column)
__device__ __forceinline__ float groups_max(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float halves_max(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float halves_sum(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Two floats passed between workgroups of different XCDs, whose caches do not
// follow each other: relaxed atomics of the whole device, which go to memory.
__device__ __forceinline__ void put_shared(uint64_t *p, float a, float b)
{
    __hip_atomic_store(p, (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 get_shared(const uint64_t *p)
{
    const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return f2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

// Four values of a row over its parts `from`, `from` + `by`, ... of n: their sum
// (relative to `top`, as `sum` is), eight parts at a time with their maxima and
// sums; `rows` rows lie between a row's parts; `by` makes a difference of maxima a
// power of two.
struct Joined {
    float top, sum;
    f4 v;
    __device__ __forceinline__ void add(float top2, float sum2, f4 v2, float by)
    {
        const float up = fmaxf(top, top2);
        const float f = top == kNone ? 0.0f : exp2_fast((top - up) * by);
        const float g = top2 == kNone ? 0.0f : exp2_fast((top2 - up) * by);
        sum = sum * f + sum2 * g;
        v = v * f + v2 * g;
        top = up;
    }
};
__device__ __forceinline__ Joined join_parts(const uint64_t *o, const uint64_t *ml, int64_t rows, int dim, int from,
                                             int step, int n, float by)
{
    constexpr int AT_ONCE = 8;
    Joined j{kNone, 0.0f, f4{}};
    for (int p0 = AT_ONCE * from; p0 < n; p0 += AT_ONCE * step) {
        f2 w[AT_ONCE], x[AT_ONCE], y[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int64_t p = min(p0 + u, n - 1) * rows;
            w[u] = get_shared(ml + p);
            x[u] = get_shared(o + p * dim / 2);
            y[u] = get_shared(o + p * dim / 2 + 1);
        }
        float up = j.top;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            up = p0 + u < n ? fmaxf(up, w[u].x) : up;
        const float f = j.top == kNone ? 0.0f : exp2_fast((j.top - up) * by);
        j.sum *= f;
        j.v *= f;
        j.top = up;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            if (p0 + u < n && w[u].y != 0.0f) { // (sum 0: a part without keys has written nothing else; NaN stays)
                const float g = w[u].x == kNone ? 0.0f : exp2_fast((w[u].x - up) * by);
                j.sum += w[u].y * g;
                j.v += f4{x[u].x, x[u].y, y[u].x, y[u].y} * g;
            }
    }
    return j;
}

// What the scores go through, each a kernel of its own: the registers of a cap
// would cost the others a wave a SIMD (64 wide: 38 us against 34 for five ragged
// chunks).
constexpr int kPlain = 0, kBias = 1, kCap = 2; // (kCap: with a bias or without)

// What a workgroup works on: a tile of rows of one sequence and KV head, and
// the part of its keys.
struct Tile {
    int head;                // KV head
    int start, row0, rows;   // the sequence's first token; the tile's first row in it; its rows
    int first, last;         // cache positions of the tile's first and last token
    int len, prefix;         // keys there are; keys every row sees
    int lo, hi;              // keys to look at (lo a multiple of the step); lo >= hi: none
    int split, parts;        // the part of its keys, of how many that have any (1 at least)
    int index;               // its place among all tiles and heads
    const int32_t *table;
};

// Workgroup `bid`'s tile; false if there is none.  Tiles are counted over the
// sequences in order; their number is only known here, the grid holds the most
// there can be.
template <int ROWS, int KEYS>
__device__ __forceinline__ bool find_tile(const AttnArgs &a, int tiles, int least, int splits, int bid, Tile &t)
{
    if (bid == 0 && a.flags)
        kv_report(a.batch, a.cache.page_shift, a.flags);
    t.head = bid % a.cache.heads;
    const int rest = bid / a.cache.heads;
    // (a prompt's last rows have the most keys: they go first)
    int want = tiles - 1 - rest % tiles;
    t.split = rest / tiles;
    int first = 0;
    KvSeq q;
    const int s = kv_find<false>(a.batch, a.cache.page_shift, want, first, q,
                          [&](int n) { return (int)(((int64_t)n * a.group + ROWS - 1) / ROWS); });
    if (s < 0)
        return false;
    t.start = q.start;
    t.row0 = (want - first) * ROWS;
    t.rows = min(ROWS, (int)((int64_t)q.n * a.group - t.row0));
    t.len = q.len;
    t.first = q.len - q.n + t.row0 / a.group;
    t.last = q.len - q.n + (t.row0 + t.rows - 1) / a.group;
    t.prefix = a.prefix ? kv_clamp(a.prefix[s], 0, q.len) : 0;
    t.table = a.batch.table + (int64_t)s * a.batch.stride;
    const int lo = a.window ? max(0, t.first - a.window + 1) & ~(KEYS - 1) : 0;
    const int hi = max(t.last + 1, t.prefix);
    // the split's part of the keys: a fixed number, or more where the most
    // splits there may be would not reach the end
    const int keys = max(0, hi - lo);
    const int per = max(least, (int)(((int64_t)keys + splits - 1) / splits + 127) & ~127);
    t.parts = max(1, (int)(((int64_t)keys + per - 1) / per));
    t.index = want * a.cache.heads + t.head;
    const int64_t from = (int64_t)lo + (int64_t)t.split * per;
    t.lo = (int)min(from, (int64_t)hi);
    t.hi = (int)min(from + per, (int64_t)hi);
    return true;
}

// The keys that position p sees: `from` .. `from` + count - 1.
struct Seen {
    int from;
    uint32_t count;
    __device__ __forceinline__ bool operator()(int j) const { return (uint32_t)(j - from) < count; }
};
__device__ __forceinline__ Seen seen_from(const AttnArgs &a, const Tile &t, int p)
{
    const int last = min(max(p, t.prefix - 1), t.len - 1);
    const int from = a.window ? max(p - a.window + 1, 0) : 0;
    return Seen{from, last >= from ? (uint32_t)(last - from) + 1u : 0u};
}

// tanh x by its Taylor series, to x^11 for |x| <= 0.35 and to x^15 for |x| < 1/2
// (what is left out is under 2^-26 of x), and as (e^2x - 1) / (e^2x + 1) from there.
// Capped scores are mostly a small part of their cap: a wave whose scores all are
// takes the short series alone (8 operations a score against 23).
constexpr float kNear = 0.35f;
__device__ __forceinline__ float tanh_near(float x)
{
    const float y = x * x;
    float p = -1382.0f / 155925.0f;
    p = fmaf(p, y, 62.0f / 2835.0f);
    p = fmaf(p, y, -17.0f / 315.0f);
    p = fmaf(p, y, 2.0f / 15.0f);
    p = fmaf(p, y, -1.0f / 3.0f);
    return fmaf(p * y, x, x);
}
__device__ __forceinline__ float tanh_any(float x)
{
    const float y = x * x;
    float p = -929569.0f / 638512875.0f;
    p = fmaf(p, y, 21844.0f / 6081075.0f);
    p = fmaf(p, y, -1382.0f / 155925.0f);
    p = fmaf(p, y, 62.0f / 2835.0f);
    p = fmaf(p, y, -17.0f / 315.0f);
    p = fmaf(p, y, 2.0f / 15.0f);
    p = fmaf(p, y, -1.0f / 3.0f);
    const float small = fmaf(p * y, x, x);
    const float e = exp2_fast(fminf(2.0f * kLog2e * fabsf(x), 64.0f));
    const float large = copysignf((e - 1.0f) * __builtin_amdgcn_rcpf(e + 1.0f), x);
    return y < 0.25f ? small : x == x ? large : x;
}

// A factor that may have passed the largest number: 0 times it stays 0.
__device__ __forceinline__ float finite(float x)
{
    return __builtin_isinf(x) ? copysignf(3.402823466e38f, x) : x;
}
__device__ __forceinline__ float power_of_two(int e) { return finite(__builtin_ldexpf(1.0f, e)); }

// q's part of a lane: KS chunks of 8 values (chunk step i + offset of the row),
// in PARTS parts, with the sign of the scale (which then is positive, so that
// the largest product gives the largest score; 0 makes q 0).  Parts are taken of q
// times 2^up, which brings the row's largest value to [2^14, 2^15): fp16 holds it
// then, and no part of either type is lost below the type's smallest numbers (rows
// that the scale leaves under 2^-85 lose bits that no score would show).
template <typename C, int PARTS, int KS>
__device__ __forceinline__ void load_q(const AttnArgs &a, int64_t row, bool live, int step, int offset,
                                       typename C::V8 (&qf)[PARTS][KS], int &up)
{
    typedef typename C::V8 V8;
    up = 0;
    const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
    if constexpr (PARTS == 1) {
        const typename C::T *q = (const typename C::T *)a.q + row * a.cache.dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int c = (step * i + offset) * 8;
            qf[0][i] = live && c < a.cache.dim ? *(const V8 *)(q + c) : V8{};
            if (sign != 1.0f)
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    qf[0][i][u] = (typename C::T)((float)qf[0][i][u] * sign);
        }
    } else {
        const float *q = (const float *)a.q + row * a.cache.dim;
        f4 v[2 * KS];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int c = (step * i + offset) * 8;
            const bool in = live && c < a.cache.dim;
            v[2 * i] = in ? *(const f4 *)(q + c) : f4{};
            v[2 * i + 1] = in ? *(const f4 *)(q + c + 4) : f4{};
#pragma unroll
            for (int u = 0; u < 4; ++u)
                most = fmaxf(most, fmaxf(fabsf(v[2 * i][u]), fabsf(v[2 * i + 1][u])));
        }
        most = step == 4 ? groups_max(most) : halves_max(most);
        if (most > 0.0f && most < __builtin_inff())
            up = min(15 - __builtin_amdgcn_frexp_expf(most), a.scale_exp + 100);
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float x = __builtin_ldexpf(v[2 * i + u / 4][u % 4] * sign, up);
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const typename C::T y = (typename C::T)x;
                    qf[part][i][u] = y;
                    x -= (float)y;
                }
            }
    }
}

// ---- few rows: one token, or a few drafted ones ------------------------------
// V's 16-byte chunk c of key row r lies at chunk c ^ swizzle(r): the four rows
// (and both of their chunks) that a transposing read takes from then lie in
// different banks.
template <int NC>
__device__ __forceinline__ int v_chunk(int r, int c)
{
    return NC == 8 ? c ^ (2 * ((r >> 1) & 3)) : c ^ (2 * (r & 7));
}

template <int DP>
constexpr int ar_wave_lds()
{
    return AR_ROWS * (DP + 4) * 4 > 2 * AR_KEYS * DP * 2 ? AR_ROWS * (DP + 4) * 4 : 2 * AR_KEYS * DP * 2;
}

// A workgroup's 4 waves walk the keys of its part 32 at a time, each its own
// steps (no shared data, no barrier): K from HBM into the matrix operand's
// registers, V by direct copies into LDS of the wave's own, both one step
// ahead and their page ids two; the waves' sums are joined at the end, and the
// parts' by the workgroup that ends last.
//
// Bound by HBM where there are many keys: 32 heads on 8, 128 wide, 54 us for one
// token over 65537 fp16 keys (4.9 TB/s), 174 us for 61 bf16 sequences of up to
// 16000 (5.1 TB/s; 211 with V staged through registers instead of copied).
// Otherwise by latency: lengths, page ids, keys, and the parts' way through
// memory one after another (777 keys: 10 us; 12.2 with the join as a launch of
// its own).  16 rows a tile: the operands of a group's heads, or a few drafted
// tokens', for the same reads of K and V.
template <typename C, int PARTS, int DP, int FEAT>
__global__ void __launch_bounds__(64 * AR_WAVES, DP == 256 ? 1 : 2)
k_attn_rows(AttnArgs a, int tiles, int least, int splits)
{
    typedef typename C::T T;
    typedef typename C::V8 V8;
    typedef typename C::V4 V4;
    constexpr int KS = DP / 32, DT = DP / 16, NC = DP / 8, NI = DP / 32; // NI: copies of 1 KB for 16 keys
    constexpr int TILE = AR_KEYS * DP * 2;
    __shared__ __attribute__((aligned(16))) uint8_t lds[AR_WAVES * ar_wave_lds<DP>()];
    __shared__ float lds_m[AR_WAVES][AR_ROWS], lds_l[AR_WAVES][AR_ROWS];
    __shared__ int lds_last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int D = a.cache.dim;
    Tile t;
    if (!find_tile<AR_ROWS, AR_KEYS>(a, tiles, least, splits, blockIdx.x, t) || t.split >= t.parts)
        return;

    uint8_t *const mine = lds + wave * ar_wave_lds<DP>();
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)mine;
    const int page_mask = (1 << a.cache.page_shift) - 1;
    const int n_steps = (t.hi - t.lo + AR_KEYS - 1) / AR_KEYS;

    // a lane's byte offsets in a run of 16 keys (chunks behind a head's end hold
    // its last one: q is 0 there, and nothing reads those columns of the output)
    uint32_t koff[KS], voff[NI];
#pragma unroll
    for (int i = 0; i < KS; ++i)
        koff[i] = 2u * (uint32_t)(col * D + 8 * min(4 * i + g, D / 8 - 1));
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = (64 * i + lane) / NC, c = (64 * i + lane) % NC;
        voff[i] = 2u * (uint32_t)(r * D + 8 * min(v_chunk<NC>(r, c), D / 8 - 1));
    }

    V8 kf[2][KS];
    int ids = -1;  // page ids of the next step's runs, in lanes 0 and 1
    int ok = 0;    // bit u: run u's page is there
    int64_t at[2]; // bytes from the pools' starts to the runs
    auto page_of = [&](int step) {
        const int j = t.lo + AR_KEYS * step + 16 * (lane & 1);
        return step < n_steps && j < t.hi ? t.table[j >> a.cache.page_shift] : -1;
    };
    auto place = [&](int step) { // the runs of `step`, whose ids are here
        ok = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = t.lo + AR_KEYS * step + 16 * u;
            const int id = __builtin_amdgcn_readlane(ids, u);
            const bool in = (unsigned)id < (unsigned)a.cache.pages;
            ok |= in << u;
            at[u] = 2 * ((in ? (int64_t)id * a.cache.page_stride : 0) +
                         (int64_t)((t.head << a.cache.page_shift) + (j & page_mask)) * D);
            if (!in && j < t.hi && a.flags && lane == 0)
                atomicOr(a.flags, kFlagKvPage);
        }
    };
    auto copy_v = [&](int step) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if ((ok >> u) & 1)
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    lds_copy16_at((const uint8_t *)a.cache.v + at[u], voff[i],
                                  lds0 + TILE * ((step / AR_WAVES) & 1) + 1024 * (NI * u + i));
    };
    auto load_k = [&]() { // (a run that is not there reads page 0, whose scores are masked)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < KS; ++i)
                kf[u][i] = *(const V8 *)((const uint8_t *)a.cache.k + at[u] + koff[i]);
    };

    const int row = t.row0 + col; // the row of this lane's column
    const bool live = col < t.rows;
    const int qhead = t.head * a.group + (live ? row % a.group : 0);
    const int64_t qrow = (int64_t)(t.start + (live ? row / a.group : 0)) * a.q_heads + qhead;
    const int pos = live ? t.first - t.row0 / a.group + row / a.group : t.first;
    V8 qf[PARTS][KS];
    int up;
    int step = wave;
    if (step < n_steps)
        ids = page_of(step);
    load_q<C, PARTS, KS>(a, qrow, live, 4, g, qf, up);
    if (step < n_steps) {
        place(step);
        ids = page_of(step + AR_WAVES);
        load_k();
        copy_v(step);
    }
    // scores become powers of two with the last factor, `by`; a cap takes the scale
    // before, and the bias is added in units of `by`.  `unit`, a power of two (the
    // row's and the scale's), brings the maxima of a row's parts to one unit.
    const float unit = FEAT == kCap ? 1.0f : power_of_two(a.scale_exp - up), by = finite(a.by * unit);
    const float slope = FEAT != kPlain && a.slopes ? finite(a.slopes[qhead] * kLog2e / by) : 0.0f;
    const Seen sees = seen_from(a, t, pos);

    float m = kNone, l = 0.0f;
    f4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
        o[d] = f4{};

    for (; step < n_steps; step += AR_WAVES) {
        const int key = t.lo + AR_KEYS * step;
        const int here = ok;
        const bool whole = here == 3 && key + AR_KEYS <= t.len &&
                           (key + AR_KEYS - 1 <= t.first || key + AR_KEYS <= t.prefix) &&
                           (a.window == 0 || t.last - key < a.window);
        uint8_t *const vt = mine + TILE * ((step / AR_WAVES) & 1);
        __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0) lgkmcnt(0): V's copies, and the other half's reads
        asm volatile("" ::: "memory");
        const bool more = step + AR_WAVES < n_steps;
        if (more) {
            place(step + AR_WAVES);
            copy_v(step + AR_WAVES);
        }
        f4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = f4{};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
                    s[u] = C::mfma16(kf[u][i], qf[part][i], s[u]);
        }
        if (more) {
            ids = page_of(step + 2 * AR_WAVES);
            load_k();
        }
        if constexpr (FEAT != kPlain) {
            const float apart = (float)(pos - key - 4 * g);
            if constexpr (FEAT == kCap) {
                const float by_cap = finite(__builtin_ldexpf(a.to_cap, a.scale_exp - up));
                float most = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[u][i] *= by_cap;
                        most = fmaxf(most, fabsf(s[u][i]));
                    }
                if (__any(most > kNear)) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[u][i] = tanh_any(s[u][i]);
                } else { // (a NaN is neither, and stays)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[u][i] = tanh_near(s[u][i]);
                }
            }
            if (a.slopes)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[u][i] = fmaf(-slope, fabsf(apart - (float)(16 * u + i)), s[u][i]);
        }
        if (!whole) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[u][i] = ((here >> u) & 1) && sees(key + 16 * u + 4 * g + i) ? s[u][i] : kNone;
        }
        float mx = kNone;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                mx = fmaxf(mx, s[u][i]);
        mx = fmaxf(groups_max(mx), m);
        // (a row without a key yet keeps its sum 0 whatever is subtracted)
        const float use = mx == kNone ? 0.0f : mx;
        if (__any(mx != m)) {
            const float f = exp2_fast((m - use) * by);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                o[d] *= f;
            m = mx;
        }
        V8 pf[PARTS];
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = exp2_fast(fmaf(s[u][i] - use, by, C::kShift));
                s[u][i] = x;
                sum += x;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const T y = (T)x;
                    pf[part][4 * u + i] = y;
                    x -= (float)y;
                }
            }
        l += sum;

        // of a step with hidden keys, the rows of V that no row of the tile sees are
        // cleared (nothing may come from them, whatever they hold)
        bool odd = false;
        if (!whole)
            for (int i = lane; i < AR_KEYS * NC; i += 64) {
                const int r = i / NC, j = key + r;
                if (((here >> (r >> 4)) & 1) && j < t.len && (j <= t.last || j < t.prefix) &&
                    (a.window == 0 || t.first - j < a.window)) {
                    const u4 w = *(const u4 *)(vt + 16 * i);
                    odd |= odd_value<C>(w.x) || odd_value<C>(w.y) || odd_value<C>(w.z) || odd_value<C>(w.w);
                } else {
                    *(u4 *)(vt + 16 * i) = u4{};
                }
            }
        asm volatile("" ::: "memory");
        if (__builtin_expect(!whole && __any(odd), 0)) {
            // infinities or NaNs that some rows of the tile see and others do not:
            // 0 times them must not reach the others.  They are added one key at a
            // time where a row has a weight for them, and the products take 0.
#pragma unroll 1
            for (int j = 0; j < AR_KEYS; ++j) {
                const int i = j & 3, u = j >> 4;
                float x = u ? (i == 0 ? s[1][0] : i == 1 ? s[1][1] : i == 2 ? s[1][2] : s[1][3])
                            : (i == 0 ? s[0][0] : i == 1 ? s[0][1] : i == 2 ? s[0][2] : s[0][3]);
                x = __shfl(x, col + 16 * ((j >> 2) & 3));
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const V4 v = *(const V4 *)(vt + j * (DP * 2) + v_chunk<NC>(j, 2 * d + (g >> 1)) * 16 + 8 * (g & 1));
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        o[d][q] += x != 0.0f && !__builtin_isfinite((float)v[q]) ? x * (float)v[q] : 0.0f;
                }
            }
            asm volatile("" ::: "memory");
            for (int i = lane; i < AR_KEYS * DP / 2; i += 64)
                ((uint32_t *)vt)[i] = without_odd<C>(((const uint32_t *)vt)[i]);
            asm volatile("" ::: "memory");
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int r = 4 * g + (col >> 2), c = 2 * d + ((col & 3) >> 1);
            const V4 lo = read_tr<V4>(vt + r * (DP * 2) + v_chunk<NC>(r, c) * 16 + 8 * (col & 1));
            const V4 hi = read_tr<V4>(vt + (r + 16) * (DP * 2) + v_chunk<NC>(r + 16, c) * 16 + 8 * (col & 1));
            const V8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
                o[d] = C::mfma16(v, pf[part], o[d]);
        }
        asm volatile("" ::: "memory");
    }

    // the waves' sums, in wave order
    l = groups_sum(l);
    asm volatile("" ::: "memory");
    float *const ol = (float *)mine;
#pragma unroll
    for (int d = 0; d < DT; ++d)
        *(f4 *)(ol + col * (DP + 4) + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        lds_m[wave][col] = m * unit;
        lds_l[wave][col] = l;
    }
    __syncthreads();
    const int64_t rows_all = (int64_t)a.batch.tokens * a.q_heads;
    auto row_of = [&](int r) {
        const int rr = t.row0 + r;
        return (int64_t)(t.start + rr / a.group) * a.q_heads + t.head * a.group + rr % a.group;
    };
    auto finish = [&](int r, int d, f4 v, float sum) {
        v = sum == 0.0f ? f4{} : v * (1.0f / sum);
        if constexpr (PARTS == 1)
            *(V4 *)((T *)a.out + row_of(r) * D + d) = __builtin_convertvector(v, V4);
        else
            *(f4 *)((float *)a.out + row_of(r) * D + d) = v;
    };
    // a part's rows lie in a.part, their maxima and sums behind
    uint64_t *const part_o = (uint64_t *)a.part;
    uint64_t *const part_ml = part_o + (int64_t)splits * rows_all * D / 2;
    const int items = t.rows * (D / 4);
    for (int e = tid; e < items; e += 64 * AR_WAVES) {
        const int r = e / (D / 4), d = 4 * (e % (D / 4));
        float top = kNone;
#pragma unroll
        for (int w = 0; w < AR_WAVES; ++w)
            top = fmaxf(top, lds_m[w][r]);
        float sum = 0.0f;
        f4 v = f4{};
#pragma unroll
        for (int w = 0; w < AR_WAVES; ++w) {
            const float f = lds_m[w][r] == kNone ? 0.0f : exp2_fast((lds_m[w][r] - top) * a.by);
            const f4 x = *(const f4 *)(lds + w * ar_wave_lds<DP>() + 4 * (r * (DP + 4) + d));
            sum += lds_l[w][r] * f;
            v += x * f;
        }
        if (t.parts == 1) {
            finish(r, d, v, sum);
        } else {
            const int64_t to = t.split * rows_all + row_of(r);
            put_shared(part_o + (to * D + d) / 2, v.x, v.y);
            put_shared(part_o + (to * D + d) / 2 + 1, v.z, v.w);
            if (d == 0)
                put_shared(part_ml + to, top, sum);
        }
    }
    if (t.parts == 1)
        return;

    // The workgroup that is the last of its tile's to come here joins the parts, in
    // their order.  Everything that passes between workgroups goes through memory
    // that all of the chip sees (put_shared, get_shared); a workgroup counts itself
    // when its stores have arrived, and the last one sets the count to 0 again.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
        lds_last = atomicInc(a.count + t.index, (uint32_t)t.parts - 1) == (uint32_t)t.parts - 1;
    __syncthreads();
    if (!lds_last)
        return;
    // four values of a row a thread; few rows: the parts are shared among groups of
    // threads, which are joined in the groups' order
    const int groups = max(1, 64 * AR_WAVES / items);
    Joined *const lds_g = (Joined *)lds;
    for (int e0 = 0; e0 < items; e0 += 64 * AR_WAVES) {
        const int group = groups > 1 ? tid / items : 0;
        const int e = groups > 1 ? tid - group * items : e0 + tid;
        const bool in = group < groups && e < items;
        const int r = in ? e / (D / 4) : 0, d = in ? 4 * (e % (D / 4)) : 0;
        Joined j = join_parts(part_o + (row_of(r) * D + d) / 2, part_ml + row_of(r), rows_all, D, group, groups,
                              in ? t.parts : 0, a.by);
        if (groups > 1) {
            if (in && group > 0)
                lds_g[tid] = j;
            __syncthreads();
            if (!in || group > 0)
                return;
            for (int q = 1; q < groups; ++q)
                j.add(lds_g[tid + q * items].top, lds_g[tid + q * items].sum, lds_g[tid + q * items].v, a.by);
        }
        if (in)
            finish(r, d, j.v, j.sum);
    }
}

// ---- many rows: chunks of a prompt ---------------------------------------------
// Operands read from LDS some products ahead, where the registers allow it.  us,
// ahead against not, 2048 rows of 32 heads over 8192 keys, 1 part: 64 wide 200, 213,
// with a bias 232, 243, with a cap 278, 280; 128 wide 296, 308, with a bias 328, 343,
// with a cap 494, 384 (it spills); 256 wide 711, 867, with a bias 865, 997, with a
// cap 1417, 996.  2 parts: 64 wide 291, 302; 128 wide 458, 466, with a cap 808, 545;
// 256 wide 2126, 1263.  3 parts: 128 wide 730, 731, with a bias 819, 846, with a cap
// 842, 897; 256 wide 3219, 1637.
constexpr bool ac_ahead(int parts, int dp, int feat)
{
    return dp <= 64 || (feat == kCap ? parts == 3 && dp <= 128 : parts == 1 || dp <= 128);
}
// K's operands on their way before the first product (2 parts, 128 wide: a
// 2048-token prompt 96.4 us with 2, 97.7 with 8; the others have the room).
constexpr int ac_first(int parts, int dp) { return parts == 2 && dp == 128 ? 2 : dp <= 64 ? dp / 16 : 8; }

// Where 16-byte chunk c of key row r lies in its row of LDS: K's so that the 16
// rows of a matrix operand's read lie in different banks, V's so that the four
// rows and 64 bytes of a pair of transposing reads do.
template <int NC>
__device__ __forceinline__ int ac_k_chunk(int r, int c)
{
    return NC == 8 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
}
template <int NC>
__device__ __forceinline__ int ac_v_chunk(int r, int c)
{
    return NC == 8 ? c ^ (4 * ((r >> 1) & 1)) : c ^ (4 * (r & 3));
}

// Four waves hold 32 rows each; where HALVES is 2, a second four hold the same
// rows for the second half of a step's keys, and the halves' sums are joined at
// the end.  The keys come into LDS by direct copies one step ahead (each wave a
// run of one page of K and of V) while the step before is multiplied; one barrier
// a step.  S^T = K Q^T and O^T = V^T P^T in 32 x 32 x 16 products: a lane holds
// half of the scores of its row and 16 of the 32 rows of each d tile.
//
// 4096 tokens over 32768 keys, 32 heads on 8, 128 wide, bf16: 2440 us, 957 TFLOP/s,
// 70 % of what a large library product of this type reaches.  Counters of that
// call: matrix cores busy 44 % of the cycles, vector work (exponentials, maxima,
// differences, rounding) 46 %, LDS 22 %, no bank conflicts, waves waiting 33 % of
// theirs; what is left is two waves a SIMD waiting for each other's step, and 128
// rows of registers allow no third.
// 128 rows a tile so that a key read from HBM or L2 serves them all: 16-row tiles
// took 11964 us.
template <typename C, int PARTS, int DP, int FEAT, int HALVES>
__global__ void __launch_bounds__(256 * HALVES, ac_waves(PARTS, DP))
k_attn_chunk(AttnArgs a, int tiles, int least, int splits)
{
    typedef typename C::T T;
    typedef typename C::V8 V8;
    typedef typename C::V4 V4;
    constexpr int WAVES = 4 * HALVES;
    constexpr int HK = ac_half_keys(PARTS, DP), KEYS = HK * HALVES, SU = HK / 32; // a half's keys of a step, and all
    constexpr int RUN = HK / 4, NI = RUN * DP / 512; // keys that a wave copies, in NI copies of 1 KB
    constexpr int KS = DP / 16, DT = DP / 32, NC = DP / 8;
    constexpr int TILE = KEYS * DP * 2;
    constexpr bool AHEAD = ac_ahead(PARTS, DP, FEAT);
    // p times 2^kUp, with room for 2^kLate below fp16's 2^16: kept down to 2^-32 of
    // the largest; the sums are scaled again when the maximum has grown by 2^kLate
    constexpr float kUp = C::kShift != 0.0f ? 8.0f : 0.0f;
    constexpr float kLate = 7.0f;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TILE]; // K, V of two steps
    __shared__ int lds_odd;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave >> 2;
    const int col = lane & 31, h = lane >> 5;
    const int D = a.cache.dim;
    Tile t;
    if (!find_tile<AC_ROWS, KEYS>(a, tiles, least, splits, blockIdx.x, t))
        return;
    if (tid == 0)
        lds_odd = -1;

    const int wrow0 = t.row0 + 32 * (wave & 3);
    const int wrows = min(32, t.row0 + t.rows - wrow0);
    const int before = t.first - t.row0 / a.group; // position of the sequence's first new token
    const int row = wrow0 + col;
    const bool live = col < wrows;
    const int qhead = t.head * a.group + (live ? row % a.group : 0);
    const int64_t qrow = (int64_t)(t.start + (live ? row / a.group : 0)) * a.q_heads + qhead;
    const int wfirst = before + wrow0 / a.group, wlast = before + (wrow0 + max(wrows, 1) - 1) / a.group;
    const int pos = live ? before + row / a.group : wfirst;
    V8 qf[PARTS][KS];
    int up;
    load_q<C, PARTS, KS>(a, qrow, live, 2, h, qf, up);
    // scores become powers of two with the last factor, `by`; a cap takes the scale
    // before, and the bias is added in units of `by`.  by / a.by, a power of two (the
    // row's and the scale's), brings the maxima of a row's parts to one unit.
    const float by = FEAT == kCap ? a.by : finite(a.by * power_of_two(a.scale_exp - up));
    const float slope = FEAT != kPlain && a.slopes ? finite(a.slopes[qhead] * kLog2e / by) : 0.0f;
    const Seen sees = seen_from(a, t, pos);

    // a lane's part of the copies: RUN keys of one page
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = (64 * i + lane) / NC, c = (64 * i + lane) % NC;
        // (chunks behind a head's end hold its last one: nothing reads them with weight)
        koff[i] = 2u * (uint32_t)(r * D + 8 * min(ac_k_chunk<NC>(RUN * wave + r, c), D / 8 - 1));
        voff[i] = 2u * (uint32_t)(r * D + 8 * min(ac_v_chunk<NC>(RUN * wave + r, c), D / 8 - 1));
    }
    const int page_mask = (1 << a.cache.page_shift) - 1;
    const int n_steps = (t.hi - t.lo + KEYS - 1) / KEYS;
    // page ids of a step's runs of 16 keys, in the first lanes
    auto page_of = [&](int step) {
        const int j = t.lo + KEYS * step + 16 * (lane & (KEYS / 16 - 1));
        return j < t.hi ? t.table[j >> a.cache.page_shift] : -1;
    };
    // the runs of a step that name no page of the pool
    auto bad_runs = [&](int step, int ids) {
        const bool bad = lane < KEYS / 16 && t.lo + KEYS * step + 16 * lane < t.hi &&
                         (unsigned)ids >= (unsigned)a.cache.pages;
        return (int)__ballot(bad);
    };
    auto copy = [&](int step, int ids) {
        const int id = __builtin_amdgcn_readlane(ids, RUN * wave / 16);
        if ((unsigned)id >= (unsigned)a.cache.pages)
            return; // (no such key, or reported: its rows of V are cleared before use)
        const int j = t.lo + KEYS * step + RUN * wave;
        const int64_t at = (int64_t)id * a.cache.page_stride +
                           ((int64_t)((t.head << a.cache.page_shift) + (j & page_mask))) * D;
        const T *k = (const T *)a.cache.k + at, *v = (const T *)a.cache.v + at;
        const uint32_t to = lds0 + 2 * TILE * (step & 1) + 1024 * NI * wave;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            lds_copy16_at(k, koff[i], to + 1024 * i);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            lds_copy16_at(v, voff[i], to + TILE + 1024 * i);
    };

    // every wave, when all have read the step's values
    auto clear_odd = [&](int step) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        lds_barrier();
        uint32_t *const v = (uint32_t *)(lds + 2 * TILE * (step & 1) + TILE);
        for (int i = tid; i < TILE / 4; i += 64 * WAVES)
            v[i] = without_odd<C>(v[i]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        lds_barrier();
    };

    // a lane's places in a tile: K's operand (row col, chunk 2 i + h), V^T's (rows
    // 4 h + q, columns of the 16-lane group).  The chunks of the other products lie
    // at these addresses with the number of the chunk xor-ed in, which is formed
    // anew each step: the registers that the addresses would take are needed.
    const int l16 = lane & 15, vrow = 4 * h + (l16 >> 2);
    const uint32_t kat = (uint32_t)(col * DP * 2 + 16 * ac_k_chunk<NC>(col, h));
    const uint32_t vat = (uint32_t)(vrow * DP * 2 +
                                    16 * ac_v_chunk<NC>(vrow, 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1)) + 8 * (l16 & 1));

    float m = kNone, l = 0.0f;
    f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
        o[d] = f16v{};

    int ids = -1, ids_next = -1;
    if (n_steps > 0) {
        ids = page_of(0);
        copy(0, ids);
        ids_next = page_of(1);
    }
    for (int step = 0; step < n_steps; ++step) {
        const int key0 = t.lo + KEYS * step, key = key0 + HK * half;
        __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0) lgkmcnt(0): this wave's copies, and its reads of the other buffer
        lds_barrier();
        const int bad_all = bad_runs(step, ids), bad = bad_all >> (HK / 16 * half) & ((1 << HK / 16) - 1);
        if (bad_all && a.flags && tid == 0)
            atomicOr(a.flags, kFlagKvPage);
        if (step + 1 < n_steps) {
            copy(step + 1, ids_next);
            ids = ids_next;
            ids_next = page_of(step + 2);
        }
        uint8_t *const vt = lds + 2 * TILE * (step & 1) + TILE + HK * half * (DP * 2);
        // a step that the whole tile does not see whole: rows of V that no row sees
        // are cleared, and an infinity or NaN among the others is looked for
        const bool edge = bad_all || key0 + KEYS > t.len || !(key0 + KEYS - 1 <= t.first || key0 + KEYS <= t.prefix) ||
                          !(a.window == 0 || t.last - key0 < a.window);
        bool odd = false;
        if (__builtin_expect(edge, 0)) {
            uint8_t *const all = lds + 2 * TILE * (step & 1) + TILE;
            for (int i = tid; i < KEYS * NC; i += 64 * WAVES) {
                const int r = i / NC, j = key0 + r;
                if (!(j < t.len && (j <= t.last || j < t.prefix) && (a.window == 0 || t.first - j < a.window)) ||
                    ((bad_all >> (r >> 4)) & 1)) {
                    *(u4 *)(all + 16 * i) = u4{};
                } else {
                    const u4 w = *(const u4 *)(all + 16 * i);
                    odd |= odd_value<C>(w.x) || odd_value<C>(w.y) || odd_value<C>(w.z) || odd_value<C>(w.w);
                }
            }
            if (odd)
                lds_odd = step;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            lds_barrier();
            odd = __builtin_amdgcn_readfirstlane(lds_odd) == step;
        }
        // keys that none of the wave's rows sees
        if (wrows <= 0 || key >= t.hi || (key > wlast && key >= t.prefix) ||
            (a.window && wfirst - (key + HK - 1) >= a.window)) {
            if (odd)
                clear_odd(step);
            continue;
        }
        const bool whole = !bad && key + HK <= t.len && (key + HK - 1 <= wfirst || key + HK <= t.prefix) &&
                           (a.window == 0 || wlast - key < a.window);

        const uint32_t k_here = lds0 + 2 * TILE * (step & 1) + HK * half * (DP * 2) + kat;
        const uint32_t v_here = lds0 + 2 * TILE * (step & 1) + HK * half * (DP * 2) + TILE + vat;
        auto read_k = [&](int u, int i) { // (256 wide: chunks 16 and up lie 256 bytes on)
            return read_lds<V8>((k_here ^ (32 * (i & 7))) + 32 * u * (DP * 2) + (i >> 3) * 256);
        };
        auto read_v = [&](int u, int d, int k) {
            const uint32_t at = (v_here ^ (64 * (d & 3))) + (32 * u + 16 * k) * (DP * 2) + (d >> 2) * 256;
            const V4 lo = read_tr_at<V4>(at), hi = read_tr_at<V4>(at + 8 * (DP * 2));
            return (V8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        f16v s[SU];
        V8 vf[AHEAD ? DT : 1][2];
        if constexpr (AHEAD) {
            V8 kf[SU][KS];
#pragma unroll
            for (int i = 0; i < KS; ++i)
                kf[0][i] = read_k(0, i);
#pragma unroll
            for (int u = 0; u < SU; ++u) {
                s[u] = f16v{};
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    if (u + 1 < SU)
                        kf[u + 1][i] = read_k(u + 1, i);
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
                        s[u] = C::mfma32(kf[u][i], qf[part][i], s[u]);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    vf[d][k] = read_v(0, d, k);
            // (in this order: LDS reads 0x100, products 8)
            constexpr int FIRST = ac_first(PARTS, DP);
            __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
            for (int i = 0; i < SU * KS - FIRST; ++i) {
                __builtin_amdgcn_sched_group_barrier(8, PARTS, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
            for (int i = 0; i < FIRST; ++i) {
                __builtin_amdgcn_sched_group_barrier(8, PARTS, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 4 * DT / FIRST, 0);
            }
        } else {
#pragma unroll
            for (int u = 0; u < SU; ++u) {
                s[u] = f16v{};
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const V8 kf = read_k(u, i);
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
                        s[u] = C::mfma32(kf, qf[part][i], s[u]);
                    if (DP == 256 && i % 8 == 7)
                        __builtin_amdgcn_sched_barrier(0); // (operands further ahead would not fit the registers)
                }
            }
        }
        if constexpr (FEAT != kPlain) {
            const float apart = (float)(pos - key - 4 * h);
            if constexpr (FEAT == kCap) {
                const float by_cap = finite(__builtin_ldexpf(a.to_cap, a.scale_exp - up));
                float most = 0.0f;
#pragma unroll
                for (int u = 0; u < SU; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[u][i] *= by_cap;
                        most = fmaxf(most, fabsf(s[u][i]));
                    }
                if (__any(most > kNear)) {
#pragma unroll
                    for (int u = 0; u < SU; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[u][i] = tanh_any(s[u][i]);
                } else { // (a NaN is neither, and stays)
#pragma unroll
                    for (int u = 0; u < SU; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[u][i] = tanh_near(s[u][i]);
                }
            }
            if (a.slopes)
#pragma unroll
                for (int u = 0; u < SU; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[u][i] = fmaf(-slope, fabsf(apart - (float)(32 * u + 8 * (i >> 2) + (i & 3))), s[u][i]);
        }
        if (__builtin_expect(!whole, 0)) {
#pragma unroll
            for (int u = 0; u < SU; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[u][i] = sees(key + 32 * u + 8 * (i >> 2) + 4 * h + (i & 3)) ? s[u][i] : kNone;
            if (__builtin_expect(bad, 0))
#pragma unroll
                for (int u = 0; u < SU; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[u][i] = (bad >> (2 * u + (i >> 3))) & 1 ? kNone : s[u][i];
        }
        float mx = kNone;
#pragma unroll
        for (int u = 0; u < SU; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                mx = fmaxf(mx, s[u][i]);
        mx = halves_max(mx);
        if (__any((mx - m) * by > kLate)) { // (a row's first key: by an infinity; without one: NaN, no)
            const float top = fmaxf(mx, m);
            const float f = top == kNone ? 1.0f : exp2_fast((m - top) * by);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                o[d] *= f;
            m = top;
        }
        const float use = m == kNone ? 0.0f : m;
        if (__builtin_expect(odd, 0)) {
            // infinities or NaNs that some rows of the tile see and others do not:
            // they are added one key at a time where a row has a weight for them,
            // then the products take 0 (see k_attn_rows)
#pragma unroll 1
            for (int j = 0; j < HK; ++j) {
                const int i = 4 * ((j & 31) >> 3) + (j & 3);
                float x = kNone;
#pragma unroll
                for (int u = 0; u < SU; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        x = i == e && u == j >> 5 ? s[u][e] : x;
                x = __shfl(exp2_fast(fmaf(x - use, by, kUp)), col + 32 * ((j >> 2) & 1));
                const uint8_t *const vj = vt + j * (DP * 2) + 8 * h;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const V4 v = *(const V4 *)(vj + ac_v_chunk<NC>(j, 4 * d + e / 4) * 16);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            o[d][e + q] += x != 0.0f && !__builtin_isfinite((float)v[q]) ? x * (float)v[q] : 0.0f;
                    }
                    __builtin_amdgcn_sched_barrier(0); // (rare: no registers for loads ahead)
                }
            }
            clear_odd(step);
            if constexpr (AHEAD)
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        vf[d][k] = read_v(0, d, k);
        }
        // 32 keys at a time: their weights, then their products
#pragma unroll
        for (int u = 0; u < SU; ++u) {
            V8 pf[PARTS][2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x = exp2_fast(fmaf(s[u][i] - use, by, kUp));
                s[u][i] = x;
                l += x;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const T y = (T)x;
                    pf[part][i >> 3][i & 7] = y;
                    x -= (float)y;
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if (DP == 256 && !AHEAD && d % 2 == 0)
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (AHEAD) {
#pragma unroll
                        for (int part = 0; part < PARTS; ++part)
                            o[d] = C::mfma32(vf[d][k], pf[part][k], o[d]);
                        if (u + 1 < SU)
                            vf[d][k] = read_v(u + 1, d, k);
                    } else {
                        const V8 v = read_v(u, d, k);
#pragma unroll
                        for (int part = 0; part < PARTS; ++part)
                            o[d] = C::mfma32(v, pf[part][k], o[d]);
                    }
                }
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070); // no copy is in flight when the workgroup ends

    if constexpr (HALVES == 2) {
        // the second half's maxima, sums and rows to the first, by lane
        lds_barrier(); // nobody reads the keys any more
        float *const to = (float *)lds + (DT * 16 + 2) * 64 * (wave & 3) + lane;
        if (half) {
            to[0] = m;
            to[64] = l;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    to[64 * (2 + 16 * d + e)] = o[d][e];
        }
        __syncthreads();
        if (half)
            return;
        const float m2 = to[0], l2 = to[64], top = fmaxf(m, m2);
        const float f = m == kNone ? 0.0f : exp2_fast((m - top) * by);
        const float f2 = m2 == kNone ? 0.0f : exp2_fast((m2 - top) * by);
        // (a half without keys has only zeros; NaN stays)
        l = l * f + l2 * f2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                o[d][e] = o[d][e] * f + to[64 * (2 + 16 * d + e)] * f2;
        m = top;
    }

    // the row's place, formed anew: kept, it takes registers that the loop spills for
    // (us, formed anew against kept, 2048 fp32 rows over 8192 keys, 256 wide: bf16
    // 1637, 2148, fp16 1253, 1273; elsewhere within 1 %)
    int at_end = lane;
    asm volatile("" : "+v"(at_end));
    const int row_end = wrow0 + (at_end & 31);
    if ((at_end & 31) >= wrows)
        return;
    const int64_t qrow_end = (int64_t)(t.start + row_end / a.group) * a.q_heads + t.head * a.group + row_end % a.group;
    l = halves_sum(l);
    const int64_t rows_all = (int64_t)a.batch.tokens * a.q_heads;
    if (splits > 1) {
        if (at_end < 32)
            *(f2 *)(a.part + (int64_t)splits * rows_all * D + 2 * (t.split * rows_all + qrow_end)) = f2{m * (by / a.by), l};
        if (l == 0.0f)
            return;
    }
    const float f = splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int at = 32 * d + 2 * e + 4 * (at_end >> 5);
            if (at >= D)
                continue;
            f4 v = f4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            v = l == 0.0f ? f4{} : v * f;
            if (splits > 1)
                *(f4 *)(a.part + (t.split * rows_all + qrow_end) * D + at) = v;
            else if constexpr (PARTS == 1)
                *(V4 *)((T *)a.out + qrow_end * D + at) = __builtin_convertvector(v, V4);
            else
                *(f4 *)((float *)a.out + qrow_end * D + at) = v;
        }
}

// The splits' partial rows joined, four values a thread: sum_i e^(m_i - m) o_i
// over sum_i e^(m_i - m) l_i.  Few splits: several rows a workgroup; many: one,
// its splits shared among groups of threads, which are joined in their order.
// Bound by reading the parts eight at a time: 8 us of the 34 that five ragged chunks
// take (64 wide, 24 heads; the call took 39 with the parts passed through LDS).
template <typename C, int PARTS>
__global__ void __launch_bounds__(256) k_attn_join(AttnArgs a, int splits)
{
    __shared__ Joined lds_g[256];
    const int D = a.cache.dim, per = D / 4, slots = 256 / per, slot = threadIdx.x / per, d = 4 * (threadIdx.x - slot * per);
    const bool many = splits > AC_FEW_SPLITS;
    const int64_t rows = (int64_t)a.batch.tokens * a.q_heads;
    const int64_t row = many ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * slots + slot;
    // (a row of no sequence is left as it is)
    const int token = (int)(row / a.q_heads);
    const bool live = slot < slots && row < rows && token >= a.batch.starts[0] && token < a.batch.starts[a.batch.sequences];
    const int64_t at = live ? row : 0;
    const uint64_t *const o = (const uint64_t *)a.part, *const ml = o + (int64_t)splits * rows * D / 2;
    Joined j = join_parts(o + (at * D + d) / 2, ml + at, rows, D, many ? slot : 0, many ? slots : 1, live ? splits : 0,
                          a.by);
    if (many) {
        lds_g[threadIdx.x] = j;
        __syncthreads();
        if (slot > 0)
            return;
        for (int q = 1; q < slots; ++q)
            j.add(lds_g[threadIdx.x + q * per].top, lds_g[threadIdx.x + q * per].sum, lds_g[threadIdx.x + q * per].v,
                  a.by);
    }
    if (!live)
        return;
    const f4 v = j.sum == 0.0f ? f4{} : j.v * (1.0f / j.sum);
    if constexpr (PARTS == 1)
        *(typename C::V4 *)((typename C::T *)a.out + row * D + d) = __builtin_convertvector(v, typename C::V4);
    else
        *(f4 *)((float *)a.out + row * D + d) = v;
}

template <typename C, int PARTS, int DP, int FEAT>
void start(const AttnArgs &a, const AttnPlan &p, hipStream_t s)
{
    const dim3 grid((uint32_t)((int64_t)p.tiles * a.cache.heads * p.splits));
    if (p.rows == AR_ROWS) {
        hipLaunchKernelGGL((k_attn_rows<C, PARTS, DP, FEAT>), grid, dim3(64 * AR_WAVES), 0, s, a, p.tiles, p.least, p.splits);
        return;
    }
    if constexpr (ac_waves(PARTS, DP) == 2 && DP <= 128) {
        if (p.halves) {
            hipLaunchKernelGGL((k_attn_chunk<C, PARTS, DP, FEAT, 2>), grid, dim3(512), 0, s, a, p.tiles, p.least, p.splits);
            return;
        }
    }
    hipLaunchKernelGGL((k_attn_chunk<C, PARTS, DP, FEAT, 1>), grid, dim3(256), 0, s, a, p.tiles, p.least, p.splits);
}

template <typename C, int PARTS, int FEAT>
void start_feat(const AttnArgs &a, const AttnPlan &p, hipStream_t s)
{
    if (a.cache.dim <= 64)
        start<C, PARTS, 64, FEAT>(a, p, s);
    else if (a.cache.dim <= 128)
        start<C, PARTS, 128, FEAT>(a, p, s);
    else
        start<C, PARTS, 256, FEAT>(a, p, s);
}

template <typename C, int PARTS>
hipError_t start_dim(const AttnArgs &a, const AttnPlan &p, hipStream_t s)
{
    if (a.cap > 0.0f)
        start_feat<C, PARTS, kCap>(a, p, s);
    else if (a.slopes)
        start_feat<C, PARTS, kBias>(a, p, s);
    else
        start_feat<C, PARTS, kPlain>(a, p, s);
    if (p.splits > 1 && p.rows == AC_ROWS) {
        const int64_t rows = (int64_t)a.batch.tokens * a.q_heads;
        const int slots = p.splits > AC_FEW_SPLITS ? 1 : 256 / (a.cache.dim / 4);
        hipLaunchKernelGGL((k_attn_join<C, PARTS>), dim3((uint32_t)((rows + slots - 1) / slots)), dim3(256), 0, s, a, p.splits);
    }
    return hipGetLastError();
}

} // namespace

hipError_t launch_attn(AttnArgs a, const AttnPlan &p, hipStream_t s)
{
    const float scale = std::frexp(a.scale == 0.0f ? 1.0f : std::fabs(a.scale), &a.scale_exp);
    a.by = a.cap > 0.0f ? std::fmin(a.cap * kLog2e, 3.402823466e38f) : scale * kLog2e;
    a.to_cap = a.cap > 0.0f ? scale / a.cap : 0.0f;
    if (a.cache.type == kF16)
        return a.act == kF32 ? start_dim<Half, 2>(a, p, s) : start_dim<Half, 1>(a, p, s);
    return a.act == kF32 ? start_dim<BHalf, 3>(a, p, s) : start_dim<BHalf, 1>(a, p, s);
}

} // namespace ihip
