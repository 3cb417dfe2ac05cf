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
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The two cache types: vectors, products, the transposing read.
struct Half {
    typedef _Float16 T;
    typedef h2 V2;
    typedef h4 V4;
    typedef h8 V8;
    // p = e^(s - m) is carried times 2^14: what fp16 keeps of small ones reaches
    // down to 2^-38 of the largest
    static constexpr float kShift = 14.0f;
    static constexpr uint32_t kExp = 0x7c007c00u;
    static __device__ __forceinline__ f4 mfma16(V8 a, V8 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
};

template <typename V4>
__device__ __forceinline__ V4 read_tr(const uint8_t *lds)
{
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)lds));
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

// What a workgroup works on: a tile of rows of one sequence and KV head, and
// the part of its keys.
struct Tile {
    int head;                // KV head
    int start, row0, rows;   // the sequence's first token; the tile's first row in it; its rows
    int first, last;         // cache positions of the tile's first and last token
    int len, prefix;         // keys there are; keys every row sees
    int lo, hi;              // keys to look at (lo a multiple of 32); lo >= hi: none
    int split;
    const int32_t *table;
};

// Workgroup `bid`'s tile; false if there is none.  Tiles are counted over the
// sequences in order; their number is only known here, the grid holds the most
// there can be.
template <int ROWS>
__device__ __forceinline__ bool find_tile(const AttnArgs &a, int tiles, int least, int splits, int bid, Tile &t)
{
    if (bid == 0 && a.flags)
        kv_report(a.batch, a.cache.page_shift, a.flags);
    t.head = bid % a.cache.heads;
    const int rest = bid / a.cache.heads;
    const int want = rest % tiles;
    t.split = rest / tiles;
    int first = 0;
    const int s = kv_find(a.batch.sequences, want, first, [&](int i) {
        const int b = kv_clamp(a.batch.starts[i], 0, a.batch.tokens);
        const int n = kv_clamp(a.batch.starts[i + 1], b, a.batch.tokens) - b;
        return (int)(((int64_t)n * a.group + ROWS - 1) / ROWS);
    });
    if (s < 0)
        return false;
    const KvSeq q = kv_seq(a.batch, a.cache.page_shift, s);
    t.start = q.start;
    t.row0 = (want - first) * ROWS;
    t.rows = min(ROWS, (int)((int64_t)q.n * a.group - t.row0));
    t.len = q.len;
    t.first = q.len - q.n + t.row0 / a.group;
    t.last = q.len - q.n + (t.row0 + t.rows - 1) / a.group;
    t.prefix = a.prefix ? kv_clamp(a.prefix[s], 0, q.len) : 0;
    t.table = a.batch.table + (int64_t)s * a.batch.stride;
    const int lo = a.window ? max(0, t.first - a.window + 1) & ~31 : 0;
    const int hi = max(t.last + 1, t.prefix);
    // the split's part of the keys: a fixed number, or more where the most
    // splits there may be would not reach the end
    const int keys = max(0, hi - lo);
    const int per = max(least, (int)(((int64_t)keys + splits - 1) / splits + 127) & ~127);
    const int64_t from = (int64_t)lo + (int64_t)t.split * per;
    t.lo = (int)min(from, (int64_t)hi);
    t.hi = (int)min(from + per, (int64_t)hi);
    return true;
}

// Whether key j is seen from position p.
__device__ __forceinline__ bool seen(const AttnArgs &a, const Tile &t, int p, int j)
{
    return (j <= p || j < t.prefix) && j < t.len && (a.window == 0 || p - j < a.window);
}

// q's part of a lane: KS chunks of 8 values (chunk 4 i + g of the row), in
// PARTS parts.  Two fp16 parts are taken of q times a power of two that brings
// the row's largest value to [2^14, 2^15), undone (`undo`) on the scores.
template <typename C, int PARTS, int KS>
__device__ __forceinline__ void load_q(const AttnArgs &a, int64_t row, bool live, int step, int offset,
                                       typename C::V8 (&qf)[PARTS][KS], float &undo)
{
    typedef typename C::V8 V8;
    undo = 1.0f;
    if constexpr (PARTS == 1) {
        const typename C::T *q = (const typename C::T *)a.q + row * a.cache.dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int c = (step * i + offset) * 8;
            qf[0][i] = live && c < a.cache.dim ? *(const V8 *)(q + c) : V8{};
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
        int up = 0;
        if constexpr (C::kShift != 0.0f) {
            most = step == 4 ? groups_max(most) : fmaxf(most, __shfl_xor(most, 32));
            const bool finite = most > 0.0f && most < __builtin_inff();
            up = finite ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
            undo = __builtin_ldexpf(1.0f, -up);
        }
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float x = __builtin_ldexpf(v[2 * i + u / 4][u % 4], up);
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
constexpr int AR_ROWS = 16;   // rows of a tile
constexpr int AR_KEYS = 32;   // keys of a wave's step
constexpr int AR_WAVES = 4;

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
    return AR_ROWS * (DP + 4) * 4 > AR_KEYS * DP * 2 ? AR_ROWS * (DP + 4) * 4 : AR_KEYS * DP * 2;
}

// A workgroup's 4 waves walk the keys of its part 32 at a time, each its own
// steps (no shared data, no barrier), K from HBM into the matrix operand's
// registers, V through 32 rows of LDS of the wave's own; the waves' sums are
// joined at the end.  Loads run one step ahead.
template <typename C, int PARTS, int DP, bool GEN>
__global__ void __launch_bounds__(64 * AR_WAVES) k_attn_rows(AttnArgs a, int tiles, int least, int splits)
{
    typedef typename C::T T;
    typedef typename C::V8 V8;
    typedef typename C::V4 V4;
    constexpr int KS = DP / 32, DT = DP / 16, NC = DP / 8, NV = AR_KEYS * NC / 64;
    __shared__ __attribute__((aligned(16))) uint8_t lds[AR_WAVES * ar_wave_lds<DP>()];
    __shared__ float lds_m[AR_WAVES][AR_ROWS], lds_l[AR_WAVES][AR_ROWS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int D = a.cache.dim;
    Tile t;
    if (!find_tile<AR_ROWS>(a, tiles, least, splits, blockIdx.x, t))
        return;

    const int row = t.row0 + col; // the row of this lane's column
    const bool live = col < t.rows;
    const int qhead = t.head * a.group + (live ? row % a.group : 0);
    const int64_t qrow = (int64_t)(t.start + (live ? row / a.group : 0)) * a.q_heads + qhead;
    const int pos = live ? t.first - t.row0 / a.group + row / a.group : t.first;
    V8 qf[PARTS][KS];
    float undo;
    load_q<C, PARTS, KS>(a, qrow, live, 4, g, qf, undo);
    const float slope = GEN && a.slopes ? a.slopes[qhead] * kLog2e : 0.0f;
    const float by = GEN && a.cap > 0.0f ? a.scale * undo / a.cap : a.scale * undo * kLog2e;

    float m = kNone, l = 0.0f;
    f4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
        o[d] = f4{};

    uint8_t *const vt = lds + wave * ar_wave_lds<DP>();
    V8 kf[2][KS];
    u4 vf[NV];
    int id[2];
    bool ok[2];
    const int page_mask = (1 << a.cache.page_shift) - 1;
    const int n_steps = (t.hi - t.lo + AR_KEYS - 1) / AR_KEYS;

    auto pages = [&](int key) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = key + 16 * u;
            id[u] = j < t.hi ? __builtin_amdgcn_readfirstlane(t.table[j >> a.cache.page_shift]) : -1;
            ok[u] = (unsigned)id[u] < (unsigned)a.cache.pages;
            if (j < t.hi && !ok[u] && a.flags && lane == 0)
                atomicOr(a.flags, kFlagKvPage);
        }
    };
    auto base = [&](int key, int u) {
        return (int64_t)id[u] * a.cache.page_stride +
               ((int64_t)((t.head << a.cache.page_shift) + ((key + 16 * u) & page_mask))) * D;
    };
    auto load_k = [&](int key) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const T *k = (const T *)a.cache.k + (ok[u] ? base(key, u) : 0) + col * D;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int c = (4 * i + g) * 8;
                kf[u][i] = ok[u] && c < D ? *(const V8 *)(k + c) : V8{};
            }
        }
    };
    auto load_v = [&](int key) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = i / (NV / 2);
            const int e = i * 64 + lane, r = e / NC - 16 * u, c = e % NC;
            const T *v = (const T *)a.cache.v + (ok[u] ? base(key, u) : 0) + r * D + c * 8;
            vf[i] = ok[u] && c * 8 < D ? *(const u4 *)v : u4{};
        }
    };

    int step = wave;
    if (step < n_steps) {
        pages(t.lo + AR_KEYS * step);
        load_k(t.lo + AR_KEYS * step);
        load_v(t.lo + AR_KEYS * step);
    }
    for (; step < n_steps; step += AR_WAVES) {
        const int key = t.lo + AR_KEYS * step;
        const bool whole = ok[0] && ok[1] && key + AR_KEYS <= t.hi &&
                           (key + AR_KEYS - 1 <= t.first || key + AR_KEYS <= t.prefix) &&
                           (a.window == 0 || t.last - key < a.window);
        const bool ok0 = ok[0], ok1 = ok[1];
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
        const bool more = step + AR_WAVES < n_steps;
        if (more) {
            pages(key + AR_KEYS * AR_WAVES);
            load_k(key + AR_KEYS * AR_WAVES);
        }
        float mx = kNone;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = s[u][i] * by;
                if (GEN && a.cap > 0.0f)
                    x = a.cap * kLog2e * tanhf(x);
                const int j = key + 16 * u + 4 * g + i;
                if (GEN)
                    x -= slope * fabsf((float)(pos - j));
                if (!whole && !(seen(a, t, pos, j) && (u ? ok1 : ok0)))
                    x = kNone;
                s[u][i] = x;
                mx = fmaxf(mx, x);
            }
        mx = fmaxf(groups_max(mx), m);
        // (a row without a key yet keeps its sum 0 whatever is subtracted)
        const float use = mx == kNone ? 0.0f : mx;
        if (__any(mx != m)) {
            const float f = exp2_fast(m - use);
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
                float x = exp2_fast(s[u][i] - use + C::kShift);
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

        // V's rows to LDS; of a step with hidden keys, the rows that no row of the
        // tile sees as zeros (nothing may come from them, whatever they hold)
        bool odd = false;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * 64 + lane, r = e / NC, c = e % NC;
            if (!whole) {
                const int j = key + r;
                if (!(j < t.len && (j <= t.last || j < t.prefix) && (a.window == 0 || t.first - j < a.window)))
                    vf[i] = u4{};
                odd |= odd_value<C>(vf[i].x) || odd_value<C>(vf[i].y) || odd_value<C>(vf[i].z) ||
                       odd_value<C>(vf[i].w);
            }
            *(u4 *)(vt + r * (DP * 2) + v_chunk<NC>(r, c) * 16) = vf[i];
        }
        asm volatile("" ::: "memory");
        if (more)
            load_v(key + AR_KEYS * AR_WAVES);
        if (!whole && __any(odd)) {
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
                    const int e = 16 * d + 4 * g;
                    const V4 v = *(const V4 *)(vt + j * (DP * 2) + v_chunk<NC>(j, e / 8) * 16 + (e % 8) * 2);
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
    float *const ol = (float *)vt;
#pragma unroll
    for (int d = 0; d < DT; ++d)
        *(f4 *)(ol + col * (DP + 4) + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        lds_m[wave][col] = m;
        lds_l[wave][col] = l;
    }
    __syncthreads();
    const int64_t rows_all = (int64_t)a.batch.tokens * a.q_heads;
    float *const ml = a.part + (int64_t)splits * rows_all * D;
    for (int e = tid; e < t.rows * (D / 4); e += 64 * AR_WAVES) {
        const int r = e / (D / 4), d = 4 * (e % (D / 4));
        float top = kNone;
#pragma unroll
        for (int w = 0; w < AR_WAVES; ++w)
            top = fmaxf(top, lds_m[w][r]);
        float sum = 0.0f;
        f4 v = f4{};
#pragma unroll
        for (int w = 0; w < AR_WAVES; ++w) {
            const float f = lds_m[w][r] == kNone ? 0.0f : exp2_fast(lds_m[w][r] - top);
            const f4 x = *(const f4 *)(lds + w * ar_wave_lds<DP>() + 4 * (r * (DP + 4) + d));
            sum += lds_l[w][r] * f;
            v += x * f;
        }
        const int rr = t.row0 + r;
        const int64_t to = (int64_t)(t.start + rr / a.group) * a.q_heads + t.head * a.group + rr % a.group;
        if (splits > 1) {
            if (sum != 0.0f) // (NaN too; a part without keys is its sum alone)
                *(f4 *)(a.part + ((int64_t)t.split * rows_all + to) * D + d) = v;
            if (d == 0) {
                ml[2 * (t.split * rows_all + to)] = top;
                ml[2 * (t.split * rows_all + to) + 1] = sum;
            }
        } else {
            const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
            v = sum == 0.0f ? f4{} : v * f;
            if constexpr (PARTS == 1)
                *(V4 *)((T *)a.out + to * D + d) = __builtin_convertvector(v, V4);
            else
                *(f4 *)((float *)a.out + to * D + d) = v;
        }
    }
}

// The splits' partial rows joined, a wave a row: sum_i e^(m_i - m) o_i over
// sum_i e^(m_i - m) l_i, in split order.
template <typename C, int PARTS>
__global__ void __launch_bounds__(256) k_attn_join(AttnArgs a, int splits)
{
    const int lane = threadIdx.x & 63, D = a.cache.dim;
    const int64_t rows = (int64_t)a.batch.tokens * a.q_heads;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows)
        return;
    int first = 0;
    if (kv_find(a.batch.sequences, (int)(row / a.q_heads), first, [&](int i) {
            const int b = kv_clamp(a.batch.starts[i], 0, a.batch.tokens);
            return kv_clamp(a.batch.starts[i + 1], b, a.batch.tokens) - b;
        }) < 0)
        return; // a row behind the last sequence
    const float *ml = a.part + (int64_t)splits * rows * D;
    float top = kNone;
    for (int i = lane; i < splits; i += 64)
        top = fmaxf(top, ml[2 * (i * rows + row)]);
    for (int d = 32; d; d /= 2)
        top = fmaxf(top, __shfl_xor(top, d));
    f4 v = f4{};
    float sum = 0.0f;
    for (int i = 0; i < splits; ++i) {
        const float m = ml[2 * (i * rows + row)], l = ml[2 * (i * rows + row) + 1];
        if (l == 0.0f)
            continue; // no key was seen: nothing else was written
        const float f = m == kNone ? 0.0f : exp2_fast(m - top);
        sum += l * f;
        if (4 * lane < D)
            v += *(const f4 *)(a.part + (i * rows + row) * D + 4 * lane) * f;
    }
    if (4 * lane < D) {
        v = sum == 0.0f ? f4{} : v * (1.0f / sum);
        if constexpr (PARTS == 1)
            *(typename C::V4 *)((typename C::T *)a.out + row * D + 4 * lane) = __builtin_convertvector(v, typename C::V4);
        else
            *(f4 *)((float *)a.out + row * D + 4 * lane) = v;
    }
}

template <typename C, int PARTS, int DP>
void start(const AttnArgs &a, const AttnPlan &p, hipStream_t s)
{
    const dim3 grid((uint32_t)((int64_t)p.tiles * a.cache.heads * p.splits));
    if (a.cap > 0.0f || a.slopes)
        hipLaunchKernelGGL((k_attn_rows<C, PARTS, DP, true>), grid, dim3(64 * AR_WAVES), 0, s, a, p.tiles, p.least, p.splits);
    else
        hipLaunchKernelGGL((k_attn_rows<C, PARTS, DP, false>), grid, dim3(64 * AR_WAVES), 0, s, a, p.tiles, p.least, p.splits);
}

template <typename C, int PARTS>
hipError_t start_dim(const AttnArgs &a, const AttnPlan &p, hipStream_t s)
{
    if (a.cache.dim <= 64)
        start<C, PARTS, 64>(a, p, s);
    else if (a.cache.dim <= 128)
        start<C, PARTS, 128>(a, p, s);
    else
        start<C, PARTS, 256>(a, p, s);
    if (p.splits > 1) {
        const int64_t rows = (int64_t)a.batch.tokens * a.q_heads;
        hipLaunchKernelGGL((k_attn_join<C, PARTS>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s, a, p.splits);
    }
    return hipGetLastError();
}

} // namespace

AttnPlan attn_plan(int act, int kv_type, int q_heads, int kv_heads, int dim, int sequences, int tokens,
                   int64_t capacity)
{
    (void)act;
    (void)kv_type;
    AttnPlan p;
    const int group = q_heads / kv_heads;
    p.rows = AR_ROWS;
    p.tiles = (int)(((int64_t)tokens * group + AR_ROWS - 1) / AR_ROWS) + sequences;
    // enough workgroups to fill the chip twice over, of at least `least` keys
    p.least = sequences == 1 ? 128 : 512;
    const int64_t most = (capacity + p.least - 1) / p.least;
    const int64_t want = (4 * 512 + (int64_t)p.tiles * kv_heads - 1) / ((int64_t)p.tiles * kv_heads);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(most, want), 128));
    p.bytes = p.splits > 1 ? (size_t)p.splits * tokens * q_heads * (dim + 2) * 4 : 0;
    return p;
}

hipError_t launch_attn(const AttnArgs &a, const AttnPlan &p, hipStream_t s)
{
    if (a.cache.type == kF16)
        return a.act == kF32 ? start_dim<Half, 2>(a, p, s) : start_dim<Half, 1>(a, p, s);
    return a.act == kF32 ? start_dim<BHalf, 3>(a, p, s) : start_dim<BHalf, 1>(a, p, s);
}

} // namespace ihip
