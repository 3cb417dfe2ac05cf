// sample.hip -- a token per row of logits, by temperature, top-k, top-p and min-p,
// from one given random number a row.
//
//   w_i = e^((l_i - max) / T);  the tokens in order of l, ties by index;
//   top-k keeps the first k, top-p the shortest prefix whose weights reach p of what
//   top-k left, min-p those with w_i >= min_p (all prefixes of that order);
//   the token is the first, by index, where the kept weights up to it pass u Z.
//
// Weights are formed (to 2^-48) and summed in 64 bits: rounded to 32, the sums of 150000 of them
// would be off by more than the weights between which the token changes.  Where atomics
// add them (top-p's boundary, and to their slices the kept ones of the bins where a prefix
// ends) they are whole numbers of 2^-46 of the largest weight (2^-44 for 151936 tokens), whose
// sums do not depend on the order; the other sums that the token comes from, and all that its
// logprob does, are floating, in a fixed order.
#include "sample_common.h"

namespace ihip {

namespace {

constexpr int ROW_THREADS = kSampleThreads;
constexpr int ROW_WAVES = ROW_THREADS / 64;

// Sum over a workgroup's threads, and of those before this one; two barriers.
template <typename T>
__device__ __forceinline__ T wg_scan(T v, T *part, T &before)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T sum = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const T up = __shfl_up(sum, d);
        sum += lane >= d ? up : T(0);
    }
    __syncthreads();
    if (lane == 63)
        part[wave] = sum;
    __syncthreads();
    T all = 0, waves = 0; // (a difference would not be the sum of the threads before)
    for (int i = 0; i < ROW_WAVES; ++i) {
        waves = i == wave ? all : waves;
        all += part[i];
    }
    const T left = __shfl_up(sum, 1);
    before = waves + (lane ? left : T(0));
    return all;
}

struct RowLds {
    uint32_t count[256];
    unsigned long long mass[256], part[ROW_WAVES], above;
    double dpart[ROW_WAVES];
    uint32_t wkey[ROW_WAVES], digit, left;
    int wat[ROW_WAVES];
};

// A whole row by one workgroup, any distribution of logits: the boundary of the kept
// tokens is found digit by digit, 8 bits of the logits' order at a time.  For rows
// with more tokens at a boundary than kSampleList: many equal logits, or tens of thousands
// that weigh alike.  Bound by one workgroup's passes: a row of 151936 normally spread logits of
// deviation 1 at T = 2 and top-p = 0.5 712 us, 61 such rows 1200; 262144 of deviation 2 at T = 2 and
// top-p = 0.9 1455 (usual rows: 58 and 95).
__device__ void sample_whole_row(const SampleArgs &a, int row, const SampleRow &r, uint32_t best, int at, uint32_t fl, RowLds &lds)
{
    auto &count = lds.count;
    auto &mass = lds.mass;
    auto &part = lds.part;
    auto &dpart = lds.dpart;
    auto &wkey = lds.wkey;
    auto &wat = lds.wat;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t base = row * a.row_step;
    const SampleScale sc = sample_scale(r.t, sample_value(best), a.vocab);

    // the boundary: tokens over `border` are kept, and the first `ties` at it
    uint32_t border = 0, ties = 0xffffffffu;
    const double low = r.min_p > 0.0f ? (double)r.min_p : 0.0;
    unsigned long long total = ~0ull; // weights of what is kept so far
    for (int by = 0; by < 2; ++by) { // 0: top-k, 1: top-p
        if (by == 0 ? r.k <= 0 || r.k >= a.vocab : !(r.p < 1.0f))
            continue;
        if (by == 1 && total == ~0ull) {
            unsigned long long sum = 0, before;
            for (int i = tid; i < a.vocab; i += ROW_THREADS)
                sum += sample_mass(sc, sample_logit(a.logits, base + i, a.type));
            total = wg_scan(sum, part, before);
        }
        const double want = by == 1 ? (double)fmaxf(r.p, 0.0f) * (double)total : 0.0;
        const uint32_t border0 = border, ties0 = ties;
        uint64_t kept = 0; // weights over the boundary
        uint32_t n = 0, prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256)
                count[tid] = 0, mass[tid] = 0;
            __syncthreads();
            for (int i = tid; i < a.vocab; i += ROW_THREADS) {
                const float l = sample_logit(a.logits, base + i, a.type);
                const uint32_t k = sample_key(l);
                if ((shift == 24 || k >> (shift + 8) == prefix >> (shift + 8)) && k >= border0) {
                    atomicAdd(&count[(k >> shift) & 255], 1u);
                    atomicAdd(&mass[(k >> shift) & 255], (unsigned long long)sample_mass(sc, l));
                }
            }
            __syncthreads();
            if (tid == 0) {
                uint64_t m = kept;
                uint32_t c = n, d = 255;
                for (;; --d) { // the digit at which the prefix ends; it has tokens
                    const bool ends = by == 0 ? c + count[d] >= (uint32_t)r.k
                                              : count[d] && (double)(m + mass[d]) >= want;
                    if (ends || d == 0)
                        break;
                    m += mass[d], c += count[d];
                }
                lds.digit = d, lds.left = c, lds.above = m;
            }
            __syncthreads();
            prefix |= lds.digit << shift;
            n = lds.left, kept = lds.above;
        }
        // n tokens of weight `kept` lie over the boundary `prefix`
        border = prefix;
        const uint64_t each = sample_mass(sc, sample_value(border));
        uint32_t at_border = count[border & 255];
        if (border == border0 && ties0 < at_border)
            at_border = ties0; // (top-k has left so many)
        uint32_t take = at_border;
        if (by == 0)
            take = (uint32_t)r.k - n;
        else if (each > 0 && (double)kept < want) {
            // the first j with kept + j each >= want
            const double j = ceil((want - (double)kept) / (double)each);
            take = j < (double)at_border ? (uint32_t)j : at_border;
            if (take > 1 && (double)(kept + (uint64_t)(take - 1) * each) >= want)
                --take; // (the quotient was rounded up)
        } else if ((double)kept >= want)
            take = 0;
        if (n == 0 && take == 0)
            take = 1; // the likeliest token is always kept
        ties = take;
        total = kept + (uint64_t)take * each;
    }

    // the weights of what is kept, then the place where they pass u of them
    const int tile = ROW_THREADS * 4;
    double sum_kept = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        double run = 0.0;
        const double want = sample_u(r.u) * sum_kept;
        unsigned long long seen = 0; // ties so far
        int last = at;
        for (int t0 = 0; t0 < a.vocab; t0 += tile) {
            double m[4], sum = 0.0, before;
            unsigned long long mine = 0, rank;
            float l[4];
            for (int j = 0; j < 4; ++j) {
                const int i = t0 + 4 * tid + j;
                l[j] = i < a.vocab ? sample_logit(a.logits, base + i, a.type) : -__builtin_inff();
                mine += i < a.vocab && sample_key(l[j]) == border;
            }
            const unsigned long long in_tile = wg_scan(mine, part, rank);
            rank += seen;
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = sample_key(l[j]);
                bool keep = k > border;
                if (k == border)
                    keep = rank++ < ties;
                m[j] = keep && t0 + 4 * tid + j < a.vocab ? sample_weight(sc, l[j]) : 0.0;
                if (m[j] < low && t0 + 4 * tid + j != at)
                    m[j] = 0.0;
                sum += m[j];
            }
            seen += in_tile;
            const double all = wg_scan(sum, dpart, before);
            if (pass == 1) {
                int mylast = -1, found = 0x7fffffff;
                double upto = run + before;
                for (int j = 0; j < 4; ++j) {
                    upto += m[j];
                    if (m[j] > 0.0) {
                        mylast = t0 + 4 * tid + j;
                        if (upto > want && found == 0x7fffffff)
                            found = mylast;
                    }
                }
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    found = min(found, __shfl_xor(found, d));
                    mylast = max(mylast, __shfl_xor(mylast, d));
                }
                __syncthreads();
                if (lane == 0)
                    wat[wave] = found, wkey[wave] = (uint32_t)(mylast + 1);
                __syncthreads();
                for (int i = 0; i < ROW_WAVES; ++i) {
                    found = min(found, wat[i]);
                    mylast = max(mylast, (int)wkey[i] - 1);
                }
                if (mylast >= 0)
                    last = mylast;
                if (found != 0x7fffffff) {
                    last = found;
                    break;
                }
            }
            run += all;
        }
        if (pass == 0)
            sum_kept = run;
        else if (tid == 0)
            sample_done(a, row, fl, last, log(sample_weight(sc, sample_logit(a.logits, base + last, a.type)) / sum_kept));
    }
}


// ---- rows in slices ------------------------------------------------------------
// A row's slices go to workgroups all over the chip, and what they find to one that
// joins them, a launch later (a launch costs what a count of ended workgroups, and
// reads past the caches, would).  One row of 151936 fp32 logits, us: best 3.2, bins 6, merge 3.2,
// bounds 4.3, list 5.8, pick 12; bound by these launches and the loads and sums that
// follow each other in them (the logits are 0.1 at the rate of reads).  61 rows of bf16
// with mixed filters: 6.7, 17.5, 4.4, 4.6, 15, 24.3; bound by atomics to shared bins,
// 64-bit weights and the longest of the rows' lists.  256 rows of fp32 without filters: best 46
// (156 MB, 3.4 TB/s: 16 operations in 64 bits a weight beside its load), join 12.

struct Part { // of a slice
    unsigned long long best; // the largest logit (its key, then ~place)
    double sum;              // of weights
    uint32_t flags, pad;
};
static_assert(sizeof(Part) == kSamplePart, "a slice's values");

// The prefixes that top-k and top-p keep end within these bins: nothing over bin
// `whole` is cut, and the tokens of bin k and of bins p_low .. p_high are listed.
struct Bounds {
    unsigned long long k_over, p_over; // weights over bin k, and over bin p_low
    unsigned long long all;            // of all tokens (where top-k is off)
    uint32_t k_count;                  // tokens over bin k
    int k, p_low, p_high, whole;
    uint32_t listed;                   // tokens
};
static_assert(sizeof(Bounds) <= kSampleRecord, "a row's bounds");

__device__ __forceinline__ Part *parts_of(const SampleArgs &a, int rr)
{
    return (Part *)a.work + (int64_t)rr * a.plan.slices;
}
__device__ __forceinline__ Bounds *bounds_of(const SampleArgs &a, int rr)
{
    return (Bounds *)(a.work + a.plan.bounds + (int64_t)rr * kSampleRecord);
}

template <int TYPE>
struct LogitOf;
template <>
struct LogitOf<kF32> {
    typedef float T;
};
template <>
struct LogitOf<kF16> {
    typedef _Float16 T;
};
template <>
struct LogitOf<kBF16> {
    typedef __bf16 T;
};

// A thread's N logits of a slice, 4 neighbours at a time, all on their way at once;
// -infinity behind the row's end.
template <int TYPE, int N>
struct Slice {
    float l[N];
    int begin, end;

    __device__ __forceinline__ Slice(const SampleArgs &a, int row, int slice)
    {
        typedef typename LogitOf<TYPE>::T T;
        typedef T T4 __attribute__((ext_vector_type(4)));
        begin = slice * (N * ROW_THREADS), end = min(begin + N * ROW_THREADS, a.vocab);
        const T *const p = (const T *)a.logits + row * a.row_step;
        const bool wide = ((uintptr_t)(p + begin) & (sizeof(T4) - 1)) == 0 && end == begin + N * ROW_THREADS;
        if (wide) {
            T4 v[N / 4];
#pragma unroll
            for (int j = 0; j < N; j += 4)
                v[j / 4] = *(const T4 *)(p + at(j));
#pragma unroll
            for (int j = 0; j < N; ++j)
                l[j] = (float)v[j / 4][j % 4];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                l[j] = (float)p[min(at(j), a.vocab - 1)];
#pragma unroll
            for (int j = 0; j < N; ++j)
                l[j] = at(j) < end ? l[j] : -__builtin_inff();
        }
    }
    __device__ __forceinline__ int at(int j) const
    {
        return begin + (j / 4 * ROW_THREADS + (int)threadIdx.x) * 4 + j % 4;
    }
};

// The larger of keys, the lowest place among equal ones
__device__ __forceinline__ unsigned long long best_of(float l, int at)
{
    return (unsigned long long)sample_key(l) << 32 | (uint32_t)~at;
}

__device__ __forceinline__ void wg_best(unsigned long long &best, uint32_t &fl, unsigned long long *wbest, uint32_t *wfl)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned long long o = __shfl_xor(best, d);
        best = o > best ? o : best;
        fl |= __shfl_xor(fl, d);
    }
    if ((threadIdx.x & 63) == 0)
        wbest[threadIdx.x >> 6] = best, wfl[threadIdx.x >> 6] = fl;
    __syncthreads();
    for (int i = 0; i < ROW_WAVES; ++i) {
        best = wbest[i] > best ? wbest[i] : best;
        fl |= wfl[i];
    }
    __syncthreads();
}

// Sum over the workgroup in a fixed order
__device__ __forceinline__ double wg_sum(double v, double *part)
{
    v = gd_wave_sum(v);
    if ((threadIdx.x & 63) == 0)
        part[threadIdx.x >> 6] = v;
    __syncthreads();
    double all = 0.0;
    for (int i = 0; i < ROW_WAVES; ++i)
        all += part[i];
    __syncthreads();
    return all;
}

// Bins by distance from the largest logit: 16 to a factor of 2 in weight down to 2^-32,
// then 32 to a factor of 2 in distance.  In order of the logits.
__device__ __forceinline__ int bin_of(float l, float most, float rate)
{
    const float d = fmaf(-0.5f, l, 0.5f * most) * rate; // (halves: the difference of two logits may pass the range)
    if (d < 32.0f)
        return (int)(d * 16.0f);
    constexpr uint32_t from = 0x42000000u >> 18; // 32
    return (int)min((__float_as_uint(d) >> 18) - from + 512u, (uint32_t)(kSampleBins - 1));
}
// From this bin on (over 1150 factors of 2 below the largest) weights are 0 in 64 bits:
// where top-k's cut falls among them it cuts nothing that counts.
constexpr int ZERO_BIN = 680;
__device__ __forceinline__ float bin_rate(float t) // of half a difference
{
    return fminf(2 * 1.44269504f / t, 3e38f);
}

__device__ __forceinline__ bool filtered(const SampleRow &r, int vocab, bool &by_k, bool &by_p)
{
    by_k = r.k > 0 && r.k < vocab;
    by_p = r.p < 1.0f;
    return by_k || by_p;
}

// The row's token from its slices' sums: `sum` (this thread's slice's, threads behind
// the last slice 0), `total` (what the logprob is a share of) and the last kept token.
struct PickLds {
    double part[ROW_WAVES], before;
    int first[ROW_WAVES], last[ROW_WAVES];
};

// The first thread for which `yes`, and the last one for which `some` (-1: none).  By
// ballots: hundreds of atomics to one address would take longer than all the rest.
__device__ __forceinline__ int2 first_and_last(bool yes, bool some, int *first, int *last)
{
    const int wave = threadIdx.x >> 6;
    const uint64_t y = __ballot(yes), h = __ballot(some);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        first[wave] = y ? 64 * wave + __builtin_ctzll(y) : 0x7fffffff;
        last[wave] = h ? 64 * wave + 63 - __builtin_clzll(h) : -1;
    }
    __syncthreads();
    int2 r = make_int2(0x7fffffff, -1);
    for (int i = 0; i < ROW_WAVES; ++i) {
        r.x = min(r.x, first[i]);
        r.y = max(r.y, last[i]);
    }
    return make_int2(r.x == 0x7fffffff ? -1 : r.x, r.y);
}

// The first thread whose sum passes `want` (the sum of the threads before it is handed
// on in lds.before), else the last one that has any; -1: none has.
__device__ __forceinline__ int first_passing(double sum, double before, double want, PickLds &lds)
{
    const int2 r = first_and_last(sum > 0.0 && before + sum > want, sum > 0.0, lds.first, lds.last);
    const int at = r.x >= 0 ? r.x : r.y;
    if ((int)threadIdx.x == at)
        lds.before = before;
    __syncthreads();
    return at;
}

// (The slice comes to its threads through LDS: read as neighbours to a thread, it costs a
// cache line a logit, 4 us of 12.)
constexpr int STAGED = kSampleWide + kSampleWide / 16;
__device__ void pick(const SampleArgs &a, int row, const SampleRow &r, const SampleScale &sc, unsigned long long best, uint32_t fl,
                     double sum, double total, unsigned long long border, double low, PickLds &lds, float *staged)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t base = row * a.row_step;
    // what token i counts
    auto weight = [&](int i, float l) {
        const unsigned long long o = best_of(l, i);
        const double w = o >= border ? sample_weight(sc, l) : 0.0;
        return w < low && o != best ? 0.0 : w;
    };
    // the slice, then the thread's share of it, then the token
    double before;
    const double want = sample_u(r.u) * wg_scan(sum, lds.part, before);
    const int slice = max(first_passing(sum, before, want, lds), 0);
    double run = lds.before;
    constexpr int MOST = kSampleWide / ROW_THREADS;
    const int share = a.plan.per / ROW_THREADS; // neighbours
    const int begin = slice * a.plan.per, end = min(begin + a.plan.per, a.vocab);
    {
        // (one look at the type for all loads: beside each, they would wait for each other)
        uint32_t bits[MOST];
        if (a.type == kF32) {
            const uint32_t *const l = (const uint32_t *)a.logits + base;
#pragma unroll
            for (int e = 0; e < MOST; ++e)
                bits[e] = l[min(begin + e * ROW_THREADS + tid, end - 1)];
        } else {
            const uint16_t *const l = (const uint16_t *)a.logits + base;
#pragma unroll
            for (int e = 0; e < MOST; ++e)
                bits[e] = l[min(begin + e * ROW_THREADS + tid, end - 1)];
        }
#pragma unroll
        for (int e = 0; e < MOST; ++e)
            staged[e * ROW_THREADS + tid + (e * ROW_THREADS + tid) / 16] =
                a.type == kF32 ? __uint_as_float(bits[e]) : a.type == kF16 ? h2f(bits[e]) : __uint_as_float(bits[e] << 16);
    }
    __syncthreads();
    sum = 0.0;
#pragma unroll 4
    for (int e = 0; e < share; ++e) {
        const int i = tid * share + e;
        sum += begin + i < end ? weight(begin + i, staged[i + i / 16]) : 0.0;
    }
    wg_scan(sum, lds.part, before);
    const int owner = first_passing(sum, run + before, want, lds);
    if (tid >= 64)
        return;
    run = lds.before;
    const int in = max(owner, 0) * share + min(lane, share - 1), i = begin + in;
    const double w = owner >= 0 && lane < share && i < end ? weight(i, staged[in + in / 16]) : 0.0;
    double upto = w;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(upto, d);
        upto += lane >= d ? up : 0.0;
    }
    const uint64_t has = __ballot(w > 0.0), passed = __ballot(w > 0.0 && run + upto > want);
    const int at = passed ? __builtin_ctzll(passed) : has ? 63 - __builtin_clzll(has) : -1;
    if (lane == max(at, 0)) // (no kept token: the likeliest)
        sample_done(a, row, fl, at < 0 ? (int)~(uint32_t)best : i, at < 0 ? 0.0 : log(w / total));
}

// Whether the row's weights matter: it is finite, and not for the greedy choice
__device__ __forceinline__ bool weighed(float t, uint32_t fl)
{
    return !(fl & (kSampleNan | kSamplePosInf)) && (fl & kSampleFinite) && t > 0.0f;
}
__device__ __forceinline__ void settle(const SampleArgs &a, int row, unsigned long long best, uint32_t fl)
{
    if (threadIdx.x == 0)
        sample_done(a, row, fl, (fl & kSampleFinite) ? (int)~(uint32_t)best : 0, 0.0);
}

// A slice's largest logit, and what is not finite in it
template <typename S>
__device__ __forceinline__ void slice_best(const S &x, unsigned long long &best, uint32_t &fl, unsigned long long *wbest, uint32_t *wfl)
{
    constexpr int N = (int)(sizeof x.l / 4);
    float most = -__builtin_inff();
    bool nan = false;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        most = fmaxf(most, x.l[j]);
        nan |= x.l[j] != x.l[j];
    }
    int at = 0x7fffffff;
#pragma unroll
    for (int j = N - 1; j >= 0; --j)
        at = x.l[j] == most ? x.at(j) : at;
    fl = (nan ? kSampleNan : 0) | sample_flags(most);
    best = best_of(most, at);
    wg_best(best, fl, wbest, wfl);
}

// A row's largest logit and flags, from its slices'
__device__ __forceinline__ void row_best(const SampleArgs &a, int rr, unsigned long long &best, uint32_t &fl, unsigned long long *wbest,
                                         uint32_t *wfl)
{
    best = 0, fl = 0;
    if ((int)threadIdx.x < a.plan.slices) {
        const Part p = parts_of(a, rr)[threadIdx.x];
        best = p.best, fl = p.flags;
    }
    wg_best(best, fl, wbest, wfl);
}

// Every slice's largest logit and, without filters, its weights relative to that.
template <int TYPE, int N, bool SUMS>
__global__ void __launch_bounds__(ROW_THREADS) k_sample_best(SampleArgs a)
{
    __shared__ unsigned long long wbest[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES];
    __shared__ double part[ROW_WAVES];
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices, row = a.row0 + rr;
    const Slice<TYPE, N> x(a, row, slice);
    if (SUMS)
        sample_fill_table();
    unsigned long long best;
    uint32_t fl;
    slice_best(x, best, fl, wbest, wfl);
    double sum = 0.0;
    if (SUMS) {
        const float t = a.temperature ? a.temperature[row] : 1.0f;
        if (weighed(t, fl)) {
            const SampleScale sc = sample_scale(t, sample_value((uint32_t)(best >> 32)), a.vocab);
#pragma unroll
            for (int j = 0; j < N; ++j)
                sum += sample_weight(sc, x.l[j]);
            sum = wg_sum(sum, part);
        }
    }
    if (threadIdx.x == 0)
        parts_of(a, rr)[slice] = Part{best, sum, fl, 0};
}

// Without filters: the slices joined, and the token looked up in the one where it lies.
__global__ void __launch_bounds__(ROW_THREADS) k_sample_join(SampleArgs a)
{
    __shared__ unsigned long long wbest[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES];
    __shared__ PickLds lds;
    __shared__ float staged[STAGED];
    const int rr = blockIdx.x, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    sample_fill_table();
    unsigned long long best;
    uint32_t fl;
    row_best(a, rr, best, fl, wbest, wfl);
    if (!weighed(r.t, fl)) {
        settle(a, row, best, fl);
        return;
    }
    const SampleScale sc = sample_scale(r.t, sample_value((uint32_t)(best >> 32)), a.vocab);
    double sum = 0.0;
    if (tid < a.plan.slices) {
        const Part p = parts_of(a, rr)[tid];
        sum = p.sum > 0.0 ? p.sum * sample_weight(sc, sample_value((uint32_t)(p.best >> 32))) : 0.0;
    }
    pick(a, row, r, sc, best, fl, sum, wg_sum(sum, lds.part), 0, 0.0, lds, staged);
}

// With top-k or top-p: the tokens and weights of every bin of a slice ...
template <int TYPE, int N>
__global__ void __launch_bounds__(ROW_THREADS) k_sample_bins(SampleArgs a)
{
    // (bins in two copies, by lane, where neighbouring tokens' atomics meet less often: 61
    // rows 18.9 us, one copy 21.6, four 19.6, with weights of six operations more)
    constexpr int COPIES = 2;
    __shared__ unsigned long long mass[COPIES * kSampleBins];
    __shared__ uint32_t count[COPIES * kSampleBins];
    __shared__ unsigned long long wbest[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES];
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    bool by_k, by_p;
    if (!filtered(r, a.vocab, by_k, by_p) || !(r.t > 0.0f))
        return;
    const Slice<TYPE, N> x(a, row, slice);
    sample_fill_table();
    for (int i = tid; i < COPIES * kSampleBins; i += ROW_THREADS)
        mass[i] = 0, count[i] = 0;
    const int copy = tid % COPIES;
    unsigned long long best;
    uint32_t fl;
    row_best(a, rr, best, fl, wbest, wfl);
    if (!weighed(r.t, fl))
        return;
    const float most = sample_value((uint32_t)(best >> 32)), rate = bin_rate(r.t);
    const SampleScale sc = sample_scale(r.t, most, a.vocab);
    // (the last bin, of tokens that a grammar rules out, is counted apart: its atomics
    // would all have one address)
    uint32_t far = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int b = bin_of(x.l[j], most, rate);
        if (x.at(j) >= x.end)
            continue;
        far += b == kSampleBins - 1;
        if (by_k && b < kSampleBins - 1)
            atomicAdd(&count[b * COPIES + copy], 1u);
        if (by_p) {
            const unsigned long long m = sample_mass(sc, x.l[j]);
            if (m)
                atomicAdd(&mass[b * COPIES + copy], m);
        }
    }
    if (by_k && far)
        atomicAdd(&count[(kSampleBins - 1) * COPIES + copy], far);
    __syncthreads();
    unsigned long long *const all_mass =
        (unsigned long long *)(a.work + a.plan.bins + ((int64_t)rr * a.plan.slices + slice) * (kSampleBins * 12));
    uint32_t *const all_count = (uint32_t *)(all_mass + kSampleBins);
    for (int i = tid; i < kSampleBins; i += ROW_THREADS) {
        unsigned long long m = 0;
        uint32_t c = 0;
#pragma unroll
        for (int k = 0; k < COPIES; ++k)
            m += mass[i * COPIES + k], c += count[i * COPIES + k];
        if (by_p)
            all_mass[i] = m;
        if (by_k)
            all_count[i] = c;
    }
}

// ... summed over the slices, 64 bins a workgroup: one workgroup alone would wait for
// hundreds of KB (38 slices: 20 us) ...
constexpr int MERGE_BINS = 64;
__global__ void __launch_bounds__(ROW_THREADS) k_sample_merge(SampleArgs a)
{
    __shared__ unsigned long long mass[ROW_WAVES][MERGE_BINS];
    __shared__ uint32_t count[ROW_WAVES][MERGE_BINS];
    constexpr int BLOCKS = kSampleBins / MERGE_BINS;
    const int rr = blockIdx.x / BLOCKS, row = a.row0 + rr, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bin = blockIdx.x % BLOCKS * MERGE_BINS + lane;
    const SampleRow r = sample_row(a, row);
    bool by_k, by_p;
    if (!filtered(r, a.vocab, by_k, by_p) || !(r.t > 0.0f))
        return;
    // (a row that is not weighed has no bins: what lies there is summed and not looked at)
    const uint8_t *const bins = a.work + a.plan.bins + (int64_t)rr * a.plan.slices * (kSampleBins * 12);
    unsigned long long m = 0;
    uint32_t c = 0;
#pragma unroll 4
    for (int q = wave; q < a.plan.slices; q += ROW_WAVES) {
        const uint8_t *const from = bins + (int64_t)q * (kSampleBins * 12);
        m += ((const unsigned long long *)from)[bin];
        c += ((const uint32_t *)(from + kSampleBins * 8))[bin];
    }
    mass[wave][lane] = m, count[wave][lane] = c;
    __syncthreads();
    if (wave)
        return;
#pragma unroll
    for (int w = 1; w < ROW_WAVES; ++w)
        m += mass[w][lane], c += count[w][lane];
    uint8_t *const to = a.work + a.plan.merged + (int64_t)rr * (kSampleBins * 12);
    ((unsigned long long *)to)[bin] = by_p ? m : 0;
    ((uint32_t *)(to + kSampleBins * 8))[bin] = by_k ? c : 0;
}

// ... from them the bins in which the kept prefixes end ...
__global__ void __launch_bounds__(ROW_THREADS) k_sample_bounds(SampleArgs a)
{
    __shared__ unsigned long long mass[kSampleBins];
    __shared__ uint32_t wfl[ROW_WAVES];
    __shared__ unsigned long long part[ROW_WAVES], over[2];
    __shared__ int ends[3];
    constexpr int E = kSampleBins / ROW_THREADS; // neighbouring bins to a thread
    static_assert(E == 2, "loaded as pairs");
    const int rr = blockIdx.x, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    bool by_k, by_p;
    if (!filtered(r, a.vocab, by_k, by_p) || !(r.t > 0.0f))
        return;
    unsigned long long best;
    uint32_t fl;
    row_best(a, rr, best, fl, part, wfl);
    if (!weighed(r.t, fl))
        return;
    const uint8_t *const bins = a.work + a.plan.merged + (int64_t)rr * (kSampleBins * 12);
    const ulonglong2 mv = ((const ulonglong2 *)bins)[tid];
    const uint2 cv = ((const uint2 *)(bins + kSampleBins * 8))[tid];
    const unsigned long long m[E]{mv.x, mv.y}, c[E]{cv.x, cv.y};
    unsigned long long before_m, before_c;
    mass[E * tid] = m[0], mass[E * tid + 1] = m[1];
    if (tid < 3)
        ends[tid] = kSampleBins;
    const unsigned long long all = wg_scan(m[0] + m[1], part, before_m);
    wg_scan(c[0] + c[1], part, before_c);
    Bounds bo{};
    bo.all = all, bo.k = bo.p_low = bo.p_high = bo.whole = kSampleBins;
    if (by_k) {
        unsigned long long upto = before_c, upto_m = before_m;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (upto < (unsigned long long)r.k && upto + c[i] >= (unsigned long long)r.k) // (one bin of one thread)
                ends[0] = E * tid + i, over[0] = upto, over[1] = upto_m;
            upto += c[i], upto_m += m[i];
        }
        __syncthreads();
        by_k = ends[0] < ZERO_BIN;
        if (by_k)
            bo.k = bo.whole = ends[0], bo.k_count = (uint32_t)over[0], bo.k_over = over[1];
    }
    __syncthreads(); // over is read
    if (by_p) {
        // p of the weights that top-k leaves, which lie between those over bin k and
        // those down to it
        const double p = (double)fmaxf(r.p, 0.0f);
        const double least = p * (double)(by_k ? bo.k_over : all);
        const double largest = p * (double)(by_k ? bo.k_over + mass[bo.k] : all);
        // the first bin with weights down to which they reach it
        unsigned long long upto = before_m;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const unsigned long long prior = upto;
            upto += m[i];
            if (m[i] && (double)upto >= least && (prior == 0 || (double)prior < least))
                ends[1] = E * tid + i, over[0] = prior;
            if (m[i] && (double)upto >= largest && (prior == 0 || (double)prior < largest))
                ends[2] = E * tid + i;
        }
        __syncthreads();
        bo.p_low = bo.whole = ends[1], bo.p_high = ends[2], bo.p_over = over[0];
    }
    if (tid == 0)
        *bounds_of(a, rr) = bo;
}

// ... and the tokens in those bins, and the weights of the ones over them.  BINS: some
// row has them; else (min-p alone) nothing is listed.
template <int TYPE, int N, bool BINS>
__global__ void __launch_bounds__(ROW_THREADS) k_sample_list(SampleArgs a)
{
    __shared__ unsigned long long mine[BINS ? kSampleList : 1];
    __shared__ unsigned long long wbest[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES], listed, first;
    __shared__ double part[ROW_WAVES];
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    if (!(r.t > 0.0f))
        return;
    const Slice<TYPE, N> x(a, row, slice);
    sample_fill_table();
    if (tid == 0)
        listed = 0;
    unsigned long long best;
    uint32_t fl;
    row_best(a, rr, best, fl, wbest, wfl);
    if (!weighed(r.t, fl))
        return;
    const float most = sample_value((uint32_t)(best >> 32)), rate = bin_rate(r.t);
    const SampleScale sc = sample_scale(r.t, most, a.vocab);
    const double low = r.min_p > 0.0f ? (double)r.min_p : 0.0;
    bool by_k = false, by_p = false;
    int k = kSampleBins, p_low = kSampleBins, p_high = kSampleBins, whole = kSampleBins;
    if (BINS && filtered(r, a.vocab, by_k, by_p)) {
        const Bounds *const bo = bounds_of(a, rr);
        k = bo->k, p_low = bo->p_low, p_high = bo->p_high, whole = bo->whole;
    }
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int b = BINS ? bin_of(x.l[j], most, rate) : 0;
        if (b < whole) {
            const double w = sample_weight(sc, x.l[j]);
            sum += w >= low || best_of(x.l[j], x.at(j)) == best ? w : 0.0;
        } else if (BINS && (b == k || (b >= p_low && b <= p_high)) && x.at(j) < x.end) {
            const uint32_t n = atomicAdd(&listed, 1u);
            if (n < (uint32_t)kSampleList)
                mine[n] = best_of(x.l[j], x.at(j));
        }
    }
    sum = wg_sum(sum, part);
    if (tid == 0)
        parts_of(a, rr)[slice].sum = sum;
    if (!BINS || listed == 0)
        return;
    if (tid == 0)
        first = atomicAdd(&bounds_of(a, rr)->listed, listed);
    __syncthreads();
    unsigned long long *const list = (unsigned long long *)(a.work + a.plan.list) + (int64_t)rr * kSampleList;
    for (uint32_t i = tid; i < listed && first + i < (uint32_t)kSampleList; i += ROW_THREADS)
        list[first + i] = mine[i];
}

// ... which are put in order and cut; then the token.
struct ListLds {
    unsigned long long order[kSampleList], masses[kSampleList], mass[kSampleSlices];
};
__global__ void __launch_bounds__(ROW_THREADS) k_sample_pick(SampleArgs a)
{
    __shared__ union {
        ListLds list;
        RowLds row;
        float staged[STAGED]; // (the list is used up by then)
    } u;
    __shared__ PickLds lds;
    __shared__ unsigned long long upart[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES];
    __shared__ int first_k, kept;
    const int rr = blockIdx.x, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    // (loaded together, before it is known whether they are looked at)
    const unsigned long long *const list = (const unsigned long long *)(a.work + a.plan.list) + (int64_t)rr * kSampleList;
    const unsigned long long early = list[tid];
    Bounds bo = *bounds_of(a, rr);
    double sum = tid < a.plan.slices ? parts_of(a, rr)[tid].sum : 0.0;
    bool by_k, by_p;
    const bool cut_row = filtered(r, a.vocab, by_k, by_p);
    if (!cut_row)
        bo.listed = 0;
    sample_fill_table();
    unsigned long long best;
    uint32_t fl;
    row_best(a, rr, best, fl, upart, wfl);
    if (!weighed(r.t, fl)) {
        settle(a, row, best, fl);
        return;
    }
    const float most = sample_value((uint32_t)(best >> 32)), rate = bin_rate(r.t);
    const SampleScale sc = sample_scale(r.t, most, a.vocab);
    const double low = r.min_p > 0.0f ? (double)r.min_p : 0.0;
    const int n = (int)bo.listed;
    if (n > kSampleList) {
        sample_whole_row(a, row, r, (uint32_t)(best >> 32), (int)~(uint32_t)best, fl, u.row);
        return;
    }
    double total = wg_sum(sum, lds.part);
    unsigned long long from = 0; // the last kept token, in the order of best_of
    if (cut_row && bo.whole < kSampleBins) {
        // the listed tokens in order, the first first; 0 behind them
        int size = 2;
        while (size < n)
            size *= 2;
        unsigned long long *const order = u.list.order;
        for (int i = tid; i < size; i += ROW_THREADS)
            order[i] = i < n ? (i < ROW_THREADS ? early : list[i]) : 0;
        for (int i = tid; i < kSampleSlices; i += ROW_THREADS)
            u.list.mass[i] = 0;
        __syncthreads();
        for (int run = 2; run <= size; run *= 2)
            for (int d = run / 2; d > 0; d /= 2) {
                for (int p = tid; p < size / 2; p += ROW_THREADS) {
                    const int i = 2 * p - (p & (d - 1)), j = i + d;
                    const unsigned long long x = order[i], y = order[j];
                    if ((x < y) == ((i & run) == 0))
                        order[i] = y, order[j] = x;
                }
                __syncthreads();
            }
        // neighbours to a thread; the weights of those before
        const int each = (n + ROW_THREADS - 1) / ROW_THREADS, at0 = each * tid, at1 = min(at0 + each, n);
        unsigned long long *const masses = u.list.masses;
        unsigned long long mine = 0, before = 0;
        if (by_p)
#pragma unroll 1
            for (int i = at0; i < at1; ++i)
                mine += masses[i] = sample_mass(sc, sample_value((uint32_t)(order[i] >> 32)));
        int cut = n; // kept by top-k: those before it
        unsigned long long left = bo.all;
        if (bo.k < kSampleBins) {
            // (bin k's tokens are the last ones)
            int ahead = 0;
#pragma unroll 1
            for (int i = at0; i < at1; ++i)
                ahead += bin_of(sample_value((uint32_t)(order[i] >> 32)), most, rate) != bo.k;
            const int2 at = first_and_last(false, ahead > 0, lds.first, lds.last);
            if (tid == max(at.y, 0))
                first_k = at.y < 0 ? 0 : at0 + ahead;
            __syncthreads();
            cut = first_k + (r.k - (int)bo.k_count);
            unsigned long long in_k = 0;
            if (by_p)
#pragma unroll 1
                for (int i = max(at0, first_k); i < min(at1, cut); ++i)
                    in_k += masses[i];
            left = bo.k_over + wg_scan(in_k, upart, before);
        }
        wg_scan(mine, upart, before);
        const double want = (double)fmaxf(r.p, 0.0f) * (double)left;
        unsigned long long over = bo.p_over + before;
        int last = 0;
#pragma unroll 1
        for (int i = at0; i < min(at1, cut); ++i) {
            if (!by_p || (double)over < want || order[i] == best)
                last = i + 1;
            over += by_p ? masses[i] : 0;
        }
        const int2 at = first_and_last(false, last > 0, lds.first, lds.last);
        if (tid == max(at.y, 0))
            kept = last;
        __syncthreads();
        from = kept ? order[kept - 1] : best;
        double w = 0.0;
#pragma unroll 1
        for (int i = at0; i < min(at1, kept); ++i) {
            double x = sample_weight(sc, sample_value((uint32_t)(order[i] >> 32)));
            x = x >= low || order[i] == best ? x : 0.0;
            w += x;
            // (to their slices as whole numbers: in any order.  Where the last kept token is
            // asked for, a slice with one is not to look empty.)
            if (x > 0.0)
                atomicAdd(&u.list.mass[~(uint32_t)order[i] / (uint32_t)a.plan.per],
                          (unsigned long long)fmax(rint(ldexp(x, sc.bits)), r.u >= 1.0f ? 1.0 : 0.0));
        }
        total += wg_sum(w, lds.part);
        if (tid < a.plan.slices)
            sum += ldexp((double)u.list.mass[tid], -sc.bits);
    }
    pick(a, row, r, sc, best, fl, sum, total, from, low, lds, u.staged);
}

template <int TYPE, int N>
void launch(const SampleArgs &a, unsigned rows, hipStream_t s)
{
    const dim3 slices(rows * (unsigned)a.plan.slices), threads(ROW_THREADS);
    const bool bins = a.top_k || a.top_p;
    if (!bins && !a.min_p) {
        hipLaunchKernelGGL((k_sample_best<TYPE, N, true>), slices, threads, 0, s, a);
        hipLaunchKernelGGL(k_sample_join, dim3(rows), threads, 0, s, a);
        return;
    }
    hipLaunchKernelGGL((k_sample_best<TYPE, N, false>), slices, threads, 0, s, a);
    if (bins) {
        hipLaunchKernelGGL((k_sample_bins<TYPE, N>), slices, threads, 0, s, a);
        hipLaunchKernelGGL(k_sample_merge, dim3(rows * (kSampleBins / MERGE_BINS)), threads, 0, s, a);
        hipLaunchKernelGGL(k_sample_bounds, dim3(rows), threads, 0, s, a);
        hipLaunchKernelGGL((k_sample_list<TYPE, N, true>), slices, threads, 0, s, a);
    } else {
        hipLaunchKernelGGL((k_sample_list<TYPE, N, false>), slices, threads, 0, s, a);
    }
    hipLaunchKernelGGL(k_sample_pick, dim3(rows), threads, 0, s, a);
}

template <int TYPE>
void launch(const SampleArgs &a, unsigned rows, hipStream_t s)
{
    if (a.plan.per == kSampleWide)
        launch<TYPE, kSampleWide / ROW_THREADS>(a, rows, s);
    else
        launch<TYPE, kSampleNarrow / ROW_THREADS>(a, rows, s);
}

} // namespace

hipError_t launch_sample(SampleArgs a, hipStream_t s)
{
    const int rows = a.rows;
    for (a.row0 = 0; a.row0 < rows; a.row0 += a.plan.rows) {
        const unsigned n = (unsigned)(rows - a.row0 < a.plan.rows ? rows - a.row0 : a.plan.rows);
        if (a.type == kF32)
            launch<kF32>(a, n, s);
        else if (a.type == kF16)
            launch<kF16>(a, n, s);
        else
            launch<kBF16>(a, n, s);
    }
    return hipGetLastError();
}

} // namespace ihip
