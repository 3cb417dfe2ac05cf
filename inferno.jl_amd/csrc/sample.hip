// sample.hip -- a token per row of logits, by temperature, top-k, top-p and min-p,
// from one given random number a row.
//
//   w_i = e^((l_i - max) / T);  the tokens in order of l, ties by index;
//   top-k keeps the first k, top-p the shortest prefix whose weights reach p of what
//   top-k left, min-p those with w_i >= min_p (all prefixes of that order);
//   the token is the first, by index, where the kept weights up to it pass u Z.
//
// Weights are formed and summed in 64 bits: rounded to 32, the sums of 150000 of them
// would be off by more than the weights between which the token changes.  Where atomics
// add them (top-p's boundary) they are whole numbers of 2^-46 of the largest weight (less
// for more than 2^16 tokens), whose sums do not depend on the order; the sums that the
// token and its logprob come from are floating, in a fixed order.
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
// with more tokens at a boundary than kSampleList (many equal logits, or temperatures
// so high that hundreds of thousands of tokens weigh alike).
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
                if (m[j] < low && k != best)
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
// What of a row is zero between calls: the largest logit seen (its key, then ~place),
// what is not finite, workgroups that have ended, tokens listed.
struct Record {
    unsigned long long best;
    uint32_t flags, ended[2], listed, pad[2];
};
static_assert(sizeof(Record) == kSampleRecord, "a row's record");

// The prefixes that top-k and top-p keep end within these bins: nothing over bin
// `whole` is cut, and the tokens of bin k and of bins p_low .. p_high are listed.
struct Bounds {
    unsigned long long k_over, p_over; // weights over bin k, and over bin p_low
    unsigned long long all;            // of all tokens (where top-k is off)
    uint32_t k_count;                  // tokens over bin k
    int k, p_low, p_high, whole;
};

struct Part { // of a slice
    unsigned long long best;
    double sum;
};

__device__ __forceinline__ Record *record_of(const SampleArgs &a, int r)
{
    return (Record *)a.work + r;
}
__device__ __forceinline__ unsigned long long agent_load(const unsigned long long *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store(unsigned long long *p, unsigned long long v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void agent_clear(uint32_t *p)
{
    __hip_atomic_store(p, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Whether this workgroup is the last of the row's `n` to come here.  What passes
// between them goes through memory that all of the chip sees (agent_load and _store,
// atomics); a workgroup counts itself when its stores have arrived, and the last one
// sets the count to 0 again.
__device__ __forceinline__ bool last_of(uint32_t *count, int n, int *lds)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        *lds = atomicInc(count, (uint32_t)n - 1) == (uint32_t)n - 1;
    __syncthreads();
    return *lds;
}

// f(logit, index) for this thread's logits of a slice, 4 neighbours a thread at a time
template <typename F>
__device__ __forceinline__ void each_logit(const SampleArgs &a, int row, int slice, F f)
{
    const int begin = slice * a.plan.per, end = (int)min((int64_t)begin + a.plan.per, (int64_t)a.vocab);
    const int64_t base = row * a.row_step;
    const int size = a.type == kF32 ? 4 : 2;
    const bool wide = (((uintptr_t)a.logits + (uintptr_t)(base * size)) & (uintptr_t)(4 * size - 1)) == 0; // (begin is a multiple of 4)
    for (int i0 = begin + 4 * (int)threadIdx.x; i0 < end; i0 += 4 * 4 * ROW_THREADS) {
        // four such groups in flight
        gd_f4 l[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int i = i0 + b * 4 * ROW_THREADS;
            if (wide && i + 3 < end)
                l[b] = gd_load4(a.logits, base + i, a.type);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    l[b][e] = i + e < end ? sample_logit(a.logits, base + i + e, a.type) : 0.0f;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i0 + b * 4 * ROW_THREADS + e < end)
                    f(l[b][e], i0 + b * 4 * ROW_THREADS + e);
    }
}

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

// Bins by distance from the largest logit: 32 to a factor of 2 in weight down to 2^-32,
// then 64 to a factor of 2 in distance.  In order of the logits.
__device__ __forceinline__ int bin_of(float l, float most, float rate)
{
    const float d = (most - l) * rate;
    if (d < 32.0f)
        return (int)(d * 32.0f);
    constexpr uint32_t from = 0x42000000u >> 17; // 32
    return (int)min((__float_as_uint(d) >> 17) - from + 1024u, (uint32_t)(kSampleBins - 1));
}
__device__ __forceinline__ float bin_rate(float t)
{
    return fminf(1.44269504f / t, 3e38f);
}

__device__ __forceinline__ bool filtered(const SampleRow &r, int vocab, bool &by_k, bool &by_p)
{
    by_k = r.k > 0 && r.k < vocab;
    by_p = r.p < 1.0f;
    return by_k || by_p;
}

// The row's token from its slices' sums: `sum` (this thread's slice's, threads behind
// the last slice 0) and what a token has to pass to be kept.
struct PickLds {
    double part[ROW_WAVES], before;
    int slice, wat[ROW_WAVES], wlast[ROW_WAVES];
};
__device__ void pick(const SampleArgs &a, int row, const SampleRow &r, const SampleScale &sc, unsigned long long best, uint32_t fl,
                     double sum, unsigned long long border, double low, PickLds &lds)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double before;
    const double total = wg_scan(sum, lds.part, before);
    const double want = sample_u(r.u) * total;
    // the first slice at which the sums pass it, else the last one that has any
    if (tid == 0)
        lds.slice = 0x7fffffff;
    __syncthreads();
    if (sum > 0.0 && before + sum > want)
        atomicMin(&lds.slice, tid);
    __syncthreads();
    if (lds.slice == 0x7fffffff) {
        __syncthreads();
        if (tid == 0)
            lds.slice = -1;
        __syncthreads();
        if (sum > 0.0)
            atomicMax(&lds.slice, tid);
        __syncthreads();
    }
    const int slice = max(lds.slice, 0);
    if (tid == slice)
        lds.before = before;
    __syncthreads();
    double run = lds.before;
    const int64_t base = row * a.row_step;
    const int begin = slice * a.plan.per, end = (int)min((int64_t)begin + a.plan.per, (int64_t)a.vocab);
    int token = (int)~(uint32_t)best;
    for (int i0 = begin; i0 < end; i0 += 4 * ROW_THREADS) {
        double m[4], mine = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = i0 + 4 * tid + e;
            const float l = i < end ? sample_logit(a.logits, base + i, a.type) : -__builtin_inff();
            const unsigned long long o = best_of(l, i);
            m[e] = i < end && o >= border ? sample_weight(sc, l) : 0.0;
            if (m[e] < low && o != best)
                m[e] = 0.0;
            mine += m[e];
        }
        double ahead;
        const double all = wg_scan(mine, lds.part, ahead);
        double upto = run + ahead;
        int found = 0x7fffffff, last = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            upto += m[e];
            if (m[e] > 0.0) {
                last = i0 + 4 * tid + e;
                if (upto > want && found == 0x7fffffff)
                    found = last;
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            found = min(found, __shfl_xor(found, d));
            last = max(last, __shfl_xor(last, d));
        }
        if (lane == 0)
            lds.wat[wave] = found, lds.wlast[wave] = last;
        __syncthreads();
        for (int i = 0; i < ROW_WAVES; ++i) {
            found = min(found, lds.wat[i]);
            last = max(last, lds.wlast[i]);
        }
        if (last >= 0)
            token = last;
        if (found != 0x7fffffff) {
            token = found;
            break;
        }
        run += all;
        __syncthreads();
    }
    if (tid == 0)
        sample_done(a, row, fl, token, log(sample_weight(sc, sample_logit(a.logits, base + token, a.type)) / total));
}

// Whether the row's token needs no sums: what is not finite, or the greedy choice
__device__ __forceinline__ bool settled(const SampleArgs &a, int row, const SampleRow &r, unsigned long long best, uint32_t fl)
{
    if (!(fl & (kSampleNan | kSamplePosInf)) && (fl & kSampleFinite) && r.t > 0.0f)
        return false;
    if (threadIdx.x == 0 && a.tokens)
        sample_done(a, row, fl, (fl & kSampleFinite) ? (int)~(uint32_t)best : 0, 0.0);
    return true;
}

// Without filters, one launch: a slice's largest logit, then its weights relative to
// that (the slice's second reading comes from the caches); the row's last workgroup
// joins the slices and looks the token up in the one where it lies.
__global__ void __launch_bounds__(ROW_THREADS) k_sample_plain(SampleArgs a)
{
    __shared__ unsigned long long wbest[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES];
    __shared__ double part[ROW_WAVES];
    __shared__ PickLds lds;
    __shared__ int lds_last;
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    unsigned long long best = 0;
    uint32_t fl = 0;
    each_logit(a, row, slice, [&](float l, int i) {
        fl |= sample_flags(l);
        const unsigned long long o = best_of(l, i);
        best = o > best ? o : best;
    });
    wg_best(best, fl, wbest, wfl);
    double sum = 0.0;
    if ((fl & kSampleFinite) && !(fl & (kSampleNan | kSamplePosInf)) && r.t > 0.0f) {
        const SampleScale sc = sample_scale(r.t, sample_value((uint32_t)(best >> 32)), a.vocab);
        each_logit(a, row, slice, [&](float l, int) { sum += sample_weight(sc, l); });
        sum = wg_sum(sum, part);
    }
    Record *const rec = record_of(a, rr);
    Part *const parts = (Part *)(a.work + a.plan.parts) + (int64_t)rr * a.plan.slices;
    if (tid == 0) {
        agent_store(&parts[slice].best, best);
        agent_store((unsigned long long *)&parts[slice].sum, __double_as_longlong(sum));
        atomicOr(&rec->flags, fl);
    }
    if (!last_of(&rec->ended[0], a.plan.slices, &lds_last))
        return;
    unsigned long long mine = 0;
    sum = 0.0;
    if (tid < a.plan.slices) {
        mine = agent_load(&parts[tid].best);
        sum = __longlong_as_double(agent_load((unsigned long long *)&parts[tid].sum));
    }
    best = mine;
    fl = __hip_atomic_load(&rec->flags, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wg_best(best, fl, wbest, wfl);
    if (tid == 0)
        agent_clear(&rec->flags);
    if (settled(a, row, r, best, fl))
        return;
    const SampleScale sc = sample_scale(r.t, sample_value((uint32_t)(best >> 32)), a.vocab);
    if (sum > 0.0)
        sum *= sample_weight(sc, sample_value((uint32_t)(mine >> 32)));
    pick(a, row, r, sc, best, fl, sum, 0, 0.0, lds);
}

// With filters: the rows' largest logits (and empty bins for the next launch) ...
__global__ void __launch_bounds__(ROW_THREADS) k_sample_best(SampleArgs a, int bins)
{
    __shared__ unsigned long long wbest[ROW_WAVES];
    __shared__ uint32_t wfl[ROW_WAVES];
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices;
    if (bins) {
        uint32_t *const b = (uint32_t *)(a.work + a.plan.bins + (int64_t)rr * kSampleBins * 12);
        for (int i = slice * ROW_THREADS + threadIdx.x; i < kSampleBins * 3; i += a.plan.slices * ROW_THREADS)
            b[i] = 0;
    }
    unsigned long long best = 0;
    uint32_t fl = 0;
    each_logit(a, a.row0 + rr, slice, [&](float l, int i) {
        fl |= sample_flags(l);
        const unsigned long long o = best_of(l, i);
        best = o > best ? o : best;
    });
    wg_best(best, fl, wbest, wfl);
    if (threadIdx.x == 0) {
        atomicMax(&record_of(a, rr)->best, best);
        atomicOr(&record_of(a, rr)->flags, fl);
    }
}

// ... the tokens and weights of every bin, and from them the bins in which the kept
// prefixes end ...
__global__ void __launch_bounds__(ROW_THREADS) k_sample_bins(SampleArgs a)
{
    __shared__ unsigned long long mass[kSampleBins];
    __shared__ uint32_t count[kSampleBins];
    __shared__ unsigned long long part[ROW_WAVES];
    __shared__ int lds_last, ends[3];
    __shared__ unsigned long long over[2];
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    Record *const rec = record_of(a, rr);
    const uint32_t fl = rec->flags;
    bool by_k, by_p;
    if ((fl & (kSampleNan | kSamplePosInf)) || !(fl & kSampleFinite) || !(r.t > 0.0f) || !filtered(r, a.vocab, by_k, by_p))
        return;
    for (int i = tid; i < kSampleBins; i += ROW_THREADS)
        mass[i] = 0, count[i] = 0;
    __syncthreads();
    const float most = sample_value((uint32_t)(rec->best >> 32)), rate = bin_rate(r.t);
    const SampleScale sc = sample_scale(r.t, most, a.vocab);
    each_logit(a, row, slice, [&](float l, int) {
        const int b = bin_of(l, most, rate);
        if (by_k)
            atomicAdd(&count[b], 1u);
        if (by_p)
            atomicAdd(&mass[b], (unsigned long long)sample_mass(sc, l));
    });
    __syncthreads();
    unsigned long long *const all_mass = (unsigned long long *)(a.work + a.plan.bins + (int64_t)rr * kSampleBins * 12);
    uint32_t *const all_count = (uint32_t *)(all_mass + kSampleBins);
    for (int i = tid; i < kSampleBins; i += ROW_THREADS) {
        if (mass[i])
            atomicAdd(&all_mass[i], mass[i]);
        if (count[i])
            atomicAdd(&all_count[i], count[i]);
    }
    if (!last_of(&rec->ended[0], a.plan.slices, &lds_last))
        return;
    // 4 neighbouring bins a thread
    constexpr int E = kSampleBins / ROW_THREADS;
    unsigned long long m[E], c[E], before_m, before_c, sum_m = 0, sum_c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        m[i] = agent_load(&all_mass[E * tid + i]);
        c[i] = __hip_atomic_load(&all_count[E * tid + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sum_m += m[i], sum_c += c[i];
    }
    const unsigned long long all = wg_scan(sum_m, part, before_m);
    wg_scan(sum_c, part, before_c);
    if (tid < 3)
        ends[tid] = kSampleBins;
    __syncthreads();
    Bounds bo{};
    bo.all = all, bo.k = bo.p_low = bo.p_high = bo.whole = kSampleBins;
    if (by_k) {
        unsigned long long upto = before_c;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (c[i] && upto < (unsigned long long)r.k && upto + c[i] >= (unsigned long long)r.k) { // (one bin of one thread)
                ends[0] = E * tid + i;
                over[0] = upto;
                over[1] = before_m;
                for (int e = 0; e < i; ++e)
                    over[1] += m[e];
            }
            upto += c[i];
        }
        __syncthreads();
        bo.k = bo.whole = ends[0], bo.k_count = (uint32_t)over[0], bo.k_over = over[1];
    }
    if (by_p) {
        // weights that top-k leaves: between those over bin k and those down to it
        const unsigned long long in_k = by_k ? agent_load(&all_mass[min(bo.k, kSampleBins - 1)]) : 0;
        const double least = (double)fmaxf(r.p, 0.0f) * (double)(by_k ? bo.k_over : all);
        const double largest = (double)fmaxf(r.p, 0.0f) * (double)(by_k ? bo.k_over + in_k : all);
        unsigned long long upto = before_m;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (m[i] && (double)(upto + m[i]) >= least)
                atomicMin(&ends[1], E * tid + i);
            if (m[i] && (double)(upto + m[i]) >= largest)
                atomicMin(&ends[2], E * tid + i);
            upto += m[i];
        }
        __syncthreads();
        bo.p_low = bo.whole = ends[1], bo.p_high = ends[2];
        upto = before_m;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (E * tid + i == ends[1])
                over[0] = upto;
            upto += m[i];
        }
        __syncthreads();
        bo.p_over = over[0];
    }
    if (tid == 0)
        ((Bounds *)(a.work + a.plan.bounds))[rr] = bo;
}

// ... and the tokens in those bins, and the weights of the ones over them.  The row's
// last workgroup resolves the former and picks the token.
struct ListLds {
    unsigned long long order[kSampleList], mass[kSampleList];
};
__global__ void __launch_bounds__(ROW_THREADS) k_sample_pick(SampleArgs a, int bins)
{
    __shared__ union {
        ListLds list;
        RowLds row;
    } u;
    __shared__ PickLds lds;
    __shared__ double part[ROW_WAVES];
    __shared__ unsigned long long upart[ROW_WAVES], border;
    __shared__ int lds_last;
    const int slice = blockIdx.x % a.plan.slices, rr = blockIdx.x / a.plan.slices, row = a.row0 + rr, tid = threadIdx.x;
    const SampleRow r = sample_row(a, row);
    Record *const rec = record_of(a, rr);
    Part *const parts = (Part *)(a.work + a.plan.parts) + (int64_t)rr * a.plan.slices;
    unsigned long long *const list = (unsigned long long *)(a.work + a.plan.list) + (int64_t)rr * kSampleList;
    const uint32_t fl = rec->flags;
    const unsigned long long best = rec->best;
    const float most = sample_value((uint32_t)(best >> 32)), rate = bin_rate(r.t);
    const bool sums = !(fl & (kSampleNan | kSamplePosInf)) && (fl & kSampleFinite) && r.t > 0.0f;
    bool by_k = false, by_p = false;
    Bounds bo{};
    bo.k = bo.p_low = bo.p_high = bo.whole = kSampleBins;
    if (sums && bins && filtered(r, a.vocab, by_k, by_p))
        bo = ((const Bounds *)(a.work + a.plan.bounds))[rr];
    const SampleScale sc = sample_scale(r.t, most, a.vocab);
    const double low = r.min_p > 0.0f ? (double)r.min_p : 0.0;
    if (sums) {
        double sum = 0.0;
        each_logit(a, row, slice, [&](float l, int i) {
            const int b = bin_of(l, most, rate);
            const unsigned long long o = best_of(l, i);
            if (b < bo.whole) {
                const double w = sample_weight(sc, l);
                sum += w >= low || o == best ? w : 0.0;
            } else if (b == bo.k || (b >= bo.p_low && b <= bo.p_high)) {
                const uint32_t n = atomicAdd(&rec->listed, 1u);
                if (n < (uint32_t)kSampleList)
                    agent_store(&list[n], o);
            }
        });
        sum = wg_sum(sum, part);
        if (tid == 0)
            agent_store((unsigned long long *)&parts[slice].sum, __double_as_longlong(sum));
    }
    if (!last_of(&rec->ended[1], a.plan.slices, &lds_last))
        return;
    const int n = (int)__hip_atomic_load(&rec->listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (tid == 0) {
        agent_store(&rec->best, 0);
        agent_clear(&rec->flags);
        agent_clear(&rec->listed);
    }
    if (settled(a, row, r, best, fl))
        return;
    if (n > kSampleList) {
        sample_whole_row(a, row, r, (uint32_t)(best >> 32), (int)~(uint32_t)best, fl, u.row);
        return;
    }
    double sum = tid < a.plan.slices ? __longlong_as_double(agent_load((unsigned long long *)&parts[tid].sum)) : 0.0;
    unsigned long long from = 0; // the last kept token, in the order of best_of
    if (by_k || by_p) {
        constexpr int E = kSampleList / ROW_THREADS;
        for (int i = tid; i < n; i += ROW_THREADS) {
            const unsigned long long o = agent_load(&list[i]);
            u.list.order[i] = o;
            u.list.mass[i] = by_p ? sample_mass(sc, sample_value((uint32_t)(o >> 32))) : 0;
        }
        if (tid == 0)
            border = ~0ull;
        __syncthreads();
        unsigned long long total = bo.all; // weights that top-k leaves
        if (by_k) {
            // the listed tokens of bin k by their places among them
            unsigned long long kept = 0, before;
            for (int e = 0; e < E; ++e) {
                const int i = tid + e * ROW_THREADS;
                if (i >= n)
                    break;
                const unsigned long long o = u.list.order[i];
                if (bin_of(sample_value((uint32_t)(o >> 32)), most, rate) != bo.k)
                    continue;
                uint32_t rank = bo.k_count;
                for (int j = 0; j < n; ++j) {
                    const unsigned long long p = u.list.order[j];
                    rank += p > o && bin_of(sample_value((uint32_t)(p >> 32)), most, rate) == bo.k;
                }
                if (rank < (uint32_t)r.k) {
                    kept += u.list.mass[i];
                    atomicMin(&border, o);
                }
            }
            total = bo.k_over + wg_scan(kept, upart, before);
            __syncthreads();
            from = border;
        }
        if (by_p) {
            const double want = (double)fmaxf(r.p, 0.0f) * (double)total;
            __syncthreads();
            if (tid == 0)
                border = ~0ull;
            __syncthreads();
            for (int e = 0; e < E; ++e) {
                const int i = tid + e * ROW_THREADS;
                if (i >= n)
                    break;
                const unsigned long long o = u.list.order[i];
                unsigned long long over = bo.p_over;
                for (int j = 0; j < n; ++j)
                    over += u.list.order[j] > o ? u.list.mass[j] : 0;
                if (o >= from && ((double)over < want || o == best))
                    atomicMin(&border, o);
            }
            __syncthreads();
            from = border;
        }
        // the kept ones' weights, in order, to their slices
        __syncthreads();
        for (int e = 0; e < E; ++e) {
            const int i = tid + e * ROW_THREADS;
            if (i >= n)
                break;
            const unsigned long long o = u.list.order[i];
            int rank = 0;
            for (int j = 0; j < n; ++j)
                rank += u.list.order[j] > o;
            u.list.mass[rank] = o; // (mass is read)
        }
        __syncthreads();
        if (tid < a.plan.slices)
            for (int i = 0; i < n; ++i) {
                const unsigned long long o = u.list.mass[i];
                if (o < from)
                    break;
                if ((int)(~(uint32_t)o / (uint32_t)a.plan.per) == tid) {
                    const double w = sample_weight(sc, sample_value((uint32_t)(o >> 32)));
                    sum += w >= low || o == best ? w : 0.0;
                }
            }
    }
    pick(a, row, r, sc, best, fl, sum, from, low, lds);
}

} // namespace

hipError_t launch_sample(SampleArgs a, hipStream_t s)
{
    const bool bins = a.top_k || a.top_p;
    const int rows = a.rows;
    for (a.row0 = 0; a.row0 < rows; a.row0 += a.plan.rows) {
        const dim3 grid((unsigned)((rows - a.row0 < a.plan.rows ? rows - a.row0 : a.plan.rows) * a.plan.slices));
        if (!bins && !a.min_p) {
            hipLaunchKernelGGL(k_sample_plain, grid, dim3(ROW_THREADS), 0, s, a);
            continue;
        }
        hipLaunchKernelGGL(k_sample_best, grid, dim3(ROW_THREADS), 0, s, a, (int)bins);
        if (bins)
            hipLaunchKernelGGL(k_sample_bins, grid, dim3(ROW_THREADS), 0, s, a);
        hipLaunchKernelGGL(k_sample_pick, grid, dim3(ROW_THREADS), 0, s, a, (int)bins);
    }
    return hipGetLastError();
}

} // namespace ihip
