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

constexpr int ROW_THREADS = 1024;
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

// One workgroup a row, any distribution of logits: the boundary of the kept tokens
// is found digit by digit, 8 bits of the logits' order at a time.
__global__ void __launch_bounds__(ROW_THREADS) k_sample_row(SampleArgs a)
{
    __shared__ uint32_t count[256];
    __shared__ unsigned long long mass[256];
    __shared__ unsigned long long part[ROW_WAVES];
    __shared__ double dpart[ROW_WAVES];
    __shared__ uint32_t wkey[ROW_WAVES], wflag[ROW_WAVES];
    __shared__ int wat[ROW_WAVES];
    __shared__ uint32_t digit, left;
    __shared__ unsigned long long above;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    const int64_t base = row * a.row_step;
    const SampleRow r = sample_row(a, row);

    // the largest logit and its first place; what is not finite
    uint32_t best = 0, fl = 0;
    int at = 0x7fffffff;
    for (int i = tid; i < a.vocab; i += ROW_THREADS) {
        const float l = sample_logit(a.logits, base + i, a.type);
        fl |= sample_flags(l);
        const uint32_t k = sample_key(l);
        if (k > best)
            best = k, at = i;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t k = __shfl_xor(best, d);
        const int i = __shfl_xor(at, d);
        fl |= __shfl_xor(fl, d);
        if (k > best || (k == best && i < at))
            best = k, at = i;
    }
    if (lane == 0)
        wkey[wave] = best, wat[wave] = at, wflag[wave] = fl;
    __syncthreads();
    for (int i = 0; i < ROW_WAVES; ++i) {
        fl |= wflag[i];
        if (wkey[i] > best || (wkey[i] == best && wat[i] < at))
            best = wkey[i], at = wat[i];
    }
    if (fl & (kSampleNan | kSamplePosInf) || !(fl & kSampleFinite) || !(r.t > 0.0f)) {
        if (tid == 0)
            sample_done(a, row, fl, (fl & kSampleFinite) ? at : 0, 0.0);
        return;
    }
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
                digit = d, left = c, above = m;
            }
            __syncthreads();
            prefix |= digit << shift;
            n = left, kept = above;
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

} // namespace

hipError_t launch_sample(const SampleArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL(k_sample_row, dim3((unsigned)a.rows), dim3(ROW_THREADS), 0, s, a);
    return hipGetLastError();
}

} // namespace ihip
