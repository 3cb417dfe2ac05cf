// kv_pages.hip -- page tables and reference counts of the paged cache: the
// tables of the next step from the parents that were picked (fork, extension,
// release), the live pages moved to the front of the pool, and the copies of
// the pages both name.
//
// Which page a table gets is fixed by the definition alone -- free pages from
// the lowest index up, in the order of (child, place in its table) -- so the
// result does not depend on the order in which workgroups run.  The counts are
// changed by integer atomics, whose order does not matter.
#include "kv_launch.h"

namespace ihip {

namespace {

// The first place of `want` in v[0 .. n), or n: the lanes of a wave look at 64
// values at a time.
__device__ __forceinline__ int wave_find(const int32_t *v, int n, int want)
{
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const uint64_t hit = __ballot(i0 + lane < n && v[i0 + lane] == want);
        if (hit)
            return i0 + __builtin_ctzll(hit);
    }
    return n;
}

// A fork is bound by its chain of dependent reads (table, counts, free pages), not
// by bytes: 7 parents of up to 3000 tokens to 29 children take 8.6 us in one launch.
//
// A wave's work on child i, or on parent i - children.  A child's row takes over
// the pages of its parent's: the first child of a parent all of them (no count
// changes), a later one the full pages (their counts rise).  What a later child
// lacks, and what a longer child lacks at its end, is left to fork_take as
// `fresh`.  A parent without a child gives its pages back.
__device__ __forceinline__ void fork_row(const ForkArgs &a, int i)
{
    const int lane = threadIdx.x & 63;
    if (i >= a.children) {
        const int p = i - a.children;
        if (wave_find(a.parents, a.children, p) < a.children)
            return;
        for (int j = lane; j < a.stride; j += 64) {
            const int id = a.table[(int64_t)p * a.stride + j];
            if ((unsigned)id < (unsigned)a.pages)
                atomicSub(&a.refs[id], 1);
            else if (id >= a.pages && a.flags)
                atomicOr(a.flags, kFlagKvPage);
        }
        return;
    }
    const int c = i, p = a.parents[c];
    const bool alive = (unsigned)p < (unsigned)a.sequences;
    const bool first = alive && wave_find(a.parents, a.children, p) == c;
    const int64_t cap = (int64_t)a.stride * a.page_size;
    const int told = alive ? a.lens[p] : 0;
    const int len = told < 0 ? 0 : told > cap ? (int)cap : told;
    const int full = len / a.page_size;
    const int64_t longer = ((int64_t)len + a.room + a.page_size - 1) / a.page_size;
    const int need = longer > a.stride ? a.stride : (int)longer;
    int fresh = 0, copied = -1, from = a.stride;
    for (int j0 = 0; j0 < a.stride; j0 += 64) {
        const int j = j0 + lane;
        const bool in = j < a.stride;
        int id = in && alive ? a.table[(int64_t)p * a.stride + j] : -1;
        if (id >= a.pages) {
            if (a.flags)
                atomicOr(a.flags, kFlagKvPage);
            id = -1;
        }
        const bool keep = id >= 0 && (first || j < full);
        if (keep && !first)
            atomicAdd(&a.refs[id], 1);
        // -2: a page that fork_take is to find
        const bool lacks = in && !keep && j < need;
        const uint64_t lack = __ballot(lacks);
        if (lack && !fresh)
            from = j0;
        fresh += __popcll(lack);
        if (in)
            a.table_out[(int64_t)c * a.stride + j] = keep ? id : lacks ? -2 : -1;
        // the page that this child shares no longer: copied into the one it gets
        const uint64_t part = __ballot(lacks && !first && id >= 0 && j == full && len % a.page_size);
        if (part)
            copied = __builtin_amdgcn_readlane(id, __builtin_ctzll(part));
    }
    if (lane == 0) {
        a.fresh[c] = fresh;
        a.fresh[a.children + c] = from; // no entry before this place is missing
        a.lens_out[c] = len;
        a.copies[2 * c] = copied;
        a.copies[2 * c + 1] = -1;
        if (a.flags && (told != len || longer > a.stride || p >= a.sequences))
            atomicOr(a.flags, kFlagKvLength);
    }
}

constexpr int FORK_THREADS = 256;
// Tables that one workgroup takes, in one launch: its 16 waves take the rows in
// turns, which costs the GPU what the second launch would cost the host.  us in a
// graph and of host time, one launch against two: 1 parent to 3 children 4.6 and
// 12.4, 5.5 and 15.1; 7 of up to 3000 tokens to 29 (6084 entries) 11.2 and 12.6, 8.9
// and 15.0; 12 to 52 17.1, 10.6; 16 of up to 4000 to 48 21.9, 11.4; 4 of up to 16000
// to 60 70, 19 (the host's times as before).
constexpr int FORK_ROWS = 40, FORK_ENTRIES = 1 << 13;

__global__ void __launch_bounds__(FORK_THREADS) k_fork_rows(ForkArgs a)
{
    const int i = blockIdx.x * (FORK_THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (i < a.children + a.sequences)
        fork_row(a, i);
}

constexpr int TAKE_THREADS = 1024;
constexpr int TAKE_PER = 4; // counts a thread looks at in one step

// Inclusive sums over the workgroup's TAKE_THREADS values; `part` holds one
// int a wave.  Every thread must call it.
__device__ __forceinline__ int block_scan(int v, int *part, int &total)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int up = __shfl_up(v, d);
        v += lane >= d ? up : 0;
    }
    if (lane == 63)
        part[wave] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < TAKE_THREADS / 64; ++w) {
        const int n = part[w];
        before += w < wave ? n : 0;
        total += n;
    }
    __syncthreads();
    return before + v;
}

// The free pages, lowest first, to the children's missing entries in order.
// One workgroup: free pages are found 4096 counts at a time and each step hands
// out what it found; the search ends with the last entry, so that it reads the
// counts only up to there.
__device__ __forceinline__ void fork_take(const ForkArgs &a)
{
    __shared__ int part[TAKE_THREADS / 64];
    __shared__ int found[TAKE_THREADS * TAKE_PER];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // fresh[] becomes the sums before each child; `total` of all of them
    int total = 0;
    for (int c0 = 0; c0 < a.children; c0 += TAKE_THREADS) {
        const int c = c0 + tid, n = c < a.children ? a.fresh[c] : 0;
        int sum;
        const int upto = block_scan(n, part, sum);
        if (c < a.children)
            a.fresh[c] = total + upto - n;
        total += sum;
    }
    __syncthreads(); // fresh[] is read by other waves below
    int given = 0;
    for (int p0 = 0; given < total && p0 < a.pages; p0 += TAKE_THREADS * TAKE_PER) {
        int free[TAKE_PER], n = 0;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u) {
            const int p = p0 + tid * TAKE_PER + u;
            free[u] = p < a.pages && a.refs[p] == 0;
            n += free[u];
        }
        int sum;
        int at = block_scan(n, part, sum) - n;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u)
            if (free[u])
                found[at++] = p0 + tid * TAKE_PER + u;
        __syncthreads();
        const int last = min(given + sum, total); // entries given .. last - 1 get a page in this step
        // a wave a child whose entries are among them
        for (int c = wave; c < a.children; c += TAKE_THREADS / 64) {
            const int lo = a.fresh[c], hi = c + 1 < a.children ? a.fresh[c + 1] : total;
            if (hi <= given || lo >= last)
                continue;
            int32_t *row = a.table_out + (int64_t)c * a.stride;
            const int old = a.copies[2 * c];
            const int full = a.lens_out[c] / a.page_size;
            // entries that an earlier step filled are no longer -2: the count
            // starts behind them
            int rank = max(lo, given);
            for (int j0 = a.fresh[a.children + c]; j0 < a.stride && rank < min(hi, last); j0 += 64) {
                const int j = j0 + lane;
                const bool lacks = j < a.stride && row[j] == -2;
                const uint64_t all = __ballot(lacks);
                const int mine = rank + __popcll(all & ((1ull << lane) - 1));
                if (lacks && mine < last) {
                    const int id = found[mine - given];
                    row[j] = id;
                    a.refs[id] = 1;
                    if (old >= 0 && j == full)
                        a.copies[2 * c + 1] = id;
                }
                rank += __popcll(all);
            }
        }
        given = last;
        __syncthreads(); // found[] is written again
    }
    // no page left: the entries stay empty and nothing is copied into them
    if (given < total) {
        if (a.flags && tid == 0)
            atomicOr(a.flags, kFlagKvFull);
        for (int64_t i = tid; i < (int64_t)a.children * a.stride; i += TAKE_THREADS)
            if (a.table_out[i] == -2)
                a.table_out[i] = -1;
        for (int c = tid; c < a.children; c += TAKE_THREADS)
            if (a.copies[2 * c + 1] < 0)
                a.copies[2 * c] = -1;
    }
}

__global__ void __launch_bounds__(TAKE_THREADS) k_fork_take(ForkArgs a) { fork_take(a); }

// Both for small tables, as one launch.
__global__ void __launch_bounds__(TAKE_THREADS) k_fork(ForkArgs a)
{
    for (int i = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); i < a.children + a.sequences; i += TAKE_THREADS / 64)
        fork_row(a, i);
    __syncthreads(); // (the counts' atomics and the rows are in L2, and no wave has read them before)
    fork_take(a);
}

// The used pages at or behind index `used` (their number), in order, to the
// free ones before it, in order.  One workgroup, two passes over the counts:
// the number of used pages, then the moves; holes and movers are matched through
// the list of copies, whose second places first collect the holes.  Bound by the
// latency of its steps: 9.6 us for 4099 pages, of which the copies that follow
// take 107.
__global__ void __launch_bounds__(TAKE_THREADS) k_compact(CompactArgs a)
{
    __shared__ int part[TAKE_THREADS / 64];
    const int tid = threadIdx.x;
    int used = 0;
    for (int p0 = 0; p0 < a.pages; p0 += TAKE_THREADS * TAKE_PER) {
        int n = 0;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u) {
            const int p = p0 + tid * TAKE_PER + u;
            n += p < a.pages && a.refs[p] > 0;
        }
        int sum;
        block_scan(n, part, sum);
        used += sum;
    }
    // the holes, in order, into copies[2 r + 1]; there are at most pages / 2
    // (a hole lies before `used`, and each has a used page behind it)
    int holes = 0;
    for (int p0 = 0; p0 < used; p0 += TAKE_THREADS * TAKE_PER) {
        int hole[TAKE_PER], n = 0;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u) {
            const int p = p0 + tid * TAKE_PER + u;
            hole[u] = p < used && a.refs[p] <= 0;
            n += hole[u];
            if (p < used)
                a.to[p] = p;
        }
        int sum;
        int at = holes + block_scan(n, part, sum) - n;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u)
            if (hole[u])
                a.copies[2 * at++ + 1] = p0 + tid * TAKE_PER + u;
        holes += sum;
    }
    __syncthreads();
    int moved = 0;
    for (int p0 = used; p0 < a.pages; p0 += TAKE_THREADS * TAKE_PER) {
        int move[TAKE_PER], n = 0;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u) {
            const int p = p0 + tid * TAKE_PER + u;
            move[u] = p < a.pages && a.refs[p] > 0;
            n += move[u];
        }
        int sum;
        int at = moved + block_scan(n, part, sum) - n;
#pragma unroll
        for (int u = 0; u < TAKE_PER; ++u) {
            const int p = p0 + tid * TAKE_PER + u;
            if (p >= a.pages)
                continue;
            if (!move[u]) {
                a.to[p] = p;
                continue;
            }
            const int id = a.copies[2 * at + 1];
            a.copies[2 * at++] = p;
            a.to[p] = id;
            a.refs[id] = a.refs[p];
            a.refs[p] = 0;
        }
        moved += sum;
    }
    for (int i = moved + tid; i < a.pages / 2; i += TAKE_THREADS)
        a.copies[2 * i] = a.copies[2 * i + 1] = -1;
    if (tid == 0)
        *a.moved = moved;
}

__global__ void __launch_bounds__(256) k_compact_tables(CompactArgs a)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * 256) {
        const int id = a.table[i];
        if ((unsigned)id < (unsigned)a.pages)
            a.table[i] = a.to[id];
        else if (id >= a.pages && a.flags)
            atomicOr(a.flags, kFlagKvPage);
    }
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
constexpr int COPY_THREADS = 256;
constexpr int COPY_PER = 4;                                // 16-byte loads in flight a thread
constexpr int COPY_BYTES = COPY_THREADS * COPY_PER * 16;   // a workgroup's item

struct CopyArgs {
    uint8_t *k, *v;
    int64_t page_bytes, page_stride, layer_stride;
    int layers, pages, n, pieces; // pieces: items of one page of K in one layer
    const int32_t *copies, *count;
    uint32_t *flags;
};

// Page copies, bound by HBM: one item is 16 KB of one page of K or V in one
// layer.  The grid fills the chip once and walks the items, so that a list
// whose length is only known on the device costs nothing for its empty end.
// 532 MB in 107 us, 5.0 TB/s (a copy of 4 GB reaches 4.75).
__global__ void __launch_bounds__(COPY_THREADS) k_kv_copy(CopyArgs a)
{
    const int tid = threadIdx.x;
    const int n = a.count ? kv_clamp(*a.count, 0, a.n) : a.n;
    const int64_t per = (int64_t)a.pieces * 2 * a.layers, items = per * n;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int c = (int)(it / per);
        int64_t r = it - (int64_t)c * per;
        const int layer = (int)(r / (2 * a.pieces));
        r -= (int64_t)layer * (2 * a.pieces);
        const int src = a.copies[2 * c], dst = a.copies[2 * c + 1];
        if (src < 0 || dst < 0 || src == dst)
            continue;
        if (src >= a.pages || dst >= a.pages) {
            if (a.flags && tid == 0)
                atomicOr(a.flags, kFlagKvPage);
            continue;
        }
        if (a.flags && r == 0 && layer == 0) {
            // a page written twice, or read by another pair, would hold a mix: said, once a pair
            bool mix = false;
            for (int i = tid; i < n; i += COPY_THREADS)
                mix |= i != c && a.copies[2 * i] >= 0 && a.copies[2 * i + 1] >= 0 &&
                       (a.copies[2 * i] == dst || a.copies[2 * i + 1] == dst);
            if (mix)
                atomicOr(a.flags, kFlagKvPage);
        }
        uint8_t *pool = (r < a.pieces ? a.k : a.v) + layer * a.layer_stride;
        const int64_t off = (r < a.pieces ? r : r - a.pieces) * COPY_BYTES;
        const uint8_t *from = pool + src * a.page_stride + off + 16 * tid;
        uint8_t *to = pool + dst * a.page_stride + off + 16 * tid;
        const int64_t left = a.page_bytes - off - 16 * tid; // bytes from this thread's first on
        u4 v[COPY_PER];
#pragma unroll
        for (int u = 0; u < COPY_PER; ++u)
            v[u] = left > 16 * COPY_THREADS * u ? *(const u4 *)(from + 16 * COPY_THREADS * u) : u4{};
#pragma unroll
        for (int u = 0; u < COPY_PER; ++u)
            if (left > 16 * COPY_THREADS * u)
                *(u4 *)(to + 16 * COPY_THREADS * u) = v[u];
    }
}

} // namespace

hipError_t launch_kv_fork(const ForkArgs &a, hipStream_t s)
{
    const int64_t rows = (int64_t)a.children + a.sequences;
    if (a.children > 0 && rows <= FORK_ROWS && rows * a.stride <= FORK_ENTRIES) {
        hipLaunchKernelGGL(k_fork, dim3(1), dim3(TAKE_THREADS), 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(k_fork_rows, dim3((uint32_t)((rows + FORK_THREADS / 64 - 1) / (FORK_THREADS / 64))), dim3(FORK_THREADS),
                       0, s, a);
    if (a.children > 0)
        hipLaunchKernelGGL(k_fork_take, dim3(1), dim3(TAKE_THREADS), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const CompactArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL(k_compact, dim3(1), dim3(TAKE_THREADS), 0, s, a);
    if (a.entries > 0) {
        const int64_t wg = (a.entries + 255) / 256, most = 4 * (int64_t)device_cus();
        hipLaunchKernelGGL(k_compact_tables, dim3((uint32_t)(wg < most ? wg : most)), dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

hipError_t launch_kv_copy(void *k, void *v, int64_t page_bytes, int64_t page_stride, int64_t layer_stride,
                          int layers, int pages, const int32_t *copies, int n, const int32_t *count,
                          uint32_t *flags, hipStream_t s)
{
    CopyArgs a{(uint8_t *)k, (uint8_t *)v, page_bytes, page_stride, layer_stride, layers, pages, n,
               (int)((page_bytes + COPY_BYTES - 1) / COPY_BYTES), copies, count, flags};
    const int64_t items = (int64_t)a.pieces * 2 * layers * n, most = 8 * (int64_t)device_cus();
    hipLaunchKernelGGL(k_kv_copy, dim3((uint32_t)(items < most ? items : most)), dim3(COPY_THREADS), 0, s, a);
    return hipGetLastError();
}

} // namespace ihip
