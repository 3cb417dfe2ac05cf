// gd_chunk.hip -- the gated delta rule over sequences with many new tokens, 64 of
// them at a time on the matrix cores.  With G_i the sum of the logarithms of the
// decays up to token i of the chunk, S the state before it, and k, q of unit length,
//
//   A_ij = beta_i k_i.k_j e^(G_i - G_j), j < i;      T = (1 + A)^-1 diag(beta)
//   V' = T (V - e^G K S)                             (what the tokens write)
//   O = scale (e^G Q S + P V'),                      P_ij = q_i.k_j e^(G_i - G_j), j <= i
//   S <- e^G_64 S + (e^(G_64 - G) K)^T V'
//
// T and P do not depend on S: k_delta_prep forms them, and K and Q as matrix operands,
// for all chunks at once.  k_delta_scan then walks down a sequence's chunks, each wave
// with 16 columns of S, which do not touch the other columns.
//
// Operands are fp16 times a power of two (of a row of K and Q, of a column of S, V and
// V'), so that the largest value lies in 2^13 .. 2^14: values of F16 and BF16 inputs
// fit one part exactly down to 2^-27 of their row's largest; fp32 values and
// everything derived is held in two parts, which leave 2^-22 of a value, and products
// of the two lower parts (2^-22) are not formed.  Sums are fp32.  Rows' factors (unit
// length, e^G) are applied to the products, in fp32, so that K and Q are shared by the
// heads that read them.
#include "gd_launch.h"

namespace ihip {

namespace {

typedef _Float16 gd_h8 __attribute__((ext_vector_type(8)));
typedef float gd_f8 __attribute__((ext_vector_type(8)));

constexpr int TOP = 13; // operands' largest values have this binary exponent

// 2^(TOP - exponent of x), and its inverse; x >= 0.  (Below 2^-113 of nothing; an
// infinity or NaN is left one.)
__device__ __forceinline__ void gd_power(float x, float &to, float &back)
{
    const int e = max((int)(__float_as_uint(x) >> 23), 127 - 113);
    to = __uint_as_float((uint32_t)(254 + TOP - e) << 23);
    back = __uint_as_float((uint32_t)(e - TOP) << 23);
}

// x * by as one fp16 part, or its rest as the next one too
__device__ __forceinline__ void gd_split(gd_f8 x, float by, gd_h8 &hi, gd_h8 &lo)
{
    x = x * by;
    hi = __builtin_convertvector(x, gd_h8);
    lo = __builtin_convertvector(x - __builtin_convertvector(hi, gd_f8), gd_h8);
}

__device__ __forceinline__ gd_f4 gd_mfma(gd_h8 a, gd_h8 b, gd_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Fragments.  A 16-row tile of an operand is stored as the matrix cores take it: for
// each step of 32 columns, lane (g, r) = (lane / 16, lane % 16) holds of row r the
// columns 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3, 16 bytes a lane.  These are the
// rows that a lane holds of two tiles of a product's result, so that results (S, V')
// are the next product's operands without leaving their registers.

// ---- chunks' operands ------------------------------------------------------------
constexpr int PREP_THREADS = 256;
constexpr int TRI = 68; // floats from a row of a 64 x 64 matrix to the next, in LDS

// Lower triangle in LDS, column j times by[j], as fragments of two parts: 6 tiles of
// 16 x 32 (the others are zeros).  M holds zeros behind the diagonal of those.
__device__ __forceinline__ void store_tri(const float *M, const float *by, uint8_t *to)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    for (int t = threadIdx.x >> 6; t < 6; t += PREP_THREADS / 64) {
        const int m = t < 2 ? t : 2 + (t - 2) / 2, k = t < 2 ? 0 : (t - 2) & 1;
        const int c = 32 * k + 4 * g;
        const float *row = M + (16 * m + r) * TRI + c;
        gd_f8 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = row[i] * (by ? by[c + i] : 1.0f);
            x[4 + i] = row[16 + i] * (by ? by[c + 16 + i] : 1.0f);
        }
        gd_h8 hi, lo;
        gd_split(x, (float)(1 << TOP), hi, lo);
        *(gd_h8 *)(to + (2 * t) * 1024 + lane * 16) = hi;
        *(gd_h8 *)(to + (2 * t + 1) * 1024 + lane * 16) = lo;
    }
}

template <int KD, int PARTS>
__global__ void __launch_bounds__(PREP_THREADS) k_delta_prep(DeltaArgs a)
{
    constexpr int KS = KD / 32;               // steps of a row of K
    constexpr int FRAG = 4 * KS * PARTS * 1024; // bytes of K or Q
    constexpr int MATS = 3 * 64 * TRI * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[FRAG > MATS ? FRAG : MATS];
    __shared__ double G[64];
    __shared__ float beta[64], rk[64];
    float *const A = (float *)lds, *const T = A + 64 * TRI, *const P = T + 64 * TRI;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, r = lane & 15;
    const int h = blockIdx.x % a.v_heads, tile = blockIdx.x / a.v_heads, kh = h / a.group;
    int c = 0;
    const int s = gd_find(a.batch, kDeltaShift, tile, c);
    if (s < 0)
        return;
    const int2 rows = gd_rows(a.batch, s);
    if (rows.y <= a.few)
        return;
    const int n = min(64, rows.y - 64 * c); // the chunk's tokens
    const int64_t first = rows.x + 64 * c;

    // this wave's 16 rows of K and Q, as fragments
    const int row = 16 * wave + r;
    gd_h8 kf[KS][PARTS], qf[KS][PARTS];
    float rq = 0.0f;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const void *src = which ? a.q : a.k;
        const int64_t at = (first + row) * (which ? a.q_step : a.k_step) + (int64_t)kh * a.k_dim + 4 * g;
        gd_f8 x[KS];
        double sum = 0.0;
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int e = 32 * i + 16 * half;
                gd_f4 v{};
                if (row < n && e + 4 * g < a.k_dim)
                    v = gd_load4(src, at + e, a.type);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[i][4 * half + j] = v[j];
                    sum += (double)v[j] * v[j];
                    most = fmaxf(most, fabsf(v[j]));
                }
            }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        // (a row's largest value may be as small as 2^-149: its power of two as an
        // exponent, not as a value)
        const int up = most > 0.0f && most < __builtin_inff() ? TOP - ilogbf(most) : 0;
        const float unit = row < n ? (float)ldexp(1.0 / sqrt(sum + (double)a.l2_eps), -up) : 0.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            gd_f8 y;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y[j] = ldexpf(x[i][j], up);
            gd_h8 hi, lo;
            gd_split(y, 1.0f, hi, lo);
            (which ? qf : kf)[i][0] = hi;
            if (PARTS > 1)
                (which ? qf : kf)[i][PARTS - 1] = lo;
        }
        if (which)
            rq = unit;
        else if (g == 0)
            rk[row] = unit;
    }
    uint8_t *const work = a.work + ((int64_t)tile * a.k_heads + kh) * 3 * FRAG;
    const bool mine = h % a.group == 0; // this head writes the operands that its group reads
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const int at = ((wave * KS + i) * PARTS + p) * 1024 + lane * 16;
            *(gd_h8 *)(lds + at) = kf[i][p];
            if (mine) {
                *(gd_h8 *)(work + at) = kf[i][p];
                *(gd_h8 *)(work + 2 * FRAG + at) = qf[i][p];
            }
        }
    // the decays' logarithms, summed in 64 bits: differences of them matter
    double sum = 0.0;
    if (lane < n)
        sum = (double)gd_log_decay(a.decay[h], a.a[(first + lane) * a.a_step + h], a.dt_bias[h]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(sum, d);
        sum += lane >= d ? up : 0.0;
    }
    if (wave == 0) {
        G[lane] = sum;
        beta[lane] = lane < n ? gd_beta(a.b[(first + lane) * a.b_step + h]) : 0.0f;
    }
    __syncthreads();

    // K^T as an operand: rows are K's columns, and tokens its columns
    if (mine)
        for (int t = wave; t < KD / 16 * 2; t += PREP_THREADS / 64) {
            const int m = t / 2, k = t % 2;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                gd_h8 v;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int token = 4 * g + i % 4, of = 2 * k + i / 4; // of tile `of`
                    v[i] = *(const _Float16 *)(lds + ((of * KS + m / 2) * PARTS + p) * 1024 + (r / 4 * 16 + token) * 16 +
                                               (4 * (m & 1) + r % 4) * 2);
                }
                *(gd_h8 *)(work + FRAG + (t * PARTS + p) * 1024 + lane * 16) = v;
            }
        }

    // this wave's rows of K K^T and Q K^T
    gd_f4 kk[4], qk[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        kk[t] = qk[t] = gd_f4{};
        if (t > wave)
            continue;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            gd_h8 b[PARTS];
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                b[p] = *(const gd_h8 *)(lds + ((t * KS + i) * PARTS + p) * 1024 + lane * 16);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int q = 0; q + p < PARTS; ++q) {
                    kk[t] = gd_mfma(kf[i][p], b[q], kk[t]);
                    qk[t] = gd_mfma(qf[i][p], b[q], qk[t]);
                }
        }
    }
    float rqs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        rqs[i] = __shfl(rq, 4 * g + i);
    __syncthreads(); // K's fragments are read: the matrices take their place
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (t > (wave | 1))
            continue; // (the tile beside an even row's diagonal one is read as zeros)
        const int j = 16 * t + r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 16 * wave + 4 * g + i;
            const float fade = j <= at ? expf((float)(G[at] - G[j])) * rk[j] : 0.0f;
            A[at * TRI + j] = j < at ? beta[at] * rk[at] * fade * kk[t][i] : 0.0f;
            P[at * TRI + j] = j <= at ? rqs[i] * fade * qk[t][i] : 0.0f;
            if (t != wave)
                T[at * TRI + j] = 0.0f;
        }
    }
    __syncthreads();

    // T = (1 + A)^-1: the diagonal 16 x 16 blocks a column a lane, by substitution
    {
        const float *D = A + 16 * wave * (TRI + 1);
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = i == r ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < i; ++m)
                x[i] = fmaf(-D[i * TRI + m], x[m], x[i]);
        }
        if (lane < 16)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                T[(16 * wave + i) * TRI + 16 * wave + r] = x[i];
    }
    // then the blocks d below the diagonal: T_ij = -T_ii sum_{j <= m < i} A_im T_mj
#pragma unroll
    for (int d = 1; d < 4; ++d) {
        __syncthreads();
        const int j = wave, i = wave + d;
        if (i >= 4)
            continue;
        gd_f4 x{};
        for (int m = j; m < i; ++m) {
            const gd_f4 left = *(const gd_f4 *)(A + (16 * i + r) * TRI + 16 * m + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(left[e], T[(16 * m + 4 * g + e) * TRI + 16 * j + r], x, 0, 0, 0);
        }
        const gd_f4 left = *(const gd_f4 *)(T + (16 * i + r) * TRI + 16 * i + 4 * g);
        gd_f4 y{};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y = __builtin_amdgcn_mfma_f32_16x16x4f32(left[e], -x[e], y, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            T[(16 * i + 4 * g + e) * TRI + 16 * j + r] = y[e];
    }
    __syncthreads();
    const int64_t unit = (int64_t)tile * a.v_heads + h;
    uint8_t *const tri = a.work + a.plan.tri + unit * 2 * kDeltaTri;
    store_tri(T, beta, tri);
    store_tri(P, nullptr, tri + kDeltaTri);
    float *const f = (float *)(a.work + a.plan.rows) + unit * kDeltaRows;
    if (wave == 0) {
        f[lane] = rk[lane] * expf((float)G[lane]);                // of K S
        f[128 + lane] = rk[lane] * expf((float)(G[63] - G[lane])); // of what is written
        if (lane == 0)
            f[192] = expf((float)G[63]);
    }
    if (g == 0)
        f[64 + row] = rq * expf((float)G[row]); // of Q S
}

// ---- down the chunks ---------------------------------------------------------------
// The largest |x| of a lane's column (in its 4 lanes)
__device__ __forceinline__ float column_most(float m)
{
    m = fmaxf(m, __shfl_xor(m, 16));
    return fmaxf(m, __shfl_xor(m, 32));
}

// Every copy but the last N has arrived, every read of LDS is done, in all waves
template <int N>
__device__ __forceinline__ void scan_sync()
{
    static_assert(N < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070); // vmcnt(N) lgkmcnt(0)
    lds_barrier();
}

// A workgroup takes NW * 16 columns of one head of one sequence.  What a chunk reads
// comes to LDS by direct copies, each operand into the place of the last chunk's as
// soon as that is read: K is on its way while V' is formed, Q, T, P and V while the
// state is, K^T meanwhile.
template <int KD, int PARTS, int NW>
__global__ void __launch_bounds__(64 * NW) k_delta_scan(DeltaArgs a)
{
    constexpr int KS = KD / 32;
    constexpr int FRAG = 4 * KS * PARTS * 1024;
    constexpr int VB = PARTS > 1 ? 4 : 2; // bytes of a value of V
    constexpr int VROW = 16 * NW * VB;    // of a row of it
    // in LDS: K | Q | K^T | T, P | V
    constexpr int Q_AT = FRAG, KT_AT = 2 * FRAG, T_AT = 3 * FRAG, P_AT = T_AT + kDeltaTri, V_AT = P_AT + kDeltaTri;
    // 1 KB copies of a wave
    constexpr int NF = FRAG / 1024 / NW, NT = 2 * kDeltaTri / 1024 / NW, NV = VB;
    static_assert(NF * NW * 1024 == FRAG && NT * NW * 1024 == 2 * kDeltaTri, "copies are shared evenly");
    __shared__ __attribute__((aligned(16))) uint8_t lds[V_AT + 64 * VROW];
    __shared__ __attribute__((aligned(16))) float rows[2][kDeltaRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    // the workgroups of the heads that read one K lie on one XCD (its L2)
    const int blocks = (a.v_dim + 16 * NW - 1) / (16 * NW), each = a.group * blocks;
    const int j = blockIdx.x / 8, u = j / each * 8 + blockIdx.x % 8;
    if (u >= a.k_heads * a.batch.sequences)
        return;
    const int s = u / a.k_heads, kh = u % a.k_heads, h = kh * a.group + j % each / blocks;
    const GdSeq seq = gd_seq(a.batch, a.pool, s, h == 0 && j % blocks == 0 ? a.flags : nullptr);
    if (seq.slot < 0 || seq.n <= a.few)
        return;
    const int col0 = j % blocks * NW * 16, col = col0 + wave * 16 + r;
    const bool live = col < a.v_dim;
    float *const state = a.state + seq.slot * a.slot_step + (int64_t)h * a.k_dim * a.v_dim + col;

    const int chunks = (seq.n + 63) / 64, tile0 = gd_base(a.batch, kDeltaShift, s);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const uint32_t rows0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float *)&rows[0][0];
    auto kq = [&](int c) { return a.work + ((int64_t)(tile0 + c) * a.k_heads + kh) * 3 * FRAG; };
    auto unit = [&](int c) { return (int64_t)(tile0 + c) * a.v_heads + h; };
    auto copy = [&](const uint8_t *from, int to, int n) { // n KB a wave
        for (int i = 0; i < n; ++i)
            lds_copy16_at(from, (uint32_t)((wave * n + i) * 1024 + lane * 16), lds0 + to + (wave * n + i) * 1024);
    };
    // K and the rows' factors (each wave the same 1 KB, so that all wait alike)
    auto copy_k = [&](int c) {
        copy(kq(c), 0, NF);
        lds_copy16_at(a.work + a.plan.rows + unit(c) * kDeltaRows * 4, lane * 16, rows0 + (c & 1) * kDeltaRows * 4);
    };
    auto copy_kt = [&](int c) { copy(kq(c) + FRAG, KT_AT, NF); };
    auto copy_rest = [&](int c) {
        copy(kq(c) + 2 * FRAG, Q_AT, NF);
        copy(a.work + a.plan.tri + unit(c) * 2 * kDeltaTri, T_AT, NT);
        const int n = min(64, seq.n - 64 * c);
        // (rows behind the last token and columns behind the last one are read as
        // others and not used)
        for (int i = 0; i < NV; ++i) {
            const int at = ((wave * NV + i) * 64 + lane) * 16, e = at % VROW / VB;
            const int64_t row = seq.start + 64 * c + min(at / VROW, n - 1);
            lds_copy16((const uint8_t *)a.v + (row * a.v_step + (int64_t)h * a.v_dim + (col0 + e < a.v_dim ? col0 + e : 0)) * VB,
                       lds0 + V_AT + (wave * NV + i) * 1024);
        }
    };
    copy_k(0);
    copy_rest(0);
    gd_f4 S[KD / 16];
#pragma unroll
    for (int m = 0; m < KD / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 16 * m + 4 * g + i;
            S[m][i] = live && !seq.begins && at < a.k_dim ? state[(int64_t)at * a.v_dim] : 0.0f;
        }
    for (int c = 0; c < chunks; ++c) {
        const int n = min(64, seq.n - 64 * c), next = min(c + 1, chunks - 1);
        const int64_t first = seq.start + 64 * c;
        const float *const fs = rows[c & 1];
        // S as an operand
        float most = 0.0f, to, back;
#pragma unroll
        for (int m = 0; m < KD / 16; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                most = fmaxf(most, fabsf(S[m][i]));
        gd_power(column_most(most), to, back);
        gd_h8 shi[KS], slo[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k)
            gd_split(__builtin_shufflevector(S[2 * k], S[2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7), to, shi[k], slo[k]);
        scan_sync<NF + NT + NV>(); // K is here; K^T is read
        copy_kt(c);
        gd_f4 ks[4], O[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            ks[m] = gd_f4{};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint8_t *at = lds + (m * KS + k) * PARTS * 1024 + lane * 16;
                const gd_h8 kf = *(const gd_h8 *)at;
                ks[m] = gd_mfma(kf, shi[k], ks[m]);
                ks[m] = gd_mfma(kf, slo[k], ks[m]);
                if (PARTS > 1)
                    ks[m] = gd_mfma(*(const gd_h8 *)(at + 1024), shi[k], ks[m]);
            }
        }
        scan_sync<NF>(); // Q, T, P and V are here; K is read
        copy_k(next);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            O[m] = gd_f4{};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint8_t *at = lds + Q_AT + (m * KS + k) * PARTS * 1024 + lane * 16;
                const gd_h8 qf = *(const gd_h8 *)at;
                O[m] = gd_mfma(qf, shi[k], O[m]);
                O[m] = gd_mfma(qf, slo[k], O[m]);
                if (PARTS > 1)
                    O[m] = gd_mfma(*(const gd_h8 *)(at + 1024), shi[k], O[m]);
            }
        }
        // X = V - e^G K S as an operand, V' = T X
        gd_f4 x[4];
        most = 0.0f;
        const float sback = back;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const gd_f4 fk = *(const gd_f4 *)(fs + 16 * m + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 16 * m + 4 * g + i;
                const uint8_t *from = lds + V_AT + at * VROW + (wave * 16 + r) * VB;
                float v = a.type == kF32 ? *(const float *)from
                        : a.type == kF16 ? (float)*(const _Float16 *)from : (float)*(const __bf16 *)from;
                if (!live || at >= n)
                    v = 0.0f;
                x[m][i] = v - fk[i] * (ks[m][i] * sback);
                most = fmaxf(most, fabsf(x[m][i]));
            }
        }
        gd_power(column_most(most), to, back);
        gd_h8 hi[2], lo[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
            gd_split(__builtin_shufflevector(x[2 * k], x[2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7), to, hi[k], lo[k]);
        back *= 1.0f / (1 << TOP);
        gd_f4 w[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            w[m] = gd_f4{};
#pragma unroll
            for (int k = 0; k <= m / 2; ++k) {
                const uint8_t *at = lds + T_AT + (m < 2 ? m : 2 * m - 2 + k) * 2048 + lane * 16;
                const gd_h8 th = *(const gd_h8 *)at, tl = *(const gd_h8 *)(at + 1024);
                w[m] = gd_mfma(th, hi[k], w[m]);
                w[m] = gd_mfma(th, lo[k], w[m]);
                w[m] = gd_mfma(tl, hi[k], w[m]);
            }
            w[m] = w[m] * back;
        }
        // O = scale (e^G Q S + P V')
        most = 0.0f;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                most = fmaxf(most, fabsf(w[m][i]));
        gd_power(column_most(most), to, back);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            gd_split(__builtin_shufflevector(w[2 * k], w[2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7), to, hi[k], lo[k]);
        back *= 1.0f / (1 << TOP);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const gd_f4 fq = *(const gd_f4 *)(fs + 64 + 16 * m + 4 * g);
            gd_f4 y{};
#pragma unroll
            for (int k = 0; k <= m / 2; ++k) {
                const uint8_t *at = lds + P_AT + (m < 2 ? m : 2 * m - 2 + k) * 2048 + lane * 16;
                const gd_h8 th = *(const gd_h8 *)at, tl = *(const gd_h8 *)(at + 1024);
                y = gd_mfma(th, hi[k], y);
                y = gd_mfma(th, lo[k], y);
                y = gd_mfma(tl, hi[k], y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 16 * m + 4 * g + i;
                const float o = a.scale * fmaf(y[i], back, fq[i] * (O[m][i] * sback));
                const int64_t where = ((first + at) * a.v_heads + h) * a.v_dim + col;
                if (live && at < n) {
                    if (a.raw)
                        a.raw[where] = o;
                    else if (a.out_type == kF16)
                        ((_Float16 *)a.out)[where] = (_Float16)o;
                    else
                        ((__bf16 *)a.out)[where] = (__bf16)o;
                }
            }
        }
        // S <- e^G_64 S + K^T (e^(G_64 - G) V')
        most = 0.0f;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            w[m] = w[m] * *(const gd_f4 *)(fs + 128 + 16 * m + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                most = fmaxf(most, fabsf(w[m][i]));
        }
        gd_power(column_most(most), to, back);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            gd_split(__builtin_shufflevector(w[2 * k], w[2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7), to, hi[k], lo[k]);
        const float keep = fs[192];
        scan_sync<NF + 1>(); // K^T is here; Q, T, P and V are read
        copy_rest(next);
#pragma unroll
        for (int m = 0; m < KD / 16; ++m) {
            gd_f4 y{};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint8_t *at = lds + KT_AT + (2 * m + k) * PARTS * 1024 + lane * 16;
                const gd_h8 kt = *(const gd_h8 *)at;
                y = gd_mfma(kt, hi[k], y);
                y = gd_mfma(kt, lo[k], y);
                if (PARTS > 1)
                    y = gd_mfma(*(const gd_h8 *)(at + 1024), hi[k], y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                S[m][i] = fmaf(keep, S[m][i], y[i] * back);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070); // no copy is in flight when the workgroup ends
#pragma unroll
    for (int m = 0; m < KD / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 16 * m + 4 * g + i;
            if (live && at < a.k_dim)
                state[(int64_t)at * a.v_dim] = S[m][i];
        }
}

// ---- the output norm ---------------------------------------------------------------
constexpr int NORM_THREADS = 256;

// raw -> out: 32 lanes a row of a head (4 columns each), 64 rows of a sequence.
__global__ void __launch_bounds__(NORM_THREADS) k_delta_norm(DeltaArgs a)
{
    int c = 0;
    const int s = gd_find(a.batch, kDeltaShift, (int)(blockIdx.x / a.v_heads), c);
    if (s < 0)
        return;
    const GdSeq seq = gd_seq(a.batch, a.pool, s, nullptr);
    if (seq.slot < 0 || seq.n <= a.few)
        return;
    const int h = blockIdx.x % a.v_heads, e = 4 * (threadIdx.x & 31);
    const bool live = e < a.v_dim;
    for (int t = 64 * c + (threadIdx.x >> 5); t < min(64 * c + 64, seq.n); t += NORM_THREADS / 32) {
        const int64_t row = seq.start + t, at = (row * a.v_heads + h) * a.v_dim + e;
        gd_f4 o = live ? *(const gd_f4 *)(a.raw + at) : gd_f4{};
        if (a.norm_w) {
            float sum = (o.x * o.x + o.y * o.y) + (o.z * o.z + o.w * o.w);
            sum = gd_add_dpp<0xb1>(sum);
            sum = gd_add_dpp<0x4e>(sum);
            sum = gd_add_dpp<0x141>(sum);
            sum = gd_add_dpp<0x140>(sum);
            sum = gd_add16(sum);
            if (live)
                o = o * (1.0f / sqrtf(sum / (float)a.v_dim + a.norm_eps)) * *(const gd_f4 *)(a.norm_w + e);
        }
        if (!live)
            continue;
        if (a.gate) {
            const gd_f4 z = *(const gd_f4 *)(a.gate + row * a.gate_step + (int64_t)h * a.v_dim + e);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] *= gd_silu(z[i]);
        }
        gd_store4(a.out, at, a.out_type, o);
    }
}

template <int KD, int PARTS>
void launch(const DeltaArgs &a, hipStream_t s)
{
    constexpr int NW = 4;
    const unsigned units = (unsigned)(a.plan.tiles * a.v_heads);
    hipLaunchKernelGGL((k_delta_prep<KD, PARTS>), dim3(units), dim3(PREP_THREADS), 0, s, a);
    const unsigned blocks = (unsigned)((a.v_dim + 16 * NW - 1) / (16 * NW)) * (unsigned)a.group;
    const unsigned heads = ((unsigned)(a.k_heads * a.batch.sequences) + 7) / 8 * 8;
    hipLaunchKernelGGL((k_delta_scan<KD, PARTS, NW>), dim3(heads * blocks), dim3(64 * NW), 0, s, a);
    if (a.norm_w || a.gate)
        hipLaunchKernelGGL(k_delta_norm, dim3(units), dim3(NORM_THREADS), 0, s, a);
}

} // namespace

hipError_t launch_delta_chunks(const DeltaArgs &a, hipStream_t s)
{
    if (a.type == kF32)
        a.k_dim <= 64 ? launch<64, 2>(a, s) : launch<128, 2>(a, s);
    else
        a.k_dim <= 64 ? launch<64, 1>(a, s) : launch<128, 1>(a, s);
    return hipGetLastError();
}

} // namespace ihip
