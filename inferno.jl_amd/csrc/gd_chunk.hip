// gd_chunk.hip -- the gated delta rule over sequences with many new tokens, 64 of
// them at a time on the matrix cores.  With G_i the sum of the logarithms of the
// decays up to token i of the chunk, S the state before it, and k, q of unit length,
//
//   A_ij = beta_i k_i.k_j e^(G_i - G_j), j < i;      T = (1 + A)^-1 diag(beta)
//   X = V - e^G K S                                  (what the state does not bring back)
//   O = scale (e^G Q S + P X),   P = [q_i.k_j e^(G_i - G_j), j <= i] T
//   S <- e^G_64 S + M X,         M = (e^(G_64 - G) K)^T T
//
// P and M do not depend on S: k_delta_prep forms them, and K and Q as matrix operands,
// for all chunks at once.  k_delta_scan then walks down a sequence's chunks; the columns
// of S do not touch each other.
//
// A chunk's tokens may be of any sizes beside each other: a quiet token before a loud one, a
// loud one that is forgotten before a quiet one, a head that hardly writes.  So X, T, P
// and M are operands of three bf16 parts, which have 24 bits and the exponents of fp32; of
// the products of their parts those below 2^-24 are not formed.  (In two fp16 parts with a
// power of two for a chunk, rows 10^7 below the largest lost their last bits, and 10^9 all.)
// A product with S sums over all of a row of K or Q and a column of S, so what is small
// beside the row's or the column's largest value counts as little there as in fp32: those
// operands are fp16 times a power of two, the largest in 2^13 .. 2^14.  Values of F16 and
// BF16 inputs fit one such part exactly down to 2^-27 of their row's largest, and to 2^-38 of
// that below; fp32 ones and S are held in two, which leave 2^-22 of a value, and products
// of the two lower parts (2^-22) are not formed.  Sums are fp32.  Rows' factors (unit
// length, e^G) are applied to the products, in fp32, so that K and Q are shared by the heads
// that read them.
#include "gd_launch.h"

namespace ihip {

namespace {

typedef _Float16 gd_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 gd_b8 __attribute__((ext_vector_type(8)));
typedef float gd_f8 __attribute__((ext_vector_type(8)));

constexpr int TOP = 13; // fp16 operands' largest values have this binary exponent

// 2^(TOP - exponent of x), and what a product of such a value with a row of K or Q takes back
// of it, and of the row's own 2^TOP, before anything else, so that it does not pass the range;
// x >= 0.  (Below 2^-100 of nothing; an infinity or NaN is left one.)
__device__ __forceinline__ void gd_power(float x, float &to, float &back)
{
    const int e = max((int)(__float_as_uint(x) >> 23), 127 - 100);
    to = __uint_as_float((uint32_t)(254 + TOP - e) << 23);
    back = __uint_as_float((uint32_t)(e - 2 * TOP) << 23);
}

// x * by as one fp16 part, and the rest of it, times 2^11, as the next: where the first is one of
// fp16's subnormal values, the rest still has bits below it.
constexpr float REST = 2048.0f;
template <typename F, typename H>
__device__ __forceinline__ void gd_split(F x, float by, H &hi, H &lo)
{
    x = x * by;
    hi = __builtin_convertvector(x, H);
    lo = __builtin_convertvector((x - __builtin_convertvector(hi, F)) * REST, H);
}

// x as three bf16 parts, each the nearest of what the ones before leave.  (In pairs, as the
// conversion takes them: 5.5 operations a value.)
template <typename F, typename B>
__device__ __forceinline__ void gd_split3(F x, B (&part)[3])
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    constexpr int PAIRS = sizeof(F) / 8;
    typedef uint32_t Pairs __attribute__((ext_vector_type(PAIRS)));
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        Pairs u;
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            u[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x[2 * j], x[2 * j + 1]}, b2));
            if (i < 2) {
                x[2 * j] -= __uint_as_float(u[j] << 16);
                x[2 * j + 1] -= __uint_as_float(u[j] & 0xffff0000u);
            }
        }
        part[i] = __builtin_bit_cast(B, u);
    }
}

// 2^x, x <= 0 (nothing below 2^-126); without a branch
__device__ __forceinline__ float gd_exp2(double x)
{
    return __builtin_amdgcn_exp2f((float)x);
}

__device__ __forceinline__ gd_f4 gd_mfma(gd_h8 a, gd_h8 b, gd_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ gd_f4 gd_mfma(gd_b8 a, gd_b8 b, gd_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// x + rest += the product of operands in 3 and N bf16 parts: x of the first ones, rest of the
// others whose sizes are over 2^-24 of that
template <int N>
__device__ __forceinline__ void gd_dot(const gd_b8 (&a)[3], const gd_b8 (&b)[N], gd_f4 &x, gd_f4 &rest)
{
    x = gd_mfma(a[0], b[0], x);
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (i + j == 1 || i + j == 2)
                rest = gd_mfma(a[i], b[j], rest);
}

// Fragments.  A 16-row tile of an operand is stored as the matrix cores take it: for
// each step of 32 columns, lane (g, r) = (lane / 16, lane % 16) holds of row r the
// columns 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3, 16 bytes a lane.  These are the
// rows that a lane holds of two tiles of a product's result, so that results (S, X)
// are the next product's operands without leaving their registers.  P and M, which come out
// of fp32 sums, lie as two such planes of 4 fp32 values a lane.

// ---- chunks' operands ------------------------------------------------------------
constexpr int PREP_THREADS = 256;
constexpr float LEAST = 0x1p-90f; // of a chunk's fades in the bound on the next S
constexpr int TRI = 68; // floats from a row of a 64 x 64 matrix to the next, in LDS

// A workgroup takes a chunk of a head of v; a wave 16 of its rows.  k's and q's products
// are on the fp16 matrix cores, P and M on the bf16 ones, the inverse in fp32: 16 x 16 blocks on
// the diagonal by substitution, the ones below from those on the fp32 matrix cores.  Heads that share
// K and Q form them again each (their rows are in L2), and one writes them.  8192 tokens of 32
// heads of 128 on 16, bf16: 105 us for 67 MB in and 253 out (P and M 185 of them), 3.0 TB/s;
// 163 with two workgroups a CU instead of three and loads that wait for each other.
template <int TYPE, int KD>
__global__ void __launch_bounds__(PREP_THREADS) k_delta_prep(DeltaArgs a)
{
    constexpr int PARTS = TYPE == kF32 ? 2 : 1;
    constexpr int KS = KD / 32;               // steps of a row of K
    constexpr int FRAG = 4 * KS * PARTS * 1024; // bytes of K or Q
    constexpr int MD = KD / 64;               // 16-row tiles of M that a wave forms
    // bf16 parts of a value of K
    constexpr int BF = TYPE == kF32 ? 3 : TYPE == kF16 ? 2 : 1;
    // K; then A (P in its place) and its inverse T; then T as two operands
    constexpr int MAT = 64 * TRI * 4, TT = 6 * 3 * 1024;
    static_assert(MAT <= TT && FRAG <= 2 * TT, "");
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * TT];
    __shared__ double G[64];
    __shared__ float beta[64], rk[64], fu[64];
    float *const A = (float *)lds, *const P = A, *const T = (float *)(lds + TT);
    uint8_t(*const tt)[6][3][1024] = (uint8_t(*)[6][3][1024])lds;
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
    // (behind the last token and the last column: others' values, not used)
    typename GdType<TYPE>::T4 raw[2][2 * KS];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int64_t at = (first + min(row, n - 1)) * (which ? a.q_step : a.k_step) + (int64_t)kh * a.k_dim;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
            raw[which][i] = gd_raw4<TYPE>(which ? a.q : a.k, at + (16 * i + 4 * g < a.k_dim ? 16 * i + 4 * g : 0));
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        gd_f8 x[KS];
        double sum = 0.0;
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
            const gd_f4 v = row < n && 16 * i + 4 * g < a.k_dim ? gd_wide(raw[which][i]) : gd_f4{};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i / 2][4 * (i & 1) + j] = v[j];
                sum += (double)v[j] * v[j];
                most = fmaxf(most, fabsf(v[j]));
            }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        // (a row's largest value may be as small as 2^-149: its power of two as an
        // exponent, not as a value)
        const int up = most > 0.0f && most < __builtin_inff() ? TOP - ilogbf(most) : 0;
        // (a row of zeros stays one)
        const float unit = row < n && most > 0.0f ? (float)ldexp(1.0 / sqrt(sum + (double)a.l2_eps), -up) : 0.0f;
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
    uint8_t *const work = a.work + ((int64_t)tile * a.k_heads + kh) * 2 * FRAG;
    const bool mine = h % a.group == 0; // this head writes the operands that its group reads
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const int at = ((wave * KS + i) * PARTS + p) * 1024 + lane * 16;
            *(gd_h8 *)(lds + at) = kf[i][p];
            if (mine) {
                *(gd_h8 *)(work + at) = kf[i][p];
                *(gd_h8 *)(work + FRAG + at) = qf[i][p];
            }
        }
    // the decays' logarithms, of base 2, summed in 64 bits: differences of them matter
    double sum = 0.0;
    if (lane < n)
        sum = (double)gd_log_decay(a.decay[h], a.a[(first + lane) * a.a_step + h], a.dt_bias[h]) * 1.4426950408889634;
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

    if (wave == 0)
        fu[lane] = rk[lane] * gd_exp2(G[63] - G[lane]);
    // this wave's columns of K, with the tokens in steps
    gd_b8 kt[MD][2][BF];
#pragma unroll
    for (int m = 0; m < MD; ++m)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            gd_f8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int token = 4 * g + i % 4, of = 2 * k + i / 4, md = MD * wave + m; // of tile `of`
                const uint8_t *const at =
                    lds + (of * KS + md / 2) * PARTS * 1024 + (r / 4 * 16 + token) * 16 + (4 * (md & 1) + r % 4) * 2;
                x[i] = (float)*(const _Float16 *)at;
                if (PARTS > 1)
                    x[i] = fmaf((float)*(const _Float16 *)(at + 1024), 1.0f / REST, x[i]);
            }
            if constexpr (BF == 3) {
                gd_split3(x, kt[m][k]);
            } else {
                kt[m][k][0] = __builtin_convertvector(x, gd_b8);
                if constexpr (BF == 2)
                    kt[m][k][1] = __builtin_convertvector(x - __builtin_convertvector(kt[m][k][0], gd_f8), gd_b8);
            }
        }

    // this wave's rows of K K^T and Q K^T
    gd_f4 kk[4], qk[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        kk[t] = qk[t] = gd_f4{};
        gd_f4 krest{}, qrest{};
        if (t > wave)
            continue;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            gd_h8 b[PARTS];
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                b[p] = *(const gd_h8 *)(lds + ((t * KS + i) * PARTS + p) * 1024 + lane * 16);
            kk[t] = gd_mfma(kf[i][0], b[0], kk[t]);
            qk[t] = gd_mfma(qf[i][0], b[0], qk[t]);
            if (PARTS > 1) {
                krest = gd_mfma(kf[i][0], b[PARTS - 1], krest);
                krest = gd_mfma(kf[i][PARTS - 1], b[0], krest);
                qrest = gd_mfma(qf[i][0], b[PARTS - 1], qrest);
                qrest = gd_mfma(qf[i][PARTS - 1], b[0], qrest);
            }
        }
        if (PARTS > 1) {
            kk[t] += krest * (1.0f / REST);
            qk[t] += qrest * (1.0f / REST);
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
            const float fade = gd_exp2(j <= at ? G[at] - G[j] : 0.0) * rk[j];
            A[at * TRI + j] = j < at ? beta[at] * rk[at] * fade * kk[t][i] : 0.0f;
            qk[t][i] = j <= at ? rqs[i] * fade * qk[t][i] : 0.0f;
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
    __syncthreads(); // A is read, T written
    // P by rows, as an operand of this wave alone
    gd_b8 pf[2][3];
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (t <= (wave | 1))
#pragma unroll
            for (int i = 0; i < 4; ++i)
                P[(16 * wave + 4 * g + i) * TRI + 16 * t + r] = qk[t][i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float *from = P + row * TRI + 32 * k + 4 * g;
        gd_f8 x{};
        if (k <= wave / 2)
            x = __builtin_shufflevector(*(const gd_f4 *)from, *(const gd_f4 *)(from + 16), 0, 1, 2, 3, 4, 5, 6, 7);
        gd_split3(x, pf[k]);
    }
    // T^T as an operand (16 x 32 tiles on and over its diagonal), its columns once as
    // they are and once times the factors of what is written to the state
    gd_b8 to[2][2][3];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int t = wave + 4 * u;
        if (t >= 6)
            continue;
        const int jt = t < 4 ? t / 2 : t - 2, k = t < 4 ? t % 2 : 1, j = 16 * jt + r;
        gd_f8 x, y;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = 32 * k + 4 * g + i % 4 + 16 * (i / 4);
            x[i] = T[at * TRI + j] * beta[j];
            y[i] = x[i] * fu[at];
        }
        gd_split3(x, to[0][u]);
        gd_split3(y, to[1][u]);
    }
    __syncthreads(); // P and T are read
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const int t = wave + 4 * u;
            if (t >= 6)
                continue;
            *(gd_b8 *)(tt[0][t][p] + lane * 16) = to[0][u][p];
            *(gd_b8 *)(tt[1][t][p] + lane * 16) = to[1][u][p];
        }
    __syncthreads();
    // P and M, transposed (T^T times the other matrix's transpose), so that a lane holds
    // the columns of a row that it stores as a fragment
    const int64_t unit = (int64_t)tile * a.v_heads + h;
    uint8_t *const tri = a.work + a.plan.tri + unit * (kDeltaTri + KD * 256) + lane * 16;
    auto store = [&](int n, gd_f4 left, gd_f4 right) { // the n-th tile of P and M
        *(gd_f4 *)(tri + n * 2048) = left;
        *(gd_f4 *)(tri + n * 2048 + 1024) = right;
    };
    auto load = [&](int which, int jt, int k, gd_b8(&part)[3]) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
            part[p] = *(const gd_b8 *)(tt[which][jt < 2 ? 2 * jt + k : 2 + jt][p] + lane * 16);
    };
    gd_f4 out[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
        gd_f4 x{}, y{};
#pragma unroll
        for (int k = jt / 2; k < 2; ++k) {
            if (jt > wave || k > wave / 2)
                continue;
            gd_b8 t[3];
            load(0, jt, k, t);
            gd_dot(t, pf[k], x, y);
        }
        out[jt] = x + y;
    }
    const int t0 = wave < 2 ? wave : 2 * wave - 2; // this wave's first tile of a triangle
    store(t0, out[0], out[1]);
    if (wave >= 2)
        store(t0 + 1, out[2], out[3]);
#pragma unroll
    for (int m = 0; m < MD; ++m) {
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
            gd_f4 x{}, y{};
#pragma unroll
            for (int k = jt / 2; k < 2; ++k) {
                gd_b8 t[3];
                load(1, jt, k, t);
                gd_dot(t, kt[m][k], x, y);
            }
            out[jt] = x + y;
        }
        const int md = MD * wave + m;
        store(6 + 2 * md, out[0], out[1]);
        store(6 + 2 * md + 1, out[2], out[3]);
    }
    constexpr float UP = 1 << TOP; // (the rows' own, which the scan takes back first)
    float *const f = (float *)(a.work + a.plan.rows) + unit * kDeltaRows;
    if (wave == 0) {
        f[lane] = rk[lane] * UP * gd_exp2(G[lane]); // of K S
        f[128 + lane] = fmaxf(beta[lane] * gd_exp2(G[63] - G[lane]), LEAST); // of what a token adds to S
        if (lane == 0)
            f[192] = gd_exp2(G[63]);
    }
    if (g == 0)
        f[64 + row] = rq * UP * gd_exp2(G[row]); // of Q S
}

// ---- down the chunks ---------------------------------------------------------------
constexpr int SCAN_WAVES = 4;

// What a wave reads of a chunk: its 16 rows of K, Q and P, its 16 MT rows of M, the factors
// of its 16 tokens and their values in its columns.
template <int KS, int MT, int PARTS>
struct ScanOps {
    gd_h8 k[KS][PARTS], q[KS][PARTS];
    gd_f4 m[MT][2][2], p[2][2]; // in fp32
    gd_f4 fk, fq, fs;
    uint32_t v[4]; // as they lie in memory
    float keep;
};

// All waves are here, and what they wrote to LDS is
__device__ __forceinline__ void scan_sync()
{
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0); loads stay on their way
    lds_barrier();
}

// A workgroup takes 16 columns of one head of one sequence, each of its waves the
// tokens 16 w .. 16 w + 15 of a chunk and KD / 4 rows of S.  A wave so reads only its own
// part of the operands, from memory into registers, two chunks ahead, and the waves exchange
// S and X as fragments in LDS, with two barriers a chunk.  Bound by that chain, as a chunk follows the other, and by the
// operands' way: 8192 tokens of 32 heads of 128 x 128 take 286 us, 2.2 a chunk of 76 KB on every CU
// (35 KB a microsecond).  (In a form with half the products, which took as long, products, exchanges and
// barriers alone were 1.2 a chunk, and the operands added 0.6 from L2 and 0.4 from further away; one
// chunk ahead was 322, three 274; 32 columns a workgroup, which halves the bytes and the CUs in
// use, 385.)  Heads up to 64 wide have half the rows of S a wave, and registers for two workgroups a
// CU: 24 heads of 3 sequences of 22 to 135 tokens and 2 shorter ones 9.9 us (two waves with 32 rows
// each: 16.3).
//
// A column of S has a power of two for every chunk, from a bound that no token passes: k and q
// have unit length at most, a token adds no more than beta |v| to a column's length, and
// all of it fades, so that S after a chunk lies below 12 e^G_64 max |S| + 66 max(e^(G_64 - G) beta
// |v|) (sqrt(128) < 12).  Values down to 2^-27 of that keep 22 bits, and smaller ones
// 2^-49 of it.  No fade counts as less than 2^-90 in it, so X is below 2^90 of it: where it is
// under 2^-60, X is lifted by 2^24, as the third parts of values under 2^-109 would have no
// room in bf16's exponents.
template <int TYPE, int KD>
__global__ void __launch_bounds__(64 * SCAN_WAVES) k_delta_scan(DeltaArgs a)
{
    constexpr int PARTS = TYPE == kF32 ? 2 : 1;
    constexpr int KS = KD / 32, MT = KD / 64; // steps of a row of K; 16-row tiles of S that a wave has
    constexpr int FRAG = 4 * KS * PARTS * 1024;
    constexpr int VB = PARTS > 1 ? 4 : 2; // bytes of a value of V
    using Ops = ScanOps<KS, MT, PARTS>;
    __shared__ __attribute__((aligned(16))) uint8_t sf[KS][2][1024], xf[2][3][1024];
    __shared__ float bounds[SCAN_WAVES][16];
    __shared__ __attribute__((aligned(16))) float turn[SCAN_WAVES][16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    if (a.flags && blockIdx.x == 0 && !a.plan.steps)
        gd_report(a.batch, a.flags);
    // the workgroups of the heads that read one K lie on one XCD (its L2)
    const int blocks = a.v_dim / 16, each = a.group * blocks;
    const int j = blockIdx.x / 8, u = j / each * 8 + blockIdx.x % 8;
    if (u >= a.k_heads * a.batch.sequences)
        return;
    const int s = u / a.k_heads, kh = u % a.k_heads, h = kh * a.group + j % each / blocks;
    GdSeq seq = gd_seq(a.batch, a.pool, s, h == 0 && j % blocks == 0 ? a.flags : nullptr);
    if (seq.slot < 0 || seq.n <= a.few)
        return;
    // (one value a workgroup, and so one address a chunk for what all lanes read beside each other)
    seq.start = __builtin_amdgcn_readfirstlane(seq.start), seq.n = __builtin_amdgcn_readfirstlane(seq.n);
    const int col0 = j % blocks * 16;
    float *const state = a.state + seq.slot * a.slot_step + (int64_t)h * a.k_dim * a.v_dim + col0 + r;
    const int chunks = (seq.n + 63) / 64, tile0 = (seq.start >> kDeltaShift) + s;
    int64_t vat[4]; // of this lane's values of V in a whole chunk
#pragma unroll
    for (int i = 0; i < 4; ++i)
        vat[i] = ((16 * wave + 4 * g + i) * a.v_step + r) * VB;
    const int64_t oat = (int64_t)(16 * wave + lane / 4) * a.v_heads * a.v_dim + 4 * (lane % 4);

    // A chunk's operands: those of the chunk after the next follow one by one, as soon as
    // their registers are free.  Loads that follow each other hold the wave up; between the
    // products they do not (8192 tokens 359 us of scan with the loads of K and Q, and of M
    // and P, together, 286 so).  (Behind the last chunk: its operands again.)
    const uint32_t mine = lane * 16;
    auto at_kq = [&](int c) { return a.work + ((int64_t)(tile0 + min(c, chunks - 1)) * a.k_heads + kh) * 2 * FRAG; };
    auto at_unit = [&](int c) { return (int64_t)(tile0 + min(c, chunks - 1)) * a.v_heads + h; };
    auto load_key = [&](Ops &o, int c, int k) {
        const uint8_t *const kq = at_kq(c) + (wave * KS + k) * PARTS * 1024;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            o.k[k][p] = *(const gd_h8 *)(kq + p * 1024 + mine);
            o.q[k][p] = *(const gd_h8 *)(kq + FRAG + p * 1024 + mine);
        }
    };
    auto load_rows = [&](Ops &o, int c) {
        const float *const f = (const float *)(a.work + a.plan.rows) + at_unit(c) * kDeltaRows;
        const uint32_t at = 16 * wave + 4 * g;
        o.fk = *(const gd_f4 *)(f + at);
        o.fq = *(const gd_f4 *)(f + 64 + at);
        o.fs = *(const gd_f4 *)(f + 128 + at);
        o.keep = f[192];
        // (rows behind the last token: others', not used)
        const int at0 = 64 * min(c, chunks - 1);
        const uint8_t *const v = (const uint8_t *)a.v + ((seq.start + at0) * a.v_step + (int64_t)h * a.v_dim + col0) * VB;
        const int last = seq.n - 1 - at0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 16 * wave + 4 * g + i;
            const uint8_t *const at = v + (last >= 63 ? vat[i] : (min(row, last) * a.v_step + r) * VB);
            o.v[i] = PARTS > 1 ? *(const uint32_t *)at : *(const uint16_t *)at;
        }
    };
    auto at_tri = [&](int c) { return a.work + a.plan.tri + at_unit(c) * (kDeltaTri + KD * 256); };
    auto load_tile = [&](gd_f4(&to)[2], int c, int n) { // the n-th of P and M
        const uint8_t *const from = at_tri(c) + n * 2048;
        to[0] = *(const gd_f4 *)(from + mine);
        to[1] = *(const gd_f4 *)(from + 1024 + mine);
    };
    const int p0 = wave < 2 ? wave : 2 * wave - 2; // this wave's first tile of P
    auto load_p = [&](Ops &o, int c) {
        load_tile(o.p[0], c, p0);
        if (wave >= 2)
            load_tile(o.p[1], c, p0 + 1);
    };
    auto load_m = [&](Ops &o, int c, int m, int k) { load_tile(o.m[m][k], c, 6 + 2 * (MT * wave + m) + k); };
    auto load_all = [&](Ops &o, int c) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
            load_key(o, c, k);
        load_rows(o, c);
        load_p(o, c);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                load_m(o, c, m, k);
    };
    auto wide = [](const gd_f4 (&half)[2]) { return __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7); };
    auto most4 = [](gd_f4 x) { return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))); };

    gd_f4 S[MT];
    float to_s, back_s;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 16 * (MT * wave + m) + 4 * g + i;
            S[m][i] = !seq.begins && at < a.k_dim ? state[(int64_t)at * a.v_dim] : 0.0f;
        }
    auto most_s = [&]() { return MT > 1 ? fmaxf(most4(S[0]), most4(S[MT - 1])) : most4(S[0]); };
    const float most = gd_max32(gd_max16(most_s()));
    if (g == 0)
        bounds[wave][r] = most;
    scan_sync();
    auto widest = [&]() {
        return fmaxf(fmaxf(bounds[0][r], bounds[1][r]), fmaxf(bounds[2][r], bounds[3][r]));
    };
    gd_power(widest(), to_s, back_s);
    scan_sync();
    // S as a fragment, or half of one
    auto put_s = [&]() {
        if constexpr (MT > 1) {
            gd_h8 hi, lo;
            gd_split(wide(S), to_s, hi, lo);
            *(gd_h8 *)(sf[wave][0] + lane * 16) = hi;
            *(gd_h8 *)(sf[wave][1] + lane * 16) = lo;
        } else {
            gd_h4 hi, lo;
            gd_split(S[0], to_s, hi, lo);
            *(gd_h4 *)(sf[wave / 2][0] + lane * 16 + 8 * (wave & 1)) = hi;
            *(gd_h4 *)(sf[wave / 2][1] + lane * 16 + 8 * (wave & 1)) = lo;
        }
    };
    put_s();

    auto chunk = [&](Ops &o, int c) {
        const int n = min(64, seq.n - 64 * c);
        gd_f4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = TYPE == kF32 ? __uint_as_float(o.v[i]) : TYPE == kF16 ? h2f(o.v[i]) : __uint_as_float(o.v[i] << 16);
            v[i] = 16 * wave + 4 * g + i < n ? x : 0.0f;
        }
        const float most = 12.0f * fmaxf(o.keep, LEAST) * most_s() + 66.0f * most4(v * o.fs);
        const float all = gd_max32(gd_max16(most));
        if (g == 0)
            bounds[wave][r] = all;
        scan_sync();
        // K S and Q S; X = V - e^G K S
        gd_f4 qs;
        const float next = widest(), keep = o.keep;
        const float lift = next < 0x1p-60f ? 0x1p24f : 1.0f, sink = next < 0x1p-60f ? 0x1p-24f : 1.0f;
        {
            gd_f4 x{}, y{}, z{}, w{};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const gd_h8 hi = *(const gd_h8 *)(sf[k][0] + lane * 16), lo = *(const gd_h8 *)(sf[k][1] + lane * 16);
                x = gd_mfma(o.k[k][0], hi, x);
                y = gd_mfma(o.k[k][0], lo, y);
                z = gd_mfma(o.q[k][0], hi, z);
                w = gd_mfma(o.q[k][0], lo, w);
                if (PARTS > 1) {
                    y = gd_mfma(o.k[k][PARTS - 1], hi, y);
                    w = gd_mfma(o.q[k][PARTS - 1], hi, w);
                }
                load_key(o, c + 2, k);
            }
            gd_b4 part[3]; // half a fragment
            gd_split3(v * lift - o.fk * ((x + y * (1.0f / REST)) * (back_s * lift)), part);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *(gd_b4 *)(xf[wave / 2][p] + lane * 16 + 8 * (wave & 1)) = part[p];
            qs = (z + w * (1.0f / REST)) * back_s * o.fq;
        }
        load_rows(o, c + 2);
        scan_sync();
        // S <- e^G_64 S + M X;  O = scale (e^G Q S + P X)
        gd_b8 xp[2][3];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int p = 0; p < 3; ++p)
                xp[k][p] = *(const gd_b8 *)(xf[k][p] + lane * 16);
        gd_power(next, to_s, back_s);
        {
            gd_f4 x[MT]{}, y[MT]{};
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    gd_b8 part[3];
                    gd_split3(wide(o.m[m][k]), part);
                    gd_dot(part, xp[k], x[m], y[m]);
                    load_m(o, c + 2, m, k);
                }
#pragma unroll
            for (int m = 0; m < MT; ++m)
                S[m] = S[m] * keep + (x[m] + y[m]) * sink;
            put_s();
        }
        gd_f4 x{}, y{};
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (k == 0 || wave >= 2) {
                gd_b8 part[3];
                gd_split3(wide(o.p[k]), part);
                gd_dot(part, xp[k], x, y);
            }
        const gd_f4 out = a.scale * qs + (a.scale * sink) * (x + y);
        // through LDS, so that a lane stores 4 neighbours
#pragma unroll
        for (int i = 0; i < 4; ++i)
            turn[wave][4 * g + i][r] = out[i];
        const gd_f4 flat = *(const gd_f4 *)&turn[wave][lane / 4][4 * (lane % 4)];
        if (16 * wave + lane / 4 < n) {
            const int64_t where = ((seq.start + 64 * (int64_t)c) * a.v_heads + h) * a.v_dim + col0 + oat;
            if (a.raw)
                *(gd_f4 *)(a.raw + where) = flat;
            else
                gd_store4(a.out, where, a.out_type, flat);
        }
        load_p(o, c + 2);
    };
    Ops even, odd;
    load_all(even, 0);
    if (chunks > 1)
        load_all(odd, 1);
    int c = 0;
    for (; c + 1 < chunks; c += 2) { // (no way out between: the operands stay in their registers)
        chunk(even, c);
        chunk(odd, c + 1);
    }
    if (c < chunks)
        chunk(even, c);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 16 * (MT * wave + m) + 4 * g + i;
            if (at < a.k_dim)
                state[(int64_t)at * a.v_dim] = S[m][i];
        }
}

// ---- the output norm ---------------------------------------------------------------
constexpr int NORM_THREADS = 256;

// raw -> out: 32 lanes a row of a head (4 columns each), 64 rows of a sequence.  (The
// scan's workgroups hold 16 columns each and no row's norm.)  Bound by bytes: 8192 tokens of
// 32 heads of 128, raw and gate fp32, bf16 out: 75 us for 336 MB, 4.5 TB/s.
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
            o = gd_rms<32>(o, a.v_dim, a.norm_eps);
            if (live)
                o = o * *(const gd_f4 *)(a.norm_w + e);
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

template <int TYPE, int KD>
void launch(const DeltaArgs &a, hipStream_t s)
{
    const unsigned units = (unsigned)(a.plan.tiles * a.v_heads);
    hipLaunchKernelGGL((k_delta_prep<TYPE, KD>), dim3(units), dim3(PREP_THREADS), 0, s, a);
    const unsigned blocks = (unsigned)(a.v_dim / 16) * (unsigned)a.group;
    const unsigned heads = ((unsigned)(a.k_heads * a.batch.sequences) + 7) / 8 * 8;
    hipLaunchKernelGGL((k_delta_scan<TYPE, KD>), dim3(heads * blocks), dim3(64 * SCAN_WAVES), 0, s, a);
    if (a.norm_w || a.gate)
        hipLaunchKernelGGL(k_delta_norm, dim3(units), dim3(NORM_THREADS), 0, s, a);
}

template <int TYPE>
void launch(const DeltaArgs &a, hipStream_t s)
{
    a.k_dim <= 64 ? launch<TYPE, 64>(a, s) : launch<TYPE, 128>(a, s);
}

} // namespace

hipError_t launch_delta_chunks(const DeltaArgs &a, hipStream_t s)
{
    a.type == kF32 ? launch<kF32>(a, s) : a.type == kF16 ? launch<kF16>(a, s) : launch<kBF16>(a, s);
    return hipGetLastError();
}

} // namespace ihip
