// gd_step.hip -- the gated delta rule a token after the other, for sequences with
// few new tokens.  A head's state S (k_dim x v_dim, fp32) forgets, and then writes
// the part of v that k does not bring back already:
//
//   S <- alpha S;  d = beta (v - k^T S);  S <- S + k d^T;  o = scale q^T S
//
// with q and k scaled to unit length, alpha = exp(decay softplus(a + dt_bias)) and
// beta = sigmoid(b).  Both products with S are formed from the state before the
// token, q^T S_new = alpha q^T S + (q.k) d, so the state is passed over once a token.
#include "gd_launch.h"

namespace ihip {

namespace {

constexpr int STEP_THREADS = 256;
constexpr int STEP_WAVES = STEP_THREADS / 64;
constexpr int STEP_TOKENS = 16; // whose q, k and o a workgroup holds in LDS at once

// A workgroup takes one head of one sequence and keeps its state in registers.  The
// columns of S do not touch each other, so a wave has VD / 4 of them to itself: a lane
// holds 4 columns of R rows, a product with S is summed over the wave's row groups by
// lane moves, and the tokens follow each other without a barrier.  Bound by the
// state's bytes for a batch (61 tokens, 32 heads of 128 x 128: 66 to 68 us for 260 MB, 3.8
// to 3.9 TB/s), by loads that wait for each other for one sequence (8.7 us), and by
// the chain of a token's sums for several (1.4 us a token).
template <int TYPE, int KD, int VD>
__global__ void __launch_bounds__(STEP_THREADS) k_delta_step(DeltaArgs a)
{
    constexpr int CL = VD / 4 / STEP_WAVES; // lanes side by side over a wave's columns
    constexpr int RG = 64 / CL;             // row groups
    constexpr int R = KD / RG;              // rows of a lane
    constexpr int PAD = R + 4;              // (row groups apart in LDS)
    __shared__ __attribute__((aligned(16))) float qs[STEP_TOKENS][RG * PAD], ks[STEP_TOKENS][RG * PAD];
    __shared__ __attribute__((aligned(16))) float os[STEP_TOKENS][VD];
    __shared__ float alpha[STEP_TOKENS], beta[STEP_TOKENS], qk[STEP_TOKENS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x % a.v_heads, s = blockIdx.x / a.v_heads, kh = h / a.group;
    if (a.flags && blockIdx.x == 0)
        gd_report(a.batch, a.flags);
    const GdSeq seq = gd_seq(a.batch, a.pool, s, h == 0 ? a.flags : nullptr);
    if (seq.slot < 0 || seq.n == 0 || (a.few >= 0 && seq.n > a.few))
        return;
    const int row0 = R * (lane / CL), col0 = wave * (VD / STEP_WAVES) + 4 * (lane % CL);
    float *state = a.state + seq.slot * a.slot_step + (int64_t)h * a.k_dim * a.v_dim;
    gd_f4 S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        S[i] = gd_f4{};
        if (!seq.begins && row0 + i < a.k_dim && col0 < a.v_dim)
            S[i] = *(const gd_f4 *)(state + (row0 + i) * a.v_dim + col0);
    }
    for (int t0 = 0; t0 < seq.n; t0 += STEP_TOKENS) {
        const int n = min(STEP_TOKENS, seq.n - t0);
        const int64_t first = seq.start + t0;
        if (t0)
            __syncthreads(); // (os is read, qs and ks are)
        // a wave a token: q and k to unit length, the sums in 64 bits, where no
        // square of an fp32 value passes the range
        for (int t = wave; t < n; t += STEP_WAVES) {
            const int64_t qa = (first + t) * a.q_step + (int64_t)kh * a.k_dim, ka = (first + t) * a.k_step + (int64_t)kh * a.k_dim;
            constexpr int E = KD / 64;
            typedef typename GdType<TYPE>::T T;
            float x[E], y[E];
            double xx = 0.0, yy = 0.0, xy = 0.0;
            T xr[E], yr[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int e = min(lane * E + i, a.k_dim - 1);
                xr[i] = ((const T *)a.q)[qa + e], yr[i] = ((const T *)a.k)[ka + e];
            }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const bool in = lane * E + i < a.k_dim;
                x[i] = in ? (float)xr[i] : 0.0f, y[i] = in ? (float)yr[i] : 0.0f;
                xx += (double)x[i] * x[i], yy += (double)y[i] * y[i], xy += (double)x[i] * y[i];
            }
            xx = gd_wave_sum(xx) + (double)a.l2_eps, yy = gd_wave_sum(yy) + (double)a.l2_eps;
            // (a row of zeros stays one, without an eps too)
            const double rq = xx == 0.0 ? 0.0 : 1.0 / sqrt(xx), rk = yy == 0.0 ? 0.0 : 1.0 / sqrt(yy);
            xy = gd_wave_sum(xy);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int e = lane * E + i, at = e / R * PAD + e % R;
                qs[t][at] = (float)(rq * x[i]);
                ks[t][at] = (float)(rk * y[i]);
            }
            if (lane == 0) {
                alpha[t] = expf(gd_log_decay(a.decay[h], a.a[(first + t) * a.a_step + h], a.dt_bias[h]));
                beta[t] = gd_beta(a.b[(first + t) * a.b_step + h]);
                qk[t] = (float)(rq * rk * xy);
            }
        }
        __syncthreads();
        for (int t = 0; t < n; ++t) {
            const gd_f4 v = col0 < a.v_dim ? gd_wide(gd_raw4<TYPE>(a.v, (first + t) * a.v_step + (int64_t)h * a.v_dim + col0)) : gd_f4{};
            float k[R];
            gd_f4 kS{}, qS{};
#pragma unroll
            for (int i = 0; i < R; i += 4) {
                const gd_f4 k4 = *(const gd_f4 *)&ks[t][lane / CL * PAD + i], q4 = *(const gd_f4 *)&qs[t][lane / CL * PAD + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    k[i + j] = k4[j];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        kS[e] = fmaf(k4[j], S[i + j][e], kS[e]);
                        qS[e] = fmaf(q4[j], S[i + j][e], qS[e]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (CL <= 4) {
                    kS[e] = gd_add_dpp<0x124>(gd_add_dpp<0x128>(kS[e])); // row_ror:8, row_ror:4
                    qS[e] = gd_add_dpp<0x124>(gd_add_dpp<0x128>(qS[e]));
                } else {
                    kS[e] = gd_add_dpp<0x128>(kS[e]);
                    qS[e] = gd_add_dpp<0x128>(qS[e]);
                }
                kS[e] = gd_add32(gd_add16(kS[e]));
                qS[e] = gd_add32(gd_add16(qS[e]));
            }
            const float al = alpha[t], be = beta[t], w = qk[t];
            gd_f4 d, o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[e] = be * (v[e] - al * kS[e]);
                o[e] = a.scale * fmaf(w, d[e], al * qS[e]);
            }
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    S[i][e] = fmaf(k[i], d[e], al * S[i][e]);
            if (lane < CL)
                *(gd_f4 *)&os[t][col0] = o;
        }
        __syncthreads();
        for (int i = tid; i < n * (VD / 4); i += STEP_THREADS) {
            const int t = i / (VD / 4), e0 = 4 * (i % (VD / 4));
            gd_f4 o = *(const gd_f4 *)&os[t][e0]; // (columns behind v_dim hold zeros)
            if (a.norm_w)
                o = gd_rms<VD / 4>(o, a.v_dim, a.norm_eps);
            if (e0 >= a.v_dim)
                continue;
            if (a.norm_w)
                o = o * *(const gd_f4 *)(a.norm_w + e0);
            if (a.gate) {
                const gd_f4 z = *(const gd_f4 *)(a.gate + (first + t) * a.gate_step + (int64_t)h * a.v_dim + e0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[e] *= gd_silu(z[e]);
            }
            gd_store4(a.out, ((first + t) * a.v_heads + h) * a.v_dim + e0, a.out_type, o);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (row0 + i < a.k_dim && col0 < a.v_dim)
            *(gd_f4 *)(state + (row0 + i) * a.v_dim + col0) = S[i];
}

template <int TYPE>
void launch(const DeltaArgs &a, hipStream_t s)
{
    const dim3 grid((unsigned)a.batch.sequences * (unsigned)a.v_heads);
    const bool k64 = a.k_dim <= 64, v64 = a.v_dim <= 64;
    if (k64 && v64)
        hipLaunchKernelGGL((k_delta_step<TYPE, 64, 64>), grid, dim3(STEP_THREADS), 0, s, a);
    else if (k64)
        hipLaunchKernelGGL((k_delta_step<TYPE, 64, 128>), grid, dim3(STEP_THREADS), 0, s, a);
    else if (v64)
        hipLaunchKernelGGL((k_delta_step<TYPE, 128, 64>), grid, dim3(STEP_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_delta_step<TYPE, 128, 128>), grid, dim3(STEP_THREADS), 0, s, a);
}

} // namespace

hipError_t launch_delta_step(const DeltaArgs &a, hipStream_t s)
{
    a.type == kF32 ? launch<kF32>(a, s) : a.type == kF16 ? launch<kF16>(a, s) : launch<kBF16>(a, s);
    return hipGetLastError();
}

} // namespace ihip
