// state_scan_fwd.cu -- forward of the selective scan.
//
//   h_t[n] = exp(d_t A[n]) h_(t-1)[n] + d_t u_t B_t[n],   o_t = sum_n C_t[n] h_t[n] + D u_t
//
// One exponential and about five multiply-adds for each (step, channel, state), against 3 or 4
// elements of traffic for all N states of a (step, channel): with N = 16 the kernel is bound by
// the 16 exponentials a clock of an SM's special-function unit, not by memory.  Everything that
// is not an exponential therefore has to fit beside them:
//   * a channel's states are spread over SL lanes, S states each, and every warp walks the whole
//     sequence of its 32 / SL channels, so the recurrence needs no second pass;
//   * steps are taken in tiles of 16, and the sums over a channel's lanes are formed for the 16
//     steps together (LaneSums): (1 - 1/SL) shuffles a step instead of log2 SL;
//   * the elementwise work (softplus, gate, skip) is done once per (step, channel) by all threads
//     of the block, before and after the tile, with the next tile's loads in flight meanwhile.
// States, decays and sums are fp32; y is rounded once.
#include "state_scan.h"

namespace dfsnn {
namespace {

constexpr int TT = kScanChunk, P = kScanPitch;

template <typename IO, int S, int SL, int NT>
__global__ void __launch_bounds__(NT) scan_fwd(const ScanParams p) {
    constexpr int CL = 32 / SL;                 // channels of a warp
    constexpr int BC = NT / 32 * CL;            // channels of the block
    constexpr int NS = S * SL;                  // states, padded
    constexpr int E = CL > 1 ? CL / 2 : 1;      // (step, channel) elements of a thread
    constexpr int F = (TT * NS + NT - 1) / NT;  // entries of B (and C) of a thread
    __shared__ __align__(16) float s_dt[BC][P], s_du[BC][P], s_B[NS][P], s_C[NS][P];
    const dfsnn_state_scan_args& a = p.a;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long bid = blockIdx.x;
    const int tile = (int)(bid % p.tiles);
    bid /= p.tiles;
    const int grp = (int)(bid % a.groups);
    const long long b = bid / a.groups;
    const int len = seq_length(a.lengths, a.lengths64, b, p.T);
    const int c_base = tile * BC;                               // within the group
    const long long g_base = (long long)grp * p.group_channels; // first channel of the group

    // elementwise role: element e is (step t_e + e * SL, channel ch)
    const int ch = tid % BC, t_e = tid / BC;
    const bool ch_ok = c_base + ch < p.group_channels && t_e < TT;
    const long long chan = g_base + c_base + ch;
    const float bias = ch_ok && a.delta_bias ? a.delta_bias[chan] : 0.0f;
    const float skip = ch_ok && a.D ? a.D[chan] : 0.0f;
    const IO* u_p = static_cast<const IO*>(a.u) + b * a.u_b + chan;
    const IO* d_p = static_cast<const IO*>(a.delta) + b * a.delta_b + chan;
    const IO* z_p = a.z ? static_cast<const IO*>(a.z) + b * a.z_b + chan : nullptr;
    IO* y_p = static_cast<IO*>(a.y) + b * a.y_b + chan;
    const IO* B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g;
    const IO* C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g;

    // recurrence role: states n = s * SL + sl of channel cl of this warp
    const int sl = lane % SL, cl = warp * CL + lane / SL;
    const bool cl_ok = c_base + cl < p.group_channels;
    const long long row = ((long long)b * a.channels + g_base + c_base + cl) * a.states;
    float A2[S], h[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int n = s * SL + sl;
        const bool ok = cl_ok && n < a.states;
        A2[s] = ok ? a.A[(g_base + c_base + cl) * a.states + n] * kLog2e : 0.0f;
        h[s] = ok && a.h0 ? a.h0[row + n] : 0.0f;
    }

    float u_r[E], d_r[E], z_r[E], B_r[F], C_r[F];
    auto load = [&](int t0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = t0 + t_e + e * SL;
            const bool ok = ch_ok && t < len;
            u_r[e] = ok ? to_f(u_p[t * a.u_t]) : 0.0f;
            d_r[e] = ok ? to_f(d_p[t * a.delta_t]) : 0.0f;
            z_r[e] = ok && z_p ? to_f(z_p[t * a.z_t]) : 0.0f;
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int i = tid + f * NT, t = t0 + i / NS, n = i % NS;
            const bool ok = i < TT * NS && n < a.states && t < len;
            B_r[f] = ok ? to_f(B_p[t * a.B_t + n]) : 0.0f;
            C_r[f] = ok ? to_f(C_p[t * a.C_t + n]) : 0.0f;
        }
    };

    load(0);
    for (int t0 = 0; t0 < len; t0 += TT) {
        float u_c[E], z_c[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            u_c[e] = u_r[e];
            z_c[e] = z_r[e];
            const int t = t_e + e * SL;
            float dt = d_r[e] + bias;
            if (a.softplus) dt = softplus_f(dt);
            if (t0 + t >= len) dt = 0.0f;       // a step behind the end leaves the state alone
            if (t < TT) {
                s_dt[ch][t] = dt;
                s_du[ch][t] = dt * u_r[e];
            }
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int i = tid + f * NT;
            if (i < TT * NS) {
                s_B[i % NS][i / NS] = B_r[f];
                s_C[i % NS][i / NS] = C_r[f];
            }
        }
        __syncthreads();
        if (t0 + TT < len) load(t0 + TT);
        if (a.kept && t0 > 0 && cl_ok) {
            float* k = a.kept + (long long)(t0 / TT - 1) * a.batch * a.channels * a.states + row;
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (s * SL + sl < a.states) k[s * SL + sl] = h[s];
        }
        float y[TT];
#pragma unroll
        for (int t4 = 0; t4 < TT; t4 += 4) {
            const float4 dt4 = *reinterpret_cast<const float4*>(&s_dt[cl][t4]);
            const float4 du4 = *reinterpret_cast<const float4*>(&s_du[cl][t4]);
            float4 B4[S], C4[S];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                B4[s] = *reinterpret_cast<const float4*>(&s_B[s * SL + sl][t4]);
                C4[s] = *reinterpret_cast<const float4*>(&s_C[s * SL + sl][t4]);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float dt = (&dt4.x)[t], du = (&du4.x)[t];
                float acc = 0.0f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    h[s] = fmaf(exp2_approx(dt * A2[s]), h[s], du * (&B4[s].x)[t]);
                    acc = s == 0 ? h[s] * (&C4[s].x)[t] : fmaf(h[s], (&C4[s].x)[t], acc);
                }
                y[t4 + t] = acc;
            }
        }
        using Sums = LaneSums<TT, SL, 1>;
        Sums::run(y, sl);
        // the sums go where the warp's own steps of d were
        __syncwarp();
        if (Sums::stores(sl)) {
#pragma unroll
            for (int i = 0; i < Sums::kHeld; ++i) s_dt[cl][Sums::first(sl) + i] = y[i];
        }
        __syncthreads();
        if (ch_ok) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int t = t_e + e * SL;
                if (t < TT && t0 + t < p.T) {
                    float o = fmaf(skip, u_c[e], s_dt[ch][t]);
                    if (z_p) o *= z_c[e] * sigmoid_f(z_c[e]);
                    if (t0 + t >= len) o = 0.0f;
                    y_p[(t0 + t) * a.y_t] = from_f<IO>(o);
                }
            }
        }
    }
    // rows behind the end
    if (ch_ok)
        for (long long t = (long long)(len + TT - 1) / TT * TT + t_e; t < p.T; t += SL)
            y_p[t * a.y_t] = from_f<IO>(0.0f);
    if (a.h_last && cl_ok) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s * SL + sl < a.states) a.h_last[row + s * SL + sl] = h[s];
    }
}

template <typename IO, int S, int SL>
cudaError_t launch(ScanParams p, cudaStream_t st) {
    constexpr int NT = 128, BC = NT / 32 * (32 / SL);
    p.tiles = (p.group_channels + BC - 1) / BC;
    const long long blocks = (long long)p.tiles * p.a.groups * p.a.batch;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    scan_fwd<IO, S, SL, NT><<<(unsigned)blocks, NT, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename IO>
cudaError_t pick(const ScanParams& p, cudaStream_t st) {
    const int n = p.a.states;
    if (n <= 4) return launch<IO, 4, 1>(p, st);
    if (n <= 8) return launch<IO, 2, 4>(p, st);
    if (n <= 16) return launch<IO, 2, 8>(p, st);
    if (n <= 32) return launch<IO, 2, 16>(p, st);
    if (n <= 64) return launch<IO, 4, 16>(p, st);
    return launch<IO, 4, 32>(p, st);
}

}  // namespace

cudaError_t state_scan_forward_launch(const ScanParams& p, cudaStream_t st) {
    switch (p.a.dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(p, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(p, st);
        default: return pick<float>(p, st);
    }
}

}  // namespace dfsnn
