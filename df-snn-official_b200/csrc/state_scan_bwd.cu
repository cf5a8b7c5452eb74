// state_scan_bwd.cu -- backward of the selective scan.
//
// With g_t the gradient of o_t (grad_y times the gate) and l_t that of h_t,
//   l_t = C_t g_t + a_(t+1) l_(t+1),   a_t = exp(d_t A),   q_t = a_t l_t h_(t-1)
//   grad C_t = sum_c g_t h_t     grad B_t = sum_c l_t d_t u_t     grad A = sum_(t,b) q_t d_t
//   grad u_t = d_t sum_n l_t B_t + D g_t      grad d_t = u_t sum_n l_t B_t + sum_n q_t A
// A warp walks the sequence of its channels backwards in chunks of 16 steps.  The forward kept
// the state in front of every chunk; from it the chunk's states and decays are formed again and
// stay in registers (2 * 16 floats for each state that a lane holds), so each exponential is
// taken once.  The sums over states (a channel's lanes) and over channels (the other lanes) are
// formed for several steps at a time (LaneSums).  The sums over channels then go over the warps
// in shared memory and over the blocks through partial sums that a second kernel adds in a fixed
// order; no atomics, so results do not change from run to run.
#include <algorithm>

#include "state_scan.h"

namespace dfsnn {
namespace {

constexpr int TT = kScanChunk, P = kScanPitch;
constexpr int NT = 128;

template <int S, int C, int SL>
struct Shape {
    static constexpr int CL = 32 / SL;               // channel lanes of a warp
    static constexpr int NW = NT / 32;
    static constexpr int BC = NW * CL * C;           // channels of the block
    static constexpr int NS = S * SL;                // states, padded
    static constexpr size_t smem(bool gate) {
        return sizeof(float) * ((size_t)(gate ? 4 : 3) * BC * P + 2 * (size_t)NS * P
                                + (size_t)NW * 2 * TT * NS);
    }
};

template <typename IO, int S, int C, int SL, bool GATE>
__global__ void __launch_bounds__(NT) scan_bwd(const ScanParams p) {
    using Sh = Shape<S, C, SL>;
    constexpr int CL = Sh::CL, NW = Sh::NW, BC = Sh::BC, NS = Sh::NS;
    constexpr int E = (TT * BC + NT - 1) / NT, TS = TT / E;
    constexpr int F = (TT * NS + NT - 1) / NT;
    extern __shared__ __align__(16) float smem[];
    float(*s_dt)[P] = reinterpret_cast<float(*)[P]>(smem);
    float(*s_u)[P] = s_dt + BC;
    float(*s_g)[P] = s_u + BC;
    float(*s_o)[P] = s_g + BC;                                 // with a gate only
    float(*s_B)[P] = GATE ? s_o + BC : s_o;
    float(*s_C)[P] = s_B + NS;
    float* s_red = reinterpret_cast<float*>(s_C + NS);         // [NW][2][TT][NS]
    const dfsnn_state_scan_args& a = p.a;
    const dfsnn_state_scan_grads& g = p.g;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long bid = blockIdx.x;
    const int tile = (int)(bid % p.tiles);
    bid /= p.tiles;
    const int grp = (int)(bid % a.groups);
    const int part = (int)(bid / a.groups);
    const int c_base = tile * BC;
    const long long g_base = (long long)grp * p.group_channels;

    // elementwise role: thread's channel ch, steps t_e + e * TS
    const int ch = tid % BC, t_e = tid / BC;
    const bool ch_ok = c_base + ch < p.group_channels && t_e < TT;
    const long long chan = g_base + c_base + ch;
    const float bias = ch_ok && a.delta_bias ? a.delta_bias[chan] : 0.0f;
    const float skip = ch_ok && a.D ? a.D[chan] : 0.0f;
    float sum_D = 0.0f, sum_bias = 0.0f;

    // recurrence role: states s * SL + sl of channels c * CL + lane / SL of this warp
    const int sl = lane % SL, cl = lane / SL;
    float A2[C][S], dA[C][S];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int k = c_base + warp * CL * C + c * CL + cl, n = s * SL + sl;
            const bool ok = k < p.group_channels && n < a.states;
            A2[c][s] = ok ? a.A[(g_base + k) * a.states + n] * kLog2e : 0.0f;
            dA[c][s] = 0.0f;
        }

    for (long long b = part; b < a.batch; b += p.batch_parts) {
        const int len = seq_length(a.lengths, a.lengths64, b, p.T);
        const IO* u_p = static_cast<const IO*>(a.u) + b * a.u_b + chan;
        const IO* d_p = static_cast<const IO*>(a.delta) + b * a.delta_b + chan;
        const IO* z_p = GATE ? static_cast<const IO*>(a.z) + b * a.z_b + chan : nullptr;
        const IO* gy_p = static_cast<const IO*>(g.grad_y) + b * a.y_b + chan;
        IO* gu_p = static_cast<IO*>(g.grad_u) + b * g.gu_b + chan;
        IO* gd_p = static_cast<IO*>(g.grad_delta) + b * g.gdelta_b + chan;
        IO* gz_p = GATE && g.grad_z ? static_cast<IO*>(g.grad_z) + b * g.gz_b + chan : nullptr;
        const IO* B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g;
        const IO* C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g;
        const long long row0 = ((long long)b * a.channels + g_base + c_base + warp * CL * C + cl) * a.states;

        float lam[C][S];                                       // a_(t+1) l_(t+1)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int n = s * SL + sl;
                const bool ok = c_base + warp * CL * C + c * CL + cl < p.group_channels && n < a.states;
                lam[c][s] = ok && g.grad_h_last ? g.grad_h_last[row0 + (long long)c * CL * a.states + n] : 0.0f;
            }

        // rows behind the end
        if (ch_ok)
            for (long long t = (long long)(len + TT - 1) / TT * TT + t_e; t < p.T; t += TS) {
                gu_p[t * g.gu_t] = from_f<IO>(0.0f);
                gd_p[t * g.gdelta_t] = from_f<IO>(0.0f);
                if (GATE && gz_p) gz_p[t * g.gz_t] = from_f<IO>(0.0f);
            }

        for (int t0 = (len - 1) / TT * TT; t0 >= 0 && len > 0; t0 -= TT) {
            float u_r[E], dt_r[E], x_r[E], g_r[E], z_r[E];     // x: input of the softplus; g: grad_y
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int tt = t_e + e * TS, t = t0 + tt;
                const bool ok = ch_ok && tt < TT && t < len;
                u_r[e] = ok ? to_f(u_p[t * a.u_t]) : 0.0f;
                x_r[e] = ok ? to_f(d_p[t * a.delta_t]) + bias : 0.0f;
                g_r[e] = ok ? to_f(gy_p[t * a.y_t]) : 0.0f;
                if (GATE) z_r[e] = ok ? to_f(z_p[t * a.z_t]) : 0.0f;
                dt_r[e] = a.softplus ? softplus_f(x_r[e]) : x_r[e];
                if (!ok) dt_r[e] = 0.0f;
                if (tt < TT) {
                    s_dt[ch][tt] = dt_r[e];
                    s_u[ch][tt] = u_r[e];
                    s_g[ch][tt] = GATE ? g_r[e] * (z_r[e] * sigmoid_f(z_r[e])) : g_r[e];
                }
            }
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int i = tid + f * NT, t = t0 + i / NS, n = i % NS;
                const bool ok = i < TT * NS && n < a.states && t < len;
                if (i < TT * NS) {
                    s_B[n][i / NS] = ok ? to_f(B_p[t * a.B_t + n]) : 0.0f;
                    s_C[n][i / NS] = ok ? to_f(C_p[t * a.C_t + n]) : 0.0f;
                }
            }
            __syncthreads();

            // the chunk's decays and states
            float da[C][S][TT], hh[C][S][TT + 1];
            const float* kept = t0 > 0 ? a.kept + (long long)(t0 / TT - 1) * a.batch * a.channels * a.states
                                       : a.h0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const int n = s * SL + sl;
                    const bool ok = c_base + warp * CL * C + c * CL + cl < p.group_channels && n < a.states;
                    hh[c][s][0] = ok && kept ? kept[row0 + (long long)c * CL * a.states + n] : 0.0f;
                }
            float o[GATE ? C : 1][TT];
#pragma unroll
            for (int t4 = 0; t4 < TT; t4 += 4) {
                float4 B4[S], C4[S];
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    B4[s] = *reinterpret_cast<const float4*>(&s_B[s * SL + sl][t4]);
                    if (GATE) C4[s] = *reinterpret_cast<const float4*>(&s_C[s * SL + sl][t4]);
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int k = warp * CL * C + c * CL + cl;
                    const float4 dt4 = *reinterpret_cast<const float4*>(&s_dt[k][t4]);
                    const float4 u4 = *reinterpret_cast<const float4*>(&s_u[k][t4]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const float dt = (&dt4.x)[t], du = dt * (&u4.x)[t];
                        float acc = 0.0f;
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            const float d = exp2_approx(dt * A2[c][s]);
                            da[c][s][t4 + t] = d;
                            hh[c][s][t4 + t + 1] = fmaf(d, hh[c][s][t4 + t], du * (&B4[s].x)[t]);
                            if (GATE) acc = fmaf(hh[c][s][t4 + t + 1], (&C4[s].x)[t], acc);
                        }
                        if (GATE) o[c][t4 + t] = acc;
                    }
                }
            }
            if (GATE) {
                using Sums = LaneSums<TT, SL, 1>;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    Sums::run(o[c], sl);
                    if (Sums::stores(sl))
#pragma unroll
                        for (int i = 0; i < Sums::kHeld; ++i)
                            s_o[warp * CL * C + c * CL + cl][Sums::first(sl) + i] = o[c][i];
                }
            }

            // and backwards through it, 8 steps at a time
            constexpr int R = 8;
#pragma unroll
            for (int tr = TT - R; tr >= 0; tr -= R) {
                float s1[C][R], s2[C][R];
#pragma unroll
                for (int t4 = R - 4; t4 >= 0; t4 -= 4) {
                    float4 B4[S], C4[S];
                    float dB[S][4], dC[S][4];
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        B4[s] = *reinterpret_cast<const float4*>(&s_B[s * SL + sl][tr + t4]);
                        C4[s] = *reinterpret_cast<const float4*>(&s_C[s * SL + sl][tr + t4]);
#pragma unroll
                        for (int t = 0; t < 4; ++t) dB[s][t] = dC[s][t] = 0.0f;
                    }
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const int k = warp * CL * C + c * CL + cl;
                        const float4 dt4 = *reinterpret_cast<const float4*>(&s_dt[k][tr + t4]);
                        const float4 u4 = *reinterpret_cast<const float4*>(&s_u[k][tr + t4]);
                        const float4 g4 = *reinterpret_cast<const float4*>(&s_g[k][tr + t4]);
#pragma unroll
                        for (int t = 3; t >= 0; --t) {
                            const float dt = (&dt4.x)[t], du = dt * (&u4.x)[t], gt = (&g4.x)[t];
                            float r1 = 0.0f, r2 = 0.0f;
#pragma unroll
                            for (int s = 0; s < S; ++s) {
                                const float l = fmaf((&C4[s].x)[t], gt, lam[c][s]);
                                lam[c][s] = l * da[c][s][tr + t4 + t];
                                const float q = lam[c][s] * hh[c][s][tr + t4 + t];
                                dB[s][t] = fmaf(l, du, dB[s][t]);
                                dC[s][t] = fmaf(gt, hh[c][s][tr + t4 + t + 1], dC[s][t]);
                                r1 = fmaf(l, (&B4[s].x)[t], r1);
                                r2 = fmaf(q, A2[c][s], r2);
                                dA[c][s] = fmaf(q, dt, dA[c][s]);
                            }
                            s1[c][t4 + t] = r1;
                            s2[c][t4 + t] = r2;
                        }
                    }
                    using Sums = LaneSums<4, CL, SL>;
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        Sums::run(dB[s], cl);
                        Sums::run(dC[s], cl);
                        if (Sums::stores(cl)) {
#pragma unroll
                            for (int i = 0; i < Sums::kHeld; ++i) {
                                const int t = tr + t4 + Sums::first(cl) + i, n = s * SL + sl;
                                s_red[((warp * 2 + 0) * TT + t) * NS + n] = dB[s][i];
                                s_red[((warp * 2 + 1) * TT + t) * NS + n] = dC[s][i];
                            }
                        }
                    }
                }
                using Sums = LaneSums<R, SL, 1>;
                __syncwarp();
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    Sums::run(s1[c], sl);
                    Sums::run(s2[c], sl);
                    // the sums go where this warp's d and u of these steps were
                    if (Sums::stores(sl)) {
                        const int k = warp * CL * C + c * CL + cl;
#pragma unroll
                        for (int i = 0; i < Sums::kHeld; ++i) {
                            s_dt[k][tr + Sums::first(sl) + i] = s1[c][i];
                            s_u[k][tr + Sums::first(sl) + i] = s2[c][i];
                        }
                    }
                }
            }
            __syncthreads();

            // elementwise gradients
            if (ch_ok) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int tt = t_e + e * TS, t = t0 + tt;
                    if (tt < TT && t < p.T) {
                        const float lb = s_dt[ch][tt], qa = s_u[ch][tt] * 0.69314718055994530942f;
                        float gt = g_r[e], gz = 0.0f;
                        if (GATE) {
                            const float sg = sigmoid_f(z_r[e]), si = z_r[e] * sg;
                            gz = gt * fmaf(skip, u_r[e], s_o[ch][tt]) * fmaf(si, 1.0f - sg, sg);
                            gt *= si;
                        }
                        float gd = fmaf(u_r[e], lb, qa);
                        if (a.softplus) gd *= sigmoid_f(x_r[e]);
                        float gu = fmaf(dt_r[e], lb, skip * gt);
                        if (t >= len) gd = gu = gz = 0.0f;
                        gu_p[t * g.gu_t] = from_f<IO>(gu);
                        gd_p[t * g.gdelta_t] = from_f<IO>(gd);
                        if (GATE && gz_p) gz_p[t * g.gz_t] = from_f<IO>(gz);
                        sum_bias += gd;
                        sum_D = fmaf(gt, u_r[e], sum_D);
                    }
                }
            }
            // this block's part of grad B and grad C
            for (int i = tid; i < 2 * TT * NS; i += NT) {
                const int n = i % NS, t = t0 + i / NS % TT, which = i / (NS * TT);
                if (n < a.states && t < len) {
                    float v = 0.0f;
#pragma unroll
                    for (int w = 0; w < NW; ++w) v += s_red[w * 2 * TT * NS + i];
                    p.part_bc[((((long long)which * p.tiles + tile) * p.T + t) * a.batch + b) * a.groups * a.states
                              + grp * a.states + n] = v;
                }
            }
            __syncthreads();
        }
        if (g.grad_h0) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const int n = s * SL + sl;
                    if (c_base + warp * CL * C + c * CL + cl < p.group_channels && n < a.states)
                        g.grad_h0[row0 + (long long)c * CL * a.states + n] = lam[c][s];
                }
        }
    }

#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int k = c_base + warp * CL * C + c * CL + cl, n = s * SL + sl;
            if (k < p.group_channels && n < a.states)
                p.part_a[((long long)part * a.channels + g_base + k) * a.states + n] = dA[c][s];
        }
    // the threads of a channel, in order
    __syncthreads();
    smem[tid] = sum_D;
    smem[NT + tid] = sum_bias;
    __syncthreads();
    if (tid < BC && c_base + tid < p.group_channels) {
        float d = 0.0f, e = 0.0f;
        for (int i = tid; i < NT; i += BC) {
            d += smem[i];
            e += smem[NT + i];
        }
        p.part_d[(long long)part * a.channels + chan] = d;
        p.part_d[((long long)p.batch_parts + part) * a.channels + chan] = e;
    }
}

// Adds the blocks' parts: grad B and grad C over the channel tiles, then grad A, D and delta_bias
// over the batch parts, one thread for an output, in order.
template <typename IO>
__global__ void scan_bwd_sums(const ScanParams p, long long n_bc, long long n_a) {
    const dfsnn_state_scan_args& a = p.a;
    const dfsnn_state_scan_grads& g = p.g;
    const long long total = 2 * n_bc + n_a + 2 * a.channels;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (long long)gridDim.x * blockDim.x) {
        float v = 0.0f;
        if (i < 2 * n_bc) {
            const int which = i >= n_bc;
            const long long k = i - which * n_bc, row = k / ((long long)a.groups * a.states);
            if (row / a.batch < seq_length(a.lengths, a.lengths64, row % a.batch, p.T)) {
                const float* q = p.part_bc + (long long)which * p.tiles * n_bc + k;
                for (int j = 0; j < p.tiles; ++j) v += q[j * n_bc];
            }
            static_cast<IO*>(which ? g.grad_C : g.grad_B)[k] = from_f<IO>(v);
        } else if (i < 2 * n_bc + n_a) {
            const long long k = i - 2 * n_bc;
            for (int j = 0; j < p.batch_parts; ++j) v += p.part_a[j * n_a + k];
            g.grad_A[k] = v;
        } else {
            const long long k = i - 2 * n_bc - n_a;
            const int which = k >= a.channels;
            float* out = which ? g.grad_delta_bias : g.grad_D;
            if (out) {
                const long long c = k - which * a.channels;
                for (int j = 0; j < p.batch_parts; ++j)
                    v += p.part_d[((long long)which * p.batch_parts + j) * a.channels + c];
                out[c] = v;
            }
        }
    }
}

// Channels of a block for a state count (the shapes that pick() launches)
int block_channels(int states) {
    if (states <= 4) return Shape<4, 1, 1>::BC;
    if (states <= 8) return Shape<2, 2, 4>::BC;
    if (states <= 16) return Shape<2, 2, 8>::BC;
    if (states <= 32) return Shape<2, 2, 16>::BC;
    if (states <= 64) return Shape<2, 2, 32>::BC;
    return Shape<4, 1, 32>::BC;
}

template <typename IO, int S, int C, int SL, bool GATE>
cudaError_t launch_gate(const ScanParams& p, cudaStream_t st) {
    const long long blocks = (long long)p.tiles * p.a.groups * p.batch_parts;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    constexpr size_t smem = Shape<S, C, SL>::smem(GATE);
    cudaError_t e = cudaFuncSetAttribute(scan_bwd<IO, S, C, SL, GATE>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    scan_bwd<IO, S, C, SL, GATE><<<(unsigned)blocks, NT, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename IO, int S, int C, int SL>
cudaError_t launch(const ScanParams& p, cudaStream_t st) {
    return p.a.z ? launch_gate<IO, S, C, SL, true>(p, st) : launch_gate<IO, S, C, SL, false>(p, st);
}

template <typename IO>
cudaError_t pick(const ScanParams& p, cudaStream_t st) {
    const int n = p.a.states;
    cudaError_t e;
    if (n <= 4) e = launch<IO, 4, 1, 1>(p, st);
    else if (n <= 8) e = launch<IO, 2, 2, 4>(p, st);
    else if (n <= 16) e = launch<IO, 2, 2, 8>(p, st);
    else if (n <= 32) e = launch<IO, 2, 2, 16>(p, st);
    else if (n <= 64) e = launch<IO, 2, 2, 32>(p, st);
    else e = launch<IO, 4, 1, 32>(p, st);
    if (e != cudaSuccess) return e;
    const long long n_bc = (long long)p.T * p.a.batch * p.a.groups * p.a.states;
    const long long n_a = p.a.channels * p.a.states;
    const long long total = 2 * n_bc + n_a + 2 * p.a.channels;
    const unsigned blocks = (unsigned)std::min<long long>((total + 255) / 256, 148 * 16);
    scan_bwd_sums<IO><<<blocks, 256, 0, st>>>(p, n_bc, n_a);
    return cudaGetLastError();
}

}  // namespace

int state_scan_bwd_tiles(int states, long long group_channels) {
    const int bc = block_channels(states);
    return (int)((group_channels + bc - 1) / bc);
}

// Blocks that share the batch: enough for 16 blocks an SM; beyond that each block takes several
// sequences and adds its grad A on the way, which keeps the partial sums small.
int state_scan_bwd_batch_parts(int states, long long batch, long long group_channels, int groups) {
    const long long per = (long long)state_scan_bwd_tiles(states, group_channels) * groups;
    const long long want = (148 * 16 + per - 1) / per;
    return (int)std::max<long long>(1, std::min(batch, want));
}

cudaError_t state_scan_backward_launch(const ScanParams& p, cudaStream_t st) {
    switch (p.a.dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(p, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(p, st);
        default: return pick<float>(p, st);
    }
}

}  // namespace dfsnn
