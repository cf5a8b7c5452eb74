// state_step.cu -- one token of the selective scan for each row of a batch.
//
//   h[n] = exp(d A[n]) h[n] + d u B[n],   y = (sum_n C[n] h[n] + D u) * gate
//
// The state goes in and out once (8 bytes for each state), everything else is N times smaller:
// a large batch is bound by memory and a small one by the launch.  A channel's N states are spread
// over LG lanes with V neighbouring states each, so a warp reads and writes whole lines.
// N = 16, bf16: 1 x 2048 2.4 us, 192 x 4096 (100 MB) 25.5 us, 3.9 TB/s.
#include "state_space.cuh"

namespace dfsnn {
namespace {

constexpr int NT = 128;

// K groups of V states a lane: n = (k * LG + sl) * V + i.  A thread takes M <= LG channels, NT / LG
// apart, whose states are all requested before the first is used.  Of the elementwise work (softplus,
// gate, skip) each lane does that of one of the M channels, and hands d and d u to the others.
template <typename IO, int V, int LG, int K, int M>
__global__ void __launch_bounds__(NT, M == 4 ? 6 : 1) scan_step(const dfsnn_state_scan_step_args a, int tiles,
                                                                int group_channels) {
    constexpr int BC = NT / LG;
    using Sums = LaneSums<M, LG, 1>;
    const int tid = threadIdx.x, lane = tid & 31, sl = tid % LG, mine = Sums::first(sl);
    const long long b = blockIdx.x / tiles;
    const long long c0 = (long long)(blockIdx.x % tiles) * BC * M + tid / LG, own = c0 + mine * BC;
    const bool own_ok = own < a.channels;
    IO* y_p = static_cast<IO*>(a.y) + b * a.y_b;
    // what does not depend on the slot, before it is known
    float u = 0.0f, d = 0.0f, z = 0.0f, skip = 0.0f;
    if (own_ok) {
        u = to_f(static_cast<const IO*>(a.u)[b * a.u_b + own]);
        d = to_f(static_cast<const IO*>(a.delta)[b * a.delta_b + own]);
        if (a.z) z = to_f(static_cast<const IO*>(a.z)[b * a.z_b + own]);
        if (a.D) skip = a.D[own];
        if (a.delta_bias) d += a.delta_bias[own];
    }
    const long long stride = (long long)BC * a.states;          // floats between a thread's channels
    auto load = [&](float(&v)[M][K][V], const float* q) {
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int n = (k * LG + sl) * V;
                if (c0 + m * BC < a.channels && n < a.states) {
                    if constexpr (V == 4) *reinterpret_cast<float4*>(v[m][k]) = *reinterpret_cast<const float4*>(q + m * stride + n);
                    else v[m][k][0] = q[m * stride + n];
                }
            }
    };
    float A[M][K][V] = {}, h[M][K][V] = {};
    load(A, a.A + c0 * a.states);
    long long slot = step_slot(a.index, a.index64, b, a.slots);
    const bool ours = slot >= 0;
    if (ours) load(h, a.state + slot * a.state_s + c0 * a.states);
    if (taken_before(a.index, a.index64, b, slot) && ours) slot = kBad;
    if (slot < 0) {
        if (Sums::stores(sl) && own_ok) y_p[own] = from_f<IO>(slot == kIdle ? 0.0f : __int_as_float(0x7fc00000));
        return;
    }
    if (a.softplus) d = softplus_f(d);
    const float du = d * u;
    float* o_p = a.state_out + slot * a.out_s + c0 * a.states;
    float Bv[K][V], Cv[K][V], acc[M];
    long long have = -1;                        // the group of Bv and Cv
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const long long c = c0 + m * BC;
        const long long grp = a.groups == 1 ? 0 : (c < a.channels ? c : a.channels - 1) / group_channels;
        if (grp != have) {
            have = grp;
            const IO* B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g;
            const IO* C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int n = (k * LG + sl) * V + i;
                    Bv[k][i] = n < a.states ? to_f(B_p[n]) : 0.0f;
                    Cv[k][i] = n < a.states ? to_f(C_p[n]) : 0.0f;
                }
        }
        const int from = (lane - sl) + m * (LG / M);
        const float dm = __shfl_sync(0xffffffffu, d, from) * kLog2e, dum = __shfl_sync(0xffffffffu, du, from);
        acc[m] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < V; i += V > 1 ? 2 : 1) {
                const int i1 = V > 1 ? i + 1 : i;
                const float2 x = __fmul2_rn(make_float2(dm, dm), make_float2(A[m][k][i], A[m][k][i1]));
                const float2 q = exp2_near1(x);
                const float2 dec = make_float2(fabsf(x.x) < kExp2Near ? q.x : exp2_approx(x.x),
                                               fabsf(x.y) < kExp2Near ? q.y : exp2_approx(x.y));
                const float2 in = __fmul2_rn(make_float2(dum, dum), make_float2(Bv[k][i], Bv[k][i1]));
                const float2 hn = __ffma2_rn(dec, make_float2(h[m][k][i], h[m][k][i1]), in);
                h[m][k][i] = hn.x;
                acc[m] = fmaf(Cv[k][i], hn.x, acc[m]);
                if (V > 1) {
                    h[m][k][i1] = hn.y;
                    acc[m] = fmaf(Cv[k][i1], hn.y, acc[m]);
                }
            }
            const int n = (k * LG + sl) * V;
            if (c < a.channels && n < a.states) {
                if constexpr (V == 4) *reinterpret_cast<float4*>(o_p + m * stride + n) = *reinterpret_cast<float4*>(h[m][k]);
                else o_p[m * stride + n] = h[m][k][0];
            }
        }
    }
    Sums::run(acc, sl);
    if (Sums::stores(sl) && own_ok) {
        float o = fmaf(skip, u, acc[0]);
        if (a.z) o *= z * sigmoid_f(z);
        y_p[own] = from_f<IO>(o);
    }
}

// One channel a thread for few rows (latency); up to four where that still leaves 4 blocks an SM:
// N = 16, bf16, 64 x 2048 5.7 us with four against 8.2 with one, 192 x 4096 25.5 against 49.3
template <typename IO, int V, int LG, int K>
cudaError_t launch(const dfsnn_state_scan_step_args& a, cudaStream_t st) {
    constexpr int M = K > 1 ? 1 : LG < 4 ? LG : 4;
    const long long bc = NT / LG;
    const bool many = (a.channels + M * bc - 1) / (M * bc) * a.batch >= 148 * 4;
    const long long per = many ? M * bc : bc, tiles = (a.channels + per - 1) / per, blocks = tiles * a.batch;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const int gc = (int)(a.channels / a.groups);
    if (many) scan_step<IO, V, LG, K, M><<<(unsigned)blocks, NT, 0, st>>>(a, (int)tiles, gc);
    else scan_step<IO, V, LG, K, 1><<<(unsigned)blocks, NT, 0, st>>>(a, (int)tiles, gc);
    return cudaGetLastError();
}

template <typename IO>
cudaError_t pick(const dfsnn_state_scan_step_args& a, cudaStream_t st) {
    const int n = a.states;
    auto vec = [](const void* p, long long stride) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 4 == 0;
    };
    // 16-byte accesses where every slot and channel starts on 16 bytes
    if (n % 4 == 0 && vec(a.state, a.state_s) && vec(a.state_out, a.out_s) && vec(a.A, 0)) {
        if (n <= 4) return launch<IO, 4, 1, 1>(a, st);
        if (n <= 8) return launch<IO, 4, 2, 1>(a, st);
        if (n <= 16) return launch<IO, 4, 4, 1>(a, st);
        if (n <= 32) return launch<IO, 4, 8, 1>(a, st);
        if (n <= 64) return launch<IO, 4, 16, 1>(a, st);
        return launch<IO, 4, 32, 1>(a, st);
    }
    if (n <= 4) return launch<IO, 1, 4, 1>(a, st);
    if (n <= 16) return launch<IO, 1, 16, 1>(a, st);
    if (n <= 32) return launch<IO, 1, 32, 1>(a, st);
    return launch<IO, 1, 32, 4>(a, st);
}

}  // namespace

cudaError_t state_scan_step_launch(const dfsnn_state_scan_step_args& a, cudaStream_t st) {
    switch (a.dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(a, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(a, st);
        default: return pick<float>(a, st);
    }
}

}  // namespace dfsnn
