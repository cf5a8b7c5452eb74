// state_step.cu -- one token of the selective scan for each row of a batch.
//
//   h[n] = exp(d A[n]) h[n] + d u B[n],   y = (sum_n C[n] h[n] + D u) * gate
//
// The state goes in and out once (8 bytes for each state), everything else is N times smaller:
// a large batch is bound by memory and a small one by the launch.  A channel's N states are spread
// over LG lanes with V neighbouring states each, so a warp reads and writes whole lines.
#include "state_space.cuh"

namespace dfsnn {
namespace {

constexpr int NT = 128;

// K groups of V states a lane: n = (k * LG + sl) * V + i
template <typename IO, int V, int LG, int K>
__global__ void __launch_bounds__(NT) scan_step(const dfsnn_state_scan_step_args a, int tiles,
                                                int group_channels) {
    constexpr int BC = NT / LG;
    const int tid = threadIdx.x, sl = tid % LG;
    const long long b = blockIdx.x / tiles;
    const long long c = (long long)(blockIdx.x % tiles) * BC + tid / LG;
    const bool c_ok = c < a.channels;
    const long long slot = step_slot(a.index, a.index64, b, a.slots);
    IO* y_p = static_cast<IO*>(a.y) + b * a.y_b + c;
    if (slot < 0) {
        if (c_ok && sl == 0) *y_p = from_f<IO>(slot == kIdle ? 0.0f : __int_as_float(0x7fc00000));
        return;
    }
    float h[K][V], acc = 0.0f, u = 0.0f, skip = 0.0f, z = 0.0f;
    const long long grp = c_ok ? c / group_channels : 0;
    if (c_ok) {
        const float* h_p = a.state + slot * a.state_s + c * a.states;
        const float* A_p = a.A + c * a.states;
        const IO* B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g;
        const IO* C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g;
        float A[K][V], Bv[K][V], Cv[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int n = (k * LG + sl) * V;
            if (n < a.states) {
                if constexpr (V == 4) {
                    *reinterpret_cast<float4*>(h[k]) = *reinterpret_cast<const float4*>(h_p + n);
                    *reinterpret_cast<float4*>(A[k]) = __ldg(reinterpret_cast<const float4*>(A_p + n));
                } else {
                    h[k][0] = h_p[n];
                    A[k][0] = A_p[n];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    Bv[k][i] = to_f(B_p[n + i]);
                    Cv[k][i] = to_f(C_p[n + i]);
                }
            }
        }
        u = to_f(static_cast<const IO*>(a.u)[b * a.u_b + c]);
        float dt = to_f(static_cast<const IO*>(a.delta)[b * a.delta_b + c]);
        skip = a.D ? a.D[c] : 0.0f;
        z = a.z ? to_f(static_cast<const IO*>(a.z)[b * a.z_b + c]) : 0.0f;
        if (a.delta_bias) dt += a.delta_bias[c];
        if (a.softplus) dt = softplus_f(dt);
        const float du = dt * u;
        float* o_p = a.state_out + slot * a.out_s + c * a.states;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int n = (k * LG + sl) * V;
            if (n < a.states) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    h[k][i] = fmaf(exp2_approx(dt * (A[k][i] * kLog2e)), h[k][i], du * Bv[k][i]);
                    acc = fmaf(Cv[k][i], h[k][i], acc);
                }
                if constexpr (V == 4) *reinterpret_cast<float4*>(o_p + n) = *reinterpret_cast<float4*>(h[k]);
                else o_p[n] = h[k][0];
            }
        }
    }
#pragma unroll
    for (int m = LG / 2; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (c_ok && sl == 0) {
        float o = fmaf(skip, u, acc);
        if (a.z) o *= z * sigmoid_f(z);
        *y_p = from_f<IO>(o);
    }
}

template <typename IO, int V, int LG, int K>
cudaError_t launch(const dfsnn_state_scan_step_args& a, cudaStream_t st) {
    const long long tiles = (a.channels + NT / LG - 1) / (NT / LG), blocks = tiles * a.batch;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    scan_step<IO, V, LG, K><<<(unsigned)blocks, NT, 0, st>>>(a, (int)tiles,
                                                            (int)(a.channels / a.groups));
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
