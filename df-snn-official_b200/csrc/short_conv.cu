// short_conv.cu -- short causal convolution per channel: forward, backward, one token.
//
//   p_t = bias + sum_j w_j x_(t-W+1+j),   y_t = p_t or p_t sigmoid(p_t)
//
// Every form reads its sequences once and writes once: bound by memory.  A warp takes 32 * V
// neighbouring channels (V elements make one 16-byte access where rows are aligned, else V = 1)
// and a run of steps, along which the last W - 1 inputs stay in registers; W is a template
// argument, so they do.  Sums are fp32; outputs are rounded once.
#include <algorithm>

#include "short_conv.h"

namespace dfsnn {
namespace {

constexpr int NT = 256, NW = NT / 32;

template <typename IO, int V>
struct Row {
    static __device__ __forceinline__ void load(float (&f)[V], const IO* p) {
        if constexpr (V == 1) {
            f[0] = to_f(*p);
        } else {
            IO r[V];
            if constexpr (sizeof(IO) * V == 16) *reinterpret_cast<uint4*>(r) = *reinterpret_cast<const uint4*>(p);
            else *reinterpret_cast<uint2*>(r) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = to_f(r[i]);
        }
    }
    static __device__ __forceinline__ void store(IO* p, const float (&f)[V]) {
        if constexpr (V == 1) {
            *p = from_f<IO>(f[0]);
        } else {
            IO r[V];
#pragma unroll
            for (int i = 0; i < V; ++i) r[i] = from_f<IO>(f[i]);
            if constexpr (sizeof(IO) * V == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(r);
            else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(r);
        }
    }
    static __device__ __forceinline__ void zero(float (&f)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = 0.0f;
    }
};

// Input of ext step t (t < 0: the state in front of the sequence), zero outside [-(W-1), len)
template <typename IO, int V, int W>
__device__ __forceinline__ void load_x(float (&f)[V], const IO* x, long long x_t, const IO* state,
                                       long long channels, long long t, long long len) {
    if (t >= 0 && t < len) Row<IO, V>::load(f, x + t * x_t);
    else if (t < 0 && t >= 1 - W && state) Row<IO, V>::load(f, state + (t + W - 1) * channels);
    else Row<IO, V>::zero(f);
}

template <typename IO, int V, int W>
__global__ void __launch_bounds__(NT) conv_fwd(const ConvParams p) {
    const dfsnn_short_conv_args& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = (long long)(blockIdx.x / p.channel_blocks) * NW + warp;
    const long long c = ((long long)(blockIdx.x % p.channel_blocks) * 32 + lane) * V;
    if (item >= p.items || c >= a.channels) return;
    const long long b = item / p.runs, t0 = item % p.runs * p.run;
    const long long len = seq_length(a.lengths, a.lengths64, b, (int)a.T);
    const IO* x = static_cast<const IO*>(a.x) + b * a.x_b + c;
    const IO* state = a.state ? static_cast<const IO*>(a.state) + b * (W - 1) * a.channels + c : nullptr;
    IO* y = static_cast<IO*>(a.y) + b * a.y_b + c;

    float w[V][W], bias[V], win[W][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = a.bias ? a.bias[c + i] : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = a.weight[(c + i) * W + j];
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
        load_x<IO, V, W>(win[j + 1], x, a.x_t, state, a.channels, t0 - (W - 1) + j, len);

    const long long t1 = t0 + p.run < a.T ? t0 + p.run : a.T;
    constexpr int U = 4;                        // steps loaded ahead
    for (long long t = t0; t < t1; t += U) {
        float in[U][V];
#pragma unroll
        for (int k = 0; k < U; ++k)
            load_x<IO, V, W>(in[k], x, a.x_t, nullptr, 0, t + k, t1 < len ? t1 : len);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
                win[W - 1][i] = in[k][i];
                float s = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) s = fmaf(w[i][j], win[j][i], s);
                o[i] = t + k >= len ? 0.0f : (a.silu ? s * sigmoid_f(s) : s);
            }
            if (t + k < t1) Row<IO, V>::store(y + (t + k) * a.y_t, o);
        }
    }
    if (a.last && t0 == 0) {
        IO* last = static_cast<IO*>(a.last) + b * (W - 1) * a.channels + c;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            float f[V];
            load_x<IO, V, W>(f, x, a.x_t, state, a.channels, len - (W - 1) + j, len);
            Row<IO, V>::store(last + j * a.channels, f);
        }
    }
}

// gp_t = gy_t act'(p_t);  grad x_s = sum_j w_j gp_(s+W-1-j);  grad w_j = sum gp_t x_(t-W+1+j).
// Walking forwards, gp_t completes the gradient of step s = t - (W - 1); a run therefore goes
// W - 1 steps past its end, and the first run starts at the state (s = -(W - 1)).
template <typename IO, int V, int W>
__global__ void __launch_bounds__(NT) conv_bwd(const ConvParams p) {
    __shared__ float s_sum[NW][32 * V];
    const dfsnn_short_conv_args& a = p.a;
    const dfsnn_short_conv_grads& g = p.g;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = blockIdx.x / p.channel_blocks;
    const long long c = ((long long)(blockIdx.x % p.channel_blocks) * 32 + lane) * V;
    const bool c_ok = c < a.channels;
    float w[V][W], bias[V], gw[V][W], gb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = c_ok && a.bias ? a.bias[c + i] : 0.0f;
        gb[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            w[i][j] = c_ok ? a.weight[(c + i) * W + j] : 0.0f;
            gw[i][j] = 0.0f;
        }
    }
    for (long long item = (long long)part * NW + warp; c_ok && item < p.items;
         item += (long long)p.parts * NW) {
        const long long b = item / p.runs, t0 = item % p.runs * p.run;
        const long long t1 = t0 + p.run < a.T ? t0 + p.run : a.T;
        const long long len = seq_length(a.lengths, a.lengths64, b, (int)a.T);
        const IO* x = static_cast<const IO*>(a.x) + b * a.x_b + c;
        const IO* state = a.state ? static_cast<const IO*>(a.state) + b * (W - 1) * a.channels + c : nullptr;
        const IO* gy = static_cast<const IO*>(g.grad_y) + b * a.y_b + c;
        const IO* glast = g.grad_last ? static_cast<const IO*>(g.grad_last) + b * (W - 1) * a.channels + c : nullptr;
        IO* gx = static_cast<IO*>(g.grad_x) + b * g.gx_b + c;
        IO* gstate = g.grad_state ? static_cast<IO*>(g.grad_state) + b * (W - 1) * a.channels + c : nullptr;
        float win[W][V], gp[W][V];              // x_(t-W+1 .. t), gp_(t-W+1 .. t)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            Row<IO, V>::zero(gp[j]);
            if (j > 0) load_x<IO, V, W>(win[j], x, a.x_t, state, a.channels, t0 - W + j, len);
        }
        // Steps of this run: gp from t0; the gradients complete from t0 on (from -(W-1) in the
        // first run), the last W - 1 of them only with the next run's gp.
        const long long end = t1 + W - 1;
        constexpr int U = 4;
        for (long long t = t0; t < end; t += U) {
            float in[U][V], gin[U][V];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const long long lim = end < len ? end : len;
                load_x<IO, V, W>(in[k], x, a.x_t, nullptr, 0, t + k, lim);
                if (t + k < lim) Row<IO, V>::load(gin[k], gy + (t + k) * a.y_t);
                else Row<IO, V>::zero(gin[k]);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const bool mine = t + k < t1;   // sums of the parameters: each step once
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        win[j][i] = win[j + 1][i];
                        gp[j][i] = gp[j + 1][i];
                    }
                    win[W - 1][i] = in[k][i];
                    float v = gin[k][i];
                    if (a.silu) {
                        float s = bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) s = fmaf(w[i][j], win[j][i], s);
                        const float sg = sigmoid_f(s);
                        v *= fmaf(s * sg, 1.0f - sg, sg);
                    }
                    if (t + k >= len) v = 0.0f;
                    gp[W - 1][i] = v;
                    if (mine) {
                        gb[i] += v;
#pragma unroll
                        for (int j = 0; j < W; ++j) gw[i][j] = fmaf(v, win[j][i], gw[i][j]);
                    }
                    float s = 0.0f;
#pragma unroll
                    for (int j = 0; j < W; ++j) s = fmaf(w[i][j], gp[W - 1 - j][i], s);
                    o[i] = s;
                }
                const long long s = t + k - (W - 1);
                if (s >= (t0 == 0 ? 1 - W : t0) && s < t1) {
                    if (glast && s >= len - (W - 1) && s < len) {
                        float f[V];
                        Row<IO, V>::load(f, glast + (s - (len - (W - 1))) * a.channels);
#pragma unroll
                        for (int i = 0; i < V; ++i) o[i] += f[i];
                    }
                    if (s >= 0) {
                        if (s >= len) Row<IO, V>::zero(o);
                        Row<IO, V>::store(gx + s * g.gx_t, o);
                    } else if (gstate) {
                        Row<IO, V>::store(gstate + (s + W - 1) * a.channels, o);
                    }
                }
            }
        }
    }
    // over the warps of the block, in order; then one row of parts for the block
    for (int j = 0; j <= W; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float v = gb[i];
#pragma unroll
            for (int q = 0; q < W; ++q) v = j == q ? gw[i][q] : v;
            s_sum[warp][lane * V + i] = v;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * V; i += NT) {
            const long long cc = (long long)(blockIdx.x % p.channel_blocks) * 32 * V + i;
            if (cc < a.channels) {
                float v = 0.0f;
#pragma unroll
                for (int q = 0; q < NW; ++q) v += s_sum[q][i];
                p.part[((long long)part * (W + 1) + j) * a.channels + cc] = v;
            }
        }
    }
}

// grad weight and grad bias from the blocks' parts: a warp for 32 / 8 outputs ... in a fixed order
__global__ void conv_bwd_sums(const ConvParams p, int W) {
    const long long total = p.a.channels * (W + 1);
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const long long j = i / p.a.channels, c = i % p.a.channels;
    float v = 0.0f;
    for (int q = 0; q < p.parts; ++q) v += p.part[q * total + i];
    if (j < W) p.g.grad_weight[c * W + j] = v;
    else if (p.g.grad_bias) p.g.grad_bias[c] = v;
}

template <typename IO, int V, int W>
__global__ void __launch_bounds__(128) conv_step(const dfsnn_short_conv_step_args a, int tiles) {
    const long long b = blockIdx.x / tiles;
    const long long c = ((long long)(blockIdx.x % tiles) * 128 + threadIdx.x) * V;
    const long long slot = step_slot(a.index, a.index64, b, a.slots);
    if (c >= a.channels) return;
    IO* y = static_cast<IO*>(a.y) + b * a.y_b + c;
    float o[V];
    if (slot < 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = slot == kIdle ? 0.0f : __int_as_float(0x7fc00000);
        Row<IO, V>::store(y, o);
        return;
    }
    const IO* in = static_cast<const IO*>(a.state) + slot * a.state_s + c;
    IO* out = static_cast<IO*>(a.state_out) + slot * a.out_s + c;
    float win[W][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) Row<IO, V>::load(win[j], in + j * a.channels);
    Row<IO, V>::load(win[W - 1], static_cast<const IO*>(a.x) + b * a.x_b + c);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float s = a.bias ? a.bias[c + i] : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) s = fmaf(a.weight[(c + i) * W + j], win[j][i], s);
        o[i] = a.silu ? s * sigmoid_f(s) : s;
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) Row<IO, V>::store(out + j * a.channels, win[j + 1]);
    Row<IO, V>::store(y, o);
}

// Whether rows of this tensor can be read V elements at a time
bool rows_fit(const void* p, size_t bytes, std::initializer_list<long long> strides, int elem) {
    if (p == nullptr) return true;
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    for (long long s : strides)
        if (s * elem % (long long)bytes) return false;
    return true;
}

enum class Form { kForward, kBackward, kStep };

template <typename IO, int V, int W>
cudaError_t launch(Form form, ConvParams& p, const dfsnn_short_conv_step_args* s, cudaStream_t st) {
    if (form == Form::kStep) {
        const long long tiles = (s->channels + 128 * V - 1) / (128 * V), blocks = tiles * s->batch;
        if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
        conv_step<IO, V, W><<<(unsigned)blocks, 128, 0, st>>>(*s, (int)tiles);
        return cudaGetLastError();
    }
    p.channel_blocks = (int)((p.a.channels + 32 * V - 1) / (32 * V));
    if (form == Form::kForward) {
        const long long blocks = (p.items + NW - 1) / NW * p.channel_blocks;
        if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
        conv_fwd<IO, V, W><<<(unsigned)blocks, NT, 0, st>>>(p);
        return cudaGetLastError();
    }
    const long long blocks = (long long)p.parts * p.channel_blocks;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    conv_bwd<IO, V, W><<<(unsigned)blocks, NT, 0, st>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const long long total = p.a.channels * (W + 1);
    conv_bwd_sums<<<(unsigned)((total + 127) / 128), 128, 0, st>>>(p, W);
    return cudaGetLastError();
}

template <typename IO, int V>
cudaError_t pick_taps(Form form, ConvParams& p, const dfsnn_short_conv_step_args* s, cudaStream_t st) {
    switch (form == Form::kStep ? s->taps : p.a.taps) {
        case 1: return launch<IO, V, 1>(form, p, s, st);
        case 2: return launch<IO, V, 2>(form, p, s, st);
        case 3: return launch<IO, V, 3>(form, p, s, st);
        case 4: return launch<IO, V, 4>(form, p, s, st);
        case 5: return launch<IO, V, 5>(form, p, s, st);
        case 6: return launch<IO, V, 6>(form, p, s, st);
        case 7: return launch<IO, V, 7>(form, p, s, st);
        default: return launch<IO, V, 8>(form, p, s, st);
    }
}

template <typename IO>
cudaError_t pick(Form form, ConvParams& p, const dfsnn_short_conv_step_args* s, cudaStream_t st) {
    constexpr int V = 4, E = (int)sizeof(IO);
    const size_t B = V * sizeof(IO);
    bool fit;
    if (form == Form::kStep) {
        fit = s->channels % V == 0 && rows_fit(s->x, B, {s->x_b}, E) && rows_fit(s->y, B, {s->y_b}, E)
              && rows_fit(s->state, B, {s->state_s}, E) && rows_fit(s->state_out, B, {s->out_s}, E);
    } else {
        fit = p.a.channels % V == 0 && rows_fit(p.a.x, B, {p.a.x_t, p.a.x_b}, E)
              && rows_fit(p.a.state, B, {}, E);
        if (form == Form::kForward)
            fit = fit && rows_fit(p.a.y, B, {p.a.y_t, p.a.y_b}, E) && rows_fit(p.a.last, B, {}, E);
        else
            fit = fit && rows_fit(p.g.grad_y, B, {p.a.y_t, p.a.y_b}, E)
                  && rows_fit(p.g.grad_x, B, {p.g.gx_t, p.g.gx_b}, E)
                  && rows_fit(p.g.grad_last, B, {}, E) && rows_fit(p.g.grad_state, B, {}, E);
    }
    return fit ? pick_taps<IO, V>(form, p, s, st) : pick_taps<IO, 1>(form, p, s, st);
}

cudaError_t run(Form form, int dtype, ConvParams& p, const dfsnn_short_conv_step_args* s, cudaStream_t st) {
    switch (dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(form, p, s, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(form, p, s, st);
        default: return pick<float>(form, p, s, st);
    }
}

// Runs of up to 32 steps: the W - 1 rows that a run reads twice stay few
void set_runs(ConvParams& p) {
    p.run = 32;
    p.runs = (p.a.T + p.run - 1) / p.run;
    p.items = p.runs * p.a.batch;
}

}  // namespace

cudaError_t short_conv_forward_launch(const dfsnn_short_conv_args& a, cudaStream_t st) {
    ConvParams p{};
    p.a = a;
    set_runs(p);
    return run(Form::kForward, a.dtype, p, nullptr, st);
}

// Rows of partial sums: blocks that share the (sequence, run) items, 8 blocks an SM at most
int short_conv_parts(long long T, long long batch, long long channels) {
    ConvParams p{};
    p.a.T = T;
    p.a.batch = batch;
    set_runs(p);
    const long long blocks = (p.items + NW - 1) / NW, cb = (channels + 127) / 128;
    return (int)std::max<long long>(1, std::min(blocks, (148 * 8 + cb - 1) / cb));
}

cudaError_t short_conv_backward_launch(const dfsnn_short_conv_args& a, const dfsnn_short_conv_grads& g,
                                       float* part, cudaStream_t st) {
    ConvParams p{};
    p.a = a;
    p.g = g;
    p.part = part;
    p.parts = short_conv_parts(a.T, a.batch, a.channels);
    set_runs(p);
    return run(Form::kBackward, a.dtype, p, nullptr, st);
}

cudaError_t short_conv_step_launch(const dfsnn_short_conv_step_args& a, cudaStream_t st) {
    ConvParams p{};
    return run(Form::kStep, a.dtype, p, &a, st);
}

}  // namespace dfsnn
