// short_conv.cu -- short causal convolution per channel: forward, backward, one token.
//
//   p_t = bias + sum_j w_j x_(t-W+1+j),   y_t = p_t or p_t sigmoid(p_t)
//
// Every form reads its sequences once and writes once: bound by memory.  A warp takes 32 * V
// neighbouring channels (V elements make one 16- or 8-byte access where rows are aligned) and a run
// of steps, along which the last W - 1 inputs stay in registers; W is a template argument, so they
// do.  The next 8 to 16 steps are on their way meanwhile, through a ring in shared memory of which
// each thread copies and reads its own part (no barriers, no registers), and the arithmetic is
// packed by pairs of channels.  Sums are fp32; outputs are rounded once.  bf16, 4 taps, silu: forward
// 8192 x 2 x 4096 55 us (4.9 TB/s of the 6.55 that a copy reaches), 2048 x 8 x 2048 34 us; backward of
// the latter 70 us (2.9 TB/s; 128 registers keep it at 16 warps an SM).
#include <algorithm>

#include "short_conv.h"
#include "state_tile.cuh"

namespace dfsnn {
namespace {

constexpr int NT = 256, NW = NT / 32;

// V neighbouring elements of a row, as they come and as pairs of floats (V = 1: one of the pair)
template <typename IO, int V>
struct __align__(V * sizeof(IO) > 16 ? 16 : V * sizeof(IO)) Row {
    IO v[V];
    static constexpr int P = (V + 1) / 2;
    __device__ __forceinline__ void get(float2 (&f)[P]) const {
#pragma unroll
        for (int i = 0; i < P; ++i) f[i] = make_float2(to_f(v[2 * i]), V == 1 ? 0.0f : to_f(v[V == 1 ? 0 : 2 * i + 1]));
    }
    __device__ __forceinline__ void set(const float2 (&f)[P]) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = from_f<IO>(i % 2 ? f[i / 2].y : f[i / 2].x);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = from_f<IO>(0.0f);
    }
};

__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }

// Input of step t: of the sequence, of the state in front of it (t < 0), or zero
template <typename IO, int V, int W>
__device__ __forceinline__ Row<IO, V> load_x(const IO* x, long long x_t, const IO* state, long long channels,
                                             long long t, long long len) {
    Row<IO, V> r;
    if (t >= 0 && t < len) r = *reinterpret_cast<const Row<IO, V>*>(x + t * x_t);
    else if (t < 0 && t >= 1 - W && state) r = *reinterpret_cast<const Row<IO, V>*>(state + (t + W - 1) * channels);
    else r.zero();
    return r;
}

// A thread's next rows of one sequence, asynchronously, G rows a group.  A row is fetched into the
// slot that it is read from; the slots of a group are filled again after its last use.
constexpr int G = 4;
template <typename IO, int V>
struct Ring {
    using R = Row<IO, V>;
    static constexpr int kBytes = (int)sizeof(R), kGroups = kBytes > 8 ? 2 : 4;
    static constexpr size_t kSize = (size_t)kGroups * G * NT * kBytes;       // for the block
    R* mine;
    __device__ __forceinline__ Ring(void* smem) : mine(static_cast<R*>(smem) + threadIdx.x) {}
    __device__ __forceinline__ R* at(int slot, int k) const { return mine + (slot * G + k) * NT; }
    __device__ __forceinline__ void fetch(int slot, int k, const IO* src, bool ok) const {
        if constexpr (kBytes >= 4) {
            copy_async<kBytes>(at(slot, k), src, ok ? kBytes : 0);     // 0: nothing is read
        } else {
            R r;
            r.zero();
            if (ok) r = *reinterpret_cast<const R*>(src);
            *at(slot, k) = r;
        }
    }
};

// Weights as pairs of channels: w[i][j] for channels 2i, 2i + 1.  Those of V = 4 channels are W
// 16-byte accesses (fits() has seen to it).
template <int V, int W>
__device__ __forceinline__ void load_weights(float2 (&w)[(V + 1) / 2][W], float2 (&bias)[(V + 1) / 2],
                                             const float* weight, const float* b, long long c) {
    float f[V * W], g[V];
    if constexpr (V == 4) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            *reinterpret_cast<float4*>(f + 4 * i) = __ldg(reinterpret_cast<const float4*>(weight + c * W) + i);
        const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        *reinterpret_cast<float4*>(g) = b ? __ldg(reinterpret_cast<const float4*>(b + c)) : none;
    } else {
#pragma unroll
        for (int i = 0; i < V * W; ++i) f[i] = weight[c * W + i];
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = b ? b[c + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) {
        const int o = V == 1 ? 0 : 2 * i + 1;
        bias[i] = make_float2(g[2 * i], g[o]);
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = make_float2(f[2 * i * W + j], f[o * W + j]);
    }
}

template <typename IO, int V, int W>
__global__ void __launch_bounds__(NT, W <= 4 ? 3 : 1) conv_fwd(const ConvParams p) {
    constexpr int P = (V + 1) / 2;
    using R = Row<IO, V>;
    const dfsnn_short_conv_args& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = (long long)(blockIdx.x / p.channel_blocks) * NW + warp;
    const long long c = ((long long)(blockIdx.x % p.channel_blocks) * 32 + lane) * V;
    if (item >= p.items || c >= a.channels) return;
    const long long b = item / p.runs;
    const int t0 = (int)(item % p.runs * p.run), T = (int)a.T;     // steps fit 32 bits, offsets do not
    const int len = seq_length(a.lengths, a.lengths64, b, T);
    const IO* x = static_cast<const IO*>(a.x) + b * a.x_b + c;
    const IO* state = a.state ? static_cast<const IO*>(a.state) + b * (W - 1) * a.channels + c : nullptr;
    IO* y = static_cast<IO*>(a.y) + b * a.y_b + c;
    const int run = (int)p.run, t1 = T - t0 > run ? t0 + run : T;
    const int lim = t1 < len ? t1 : len;

    extern __shared__ __align__(16) unsigned char smem[];
    const Ring<IO, V> ring(smem);
    constexpr int N = Ring<IO, V>::kGroups;
    const IO* ahead = x + t0 * a.x_t;           // next row to fetch
    int t_ahead = t0;
    auto fetch = [&](int slot) {
#pragma unroll
        for (int k = 0; k < G; ++k) {
            ring.fetch(slot, k, ahead, t_ahead + k < lim);
            ahead += a.x_t;
        }
        t_ahead += G;
        copy_commit();
    };
#pragma unroll
    for (int n = 0; n < N; ++n) fetch(n);
    float2 w[P][W], bias[P], win[W][P];
#pragma unroll
    for (int j = 1; j < W; ++j) load_x<IO, V, W>(x, a.x_t, state, a.channels, t0 - W + j, len).get(win[j]);
    load_weights<V, W>(w, bias, a.weight, a.bias, c);
    IO* yt = y + t0 * a.y_t;
    int slot = 0;
    for (int t = t0; t < t1; t += G) {
        copy_wait<N - 1>();
        const bool inner = t + G <= lim;        // all of them in the run and in the sequence
#pragma unroll
        for (int k = 0; k < G; ++k) {
            float2 f[P], o[P];
            ring.at(slot, k)->get(f);
#pragma unroll
            for (int i = 0; i < P; ++i) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
                win[W - 1][i] = f[i];
                float2 s = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) s = __ffma2_rn(w[i][j], win[j][i], s);
                o[i] = a.silu ? __fmul2_rn(s, sigmoid_f(s)) : s;
            }
            if (inner || t + k < t1) {
                R out;
                out.set(o);
                if (!inner && t + k >= len) out.zero();
                *reinterpret_cast<R*>(yt) = out;
            }
            yt += a.y_t;
        }
        fetch(slot);
        slot = slot + 1 == N ? 0 : slot + 1;
    }
    if (a.last && t0 == 0) {
        IO* last = static_cast<IO*>(a.last) + b * (W - 1) * a.channels + c;
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            *reinterpret_cast<R*>(last + j * a.channels) =
                load_x<IO, V, W>(x, a.x_t, state, a.channels, len - (W - 1) + j, len);
    }
}

// gp_t = gy_t act'(p_t);  grad x_s = sum_j w_j gp_(s+W-1-j);  grad w_j = sum gp_t x_(t-W+1+j).
// Walking forwards, gp_t completes the gradient of step s = t - (W - 1); a run therefore goes
// W - 1 steps past its end, and the first run starts at the state (s = -(W - 1)).
template <typename IO, int V, int W>
__global__ void __launch_bounds__(NT, W <= 4 ? 2 : 1) conv_bwd(const ConvParams p) {
    constexpr int P = (V + 1) / 2;
    using R = Row<IO, V>;
    __shared__ float s_sum[NW][32 * V];
    extern __shared__ __align__(16) unsigned char smem[];
    const Ring<IO, V> ring(smem), gring(smem + Ring<IO, V>::kSize);
    constexpr int N = Ring<IO, V>::kGroups;
    const dfsnn_short_conv_args& a = p.a;
    const dfsnn_short_conv_grads& g = p.g;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = blockIdx.x / p.channel_blocks;
    const long long c = ((long long)(blockIdx.x % p.channel_blocks) * 32 + lane) * V;
    const bool c_ok = c < a.channels;
    float2 w[P][W] = {}, bias[P] = {}, gw[P][W] = {}, gb[P] = {};
    if (c_ok) load_weights<V, W>(w, bias, a.weight, a.bias, c);
    for (long long item = (long long)part * NW + warp; c_ok && item < p.items;
         item += (long long)p.parts * NW) {
        const long long b = item / p.runs;
        const int t0 = (int)(item % p.runs * p.run), T = (int)a.T, run = (int)p.run;
        const int t1 = T - t0 > run ? t0 + run : T;
        const int len = seq_length(a.lengths, a.lengths64, b, T);
        const IO* x = static_cast<const IO*>(a.x) + b * a.x_b + c;
        const IO* state = a.state ? static_cast<const IO*>(a.state) + b * (W - 1) * a.channels + c : nullptr;
        const IO* gy = static_cast<const IO*>(g.grad_y) + b * a.y_b + c;
        const IO* glast = g.grad_last ? static_cast<const IO*>(g.grad_last) + b * (W - 1) * a.channels + c : nullptr;
        IO* gstate = g.grad_state ? static_cast<IO*>(g.grad_state) + b * (W - 1) * a.channels + c : nullptr;
        // Steps of this run: gp from t0; the gradients complete from t0 on (from -(W-1) in the
        // first run), the last W - 1 of them only with the next run's gp.
        const int end = t1 + W - 1, lim = end < len ? end : len;
        const IO *ahead = x + t0 * a.x_t, *gahead = gy + t0 * a.y_t;    // next rows to fetch
        int t_ahead = t0;
        auto fetch = [&](int slot) {
#pragma unroll
            for (int k = 0; k < G; ++k) {
                ring.fetch(slot, k, ahead, t_ahead + k < lim);
                gring.fetch(slot, k, gahead, t_ahead + k < lim);
                ahead += a.x_t;
                gahead += a.y_t;
            }
            t_ahead += G;
            copy_commit();
        };
        copy_wait<0>();                         // what is left of the last run's fetches
#pragma unroll
        for (int n = 0; n < N; ++n) fetch(n);
        float2 win[W][P], gp[W][P] = {};        // x_(t-W+1 .. t), gp_(t-W+1 .. t)
#pragma unroll
        for (int j = 1; j < W; ++j) load_x<IO, V, W>(x, a.x_t, state, a.channels, t0 - W + j, len).get(win[j]);
        IO* gx = static_cast<IO*>(g.grad_x) + b * g.gx_b + c + (t0 - (W - 1)) * g.gx_t;
        const int inner_end = t1 < len ? t1 : len;
        int slot = 0;
        for (int t = t0; t < end; t += G) {
            copy_wait<N - 1>();
            // gp and the completed gradients all in the run and in the sequence
            const bool inner = t >= t0 + W - 1 && t + G <= inner_end;
#pragma unroll
            for (int k = 0; k < G; ++k) {
                float2 f[P], v[P], o[P];
                ring.at(slot, k)->get(f);
                gring.at(slot, k)->get(v);
#pragma unroll
                for (int i = 0; i < P; ++i) {
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        win[j][i] = win[j + 1][i];
                        gp[j][i] = gp[j + 1][i];
                    }
                    win[W - 1][i] = f[i];
                    if (a.silu) {
                        float2 s = bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) s = __ffma2_rn(w[i][j], win[j][i], s);
                        const float2 sg = sigmoid_f(s), si = __fmul2_rn(s, sg);
                        // silu' = sg + si (1 - sg)
                        v[i] = __fmul2_rn(v[i], __ffma2_rn(si, __ffma2_rn(sg, two(-1.0f), two(1.0f)), sg));
                    }
                    if (!inner && t + k >= lim) v[i] = two(0.0f);
                    gp[W - 1][i] = v[i];
                    if (inner || t + k < t1) {  // sums of the parameters: each step in one run only
                        gb[i] = __fadd2_rn(gb[i], v[i]);
#pragma unroll
                        for (int j = 0; j < W; ++j) gw[i][j] = __ffma2_rn(v[i], win[j][i], gw[i][j]);
                    }
                    float2 s = __fmul2_rn(w[i][0], gp[W - 1][i]);
#pragma unroll
                    for (int j = 1; j < W; ++j) s = __ffma2_rn(w[i][j], gp[W - 1 - j][i], s);
                    o[i] = s;
                }
                R out;
                if (inner) {
                    out.set(o);
                    *reinterpret_cast<R*>(gx) = out;
                } else {
                    const int s = t + k - (W - 1);
                    if (s >= (t0 == 0 ? 1 - W : t0) && s < t1) {
                        if (glast && s >= len - (W - 1) && s < len) {
                            float2 l[P];
                            reinterpret_cast<const R*>(glast + (s - (len - (W - 1))) * a.channels)->get(l);
#pragma unroll
                            for (int i = 0; i < P; ++i) o[i] = __fadd2_rn(o[i], l[i]);
                        }
                        out.set(o);
                        if (s >= 0) {
                            if (s >= len) out.zero();
                            *reinterpret_cast<R*>(gx) = out;
                        } else if (gstate) {
                            *reinterpret_cast<R*>(gstate + (s + W - 1) * a.channels) = out;
                        }
                    }
                }
                gx += g.gx_t;
            }
            fetch(slot);
            slot = slot + 1 == N ? 0 : slot + 1;
        }
    }
    copy_wait<0>();
    // over the warps of the block, in order; then one row of parts for the block
#pragma unroll
    for (int j = 0; j <= W; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 v = j < W ? gw[i / 2][j < W ? j : 0] : gb[i / 2];
            s_sum[warp][lane * V + i] = i % 2 ? v.y : v.x;
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

// grad weight and grad bias from the blocks' parts, 32 outputs a block: its 8 warps add every eighth
// part, then the warps' sums are added in order
__global__ void __launch_bounds__(NT) conv_bwd_sums(const ConvParams p, int W) {
    __shared__ float s_sum[NW][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long total = p.a.channels * (W + 1), i = (long long)blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (i < total) {
#pragma unroll 4
        for (int q = warp; q < p.parts; q += NW) v += p.part[q * total + i];
    }
    s_sum[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && i < total) {
        v = 0.0f;
        for (int q = 0; q < NW; ++q) v += s_sum[q][lane];
        const long long j = i / p.a.channels, c = i % p.a.channels;
        if (j < W) p.g.grad_weight[c * W + j] = v;
        else if (p.g.grad_bias) p.g.grad_bias[c] = v;
    }
}

template <typename IO, int V, int W>
__global__ void __launch_bounds__(128) conv_step(const dfsnn_short_conv_step_args a, int tiles) {
    const long long b = blockIdx.x / tiles;
    const long long c = ((long long)(blockIdx.x % tiles) * 128 + threadIdx.x) * V;
    using R = Row<IO, V>;
    constexpr int P = R::P;
    long long slot = step_slot(a.index, a.index64, b, a.slots);
    const bool ours = slot >= 0, c_ok = c < a.channels;
    const IO* in = static_cast<const IO*>(a.state) + slot * a.state_s + c;      // not read unless the slot is one
    IO* out = static_cast<IO*>(a.state_out) + slot * a.out_s + c;
    R* y = reinterpret_cast<R*>(static_cast<IO*>(a.y) + b * a.y_b + c);
    R row[W];
    if (ours && c_ok) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) row[j] = *reinterpret_cast<const R*>(in + j * a.channels);
        row[W - 1] = *reinterpret_cast<const R*>(static_cast<const IO*>(a.x) + b * a.x_b + c);
    }
    if (taken_before(a.index, a.index64, b, slot) && ours) slot = kBad;
    if (!c_ok) return;
    if (slot < 0) {
        float2 o[P];
#pragma unroll
        for (int i = 0; i < P; ++i) o[i] = two(slot == kIdle ? 0.0f : __int_as_float(0x7fc00000));
        y->set(o);
        return;
    }
    float2 w[P][W], s[P];
    load_weights<V, W>(w, s, a.weight, a.bias, c);
#pragma unroll
    for (int j = 0; j < W; ++j) {
        float2 f[P];
        row[j].get(f);
#pragma unroll
        for (int i = 0; i < P; ++i) s[i] = __ffma2_rn(w[i][j], f[i], s[i]);
    }
    if (a.silu) {
#pragma unroll
        for (int i = 0; i < P; ++i) s[i] = __fmul2_rn(s[i], sigmoid_f(s[i]));
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) *reinterpret_cast<R*>(out + j * a.channels) = row[j + 1];
    R o;
    o.set(s);
    *y = o;
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
        static_assert(Ring<IO, V>::kSize <= 48 * 1024, "within the default");
        conv_fwd<IO, V, W><<<(unsigned)blocks, NT, Ring<IO, V>::kSize, st>>>(p);
        return cudaGetLastError();
    }
    const long long blocks = (long long)p.parts * p.channel_blocks;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    constexpr size_t smem = 2 * Ring<IO, V>::kSize;
    cudaError_t e = allow_shared<conv_bwd<IO, V, W>>(smem);
    if (e != cudaSuccess) return e;
    conv_bwd<IO, V, W><<<(unsigned)blocks, NT, smem, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const long long total = p.a.channels * (W + 1);
    conv_bwd_sums<<<(unsigned)((total + 31) / 32), NT, 0, st>>>(p, W);
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

// Whether every row of a call starts on a multiple of V elements
template <typename IO, int V>
bool fits(Form form, const ConvParams& p, const dfsnn_short_conv_step_args* s) {
    constexpr int E = (int)sizeof(IO);
    constexpr size_t B = V * sizeof(IO);
    const float *weight = form == Form::kStep ? s->weight : p.a.weight, *bias = form == Form::kStep ? s->bias : p.a.bias;
    if (V == 4 && ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias)) & 15)) return false;
    if (form == Form::kStep)
        return s->channels % V == 0 && rows_fit(s->x, B, {s->x_b}, E) && rows_fit(s->y, B, {s->y_b}, E)
               && rows_fit(s->state, B, {s->state_s}, E) && rows_fit(s->state_out, B, {s->out_s}, E);
    if (p.a.channels % V || !rows_fit(p.a.x, B, {p.a.x_t, p.a.x_b}, E) || !rows_fit(p.a.state, B, {}, E)) return false;
    if (form == Form::kForward)
        return rows_fit(p.a.y, B, {p.a.y_t, p.a.y_b}, E) && rows_fit(p.a.last, B, {}, E);
    return rows_fit(p.g.grad_y, B, {p.a.y_t, p.a.y_b}, E) && rows_fit(p.g.grad_x, B, {p.g.gx_t, p.g.gx_b}, E)
           && rows_fit(p.g.grad_last, B, {}, E) && rows_fit(p.g.grad_state, B, {}, E);
}

// 8-byte accesses (16 for fp32) where rows allow it, else pairs of channels, else single ones.
template <typename IO>
cudaError_t pick(Form form, ConvParams& p, const dfsnn_short_conv_step_args* s, cudaStream_t st) {
    if (fits<IO, 4>(form, p, s)) return pick_taps<IO, 4>(form, p, s, st);
    if (fits<IO, 2>(form, p, s)) return pick_taps<IO, 2>(form, p, s, st);
    return pick_taps<IO, 1>(form, p, s, st);
}

cudaError_t run(Form form, int dtype, ConvParams& p, const dfsnn_short_conv_step_args* s, cudaStream_t st) {
    switch (dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(form, p, s, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(form, p, s, st);
        default: return pick<float>(form, p, s, st);
    }
}

// Runs of 64 steps, or fewer (down to 8) where that would leave warps without work: the W - 1 rows
// that a run reads twice stay few.  bf16, 4 taps, forward: 2048 x 1 x 512 4.1 us in short runs
// against 13.8 in runs of 64, 4096 x 1 x 1024 8.3 against 14.0.
void set_runs(ConvParams& p) {
    const long long lanes = (p.a.channels + 127) / 128;
    p.run = 64;
    while (p.run > 8 && (p.a.T + p.run - 1) / p.run * p.a.batch * lanes < 148 * 32) p.run /= 2;
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
    p.a.channels = channels;
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
