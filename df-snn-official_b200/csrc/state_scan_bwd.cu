// state_scan_bwd.cu -- backward of the selective scan.
//
// With g_t the gradient of o_t (grad_y times the gate) and l_t that of h_t,
//   l_t = C_t g_t + a_(t+1) l_(t+1),   a_t = exp(d_t A),   q_t = a_t l_t h_(t-1)
//   grad C_t = sum_c g_t h_t     grad B_t = sum_c l_t d_t u_t     grad A = sum_(t,b) q_t d_t
//   grad u_t = d_t sum_n l_t B_t + D g_t      grad d_t = u_t sum_n l_t B_t + sum_n q_t A
// A warp walks the sequence of its channels backwards.  The forward kept the state in front of
// every 8 steps; from it the 8 steps' states and decays are formed again and stay in registers, so
// each exponential is taken once.  About 12 multiply-adds and one exponential for each (step,
// channel, state), and two kinds of sums: over states (a channel's SL lanes) and over channels (the
// other lanes; grad B and grad C), both formed for 4 steps at a time (LaneSums).  Packed pairs of
// states halve the arithmetic's issue slots; elementwise work is done once per (step, channel) by
// all threads.  The sums over channels go on over the warps in shared memory and over the blocks
// through partial sums that a second kernel adds in a fixed order: no atomic sums, so results do not
// change from run to run.
//
// Bound by instruction issue (58 % of the slots) and the shared-memory pipe (69 %) together, at
// three blocks an SM: T = 2048, 8 sequences, 2048 channels, bf16, N = 16: 893 us (the second kernel 30),
// 537 M (step, channel, state) at 0.60 T/s.  Four states on a lane and one channel: two channels a lane halve the
// shuffles of the sums over channels, but leave 8 warps an SM (1150 us).
#include <algorithm>
#include <type_traits>

#include "state_scan.h"
#include "state_tile.cuh"

namespace dfsnn {
namespace {

constexpr int TT = kScanTile, R = kScanChunk;
constexpr int Q = 4;                                 // steps whose sums over lanes are formed together
constexpr int NT = 128, NW = NT / 32;

// S states on each of a channel's SL lanes, C channels a lane
template <typename IO, int S, int SL, int C>
struct Tile {
    static constexpr int CL = 32 / SL;               // channel lanes of a warp
    static constexpr int CW = CL * C;                // channels of a warp
    static constexpr int BC = NW * CW;               // channels of the block
    static constexpr int NS = S * SL;                // states, padded
    struct Raw {                                     // as the sequences have them
        IO u[TT][BC], d[TT][BC], z[TT][BC], g[TT][BC], B[TT][NS], C_[TT][NS];
    };
    __align__(16) Raw raw[2];                        // this tile's and the next one's
    __align__(16) float B[TT][NS], C_[TT][NS];
    __align__(16) float red[NW][2][TT][NS];          // the warps' sums over channels (grad B, grad C)
    float2 d[BC][TT + 1];                            // (d, d u)
    float g[BC][TT + 1];                             // grad o
    float lb[BC][TT + 1], qa[BC][TT + 1], o[BC][TT + 1];    // sums over states
    // a thread's sums of grad A (pairs of states) and of grad D and delta_bias (a pack's channels),
    // added to after every tile: one fp32 register each for the many steps of many sequences that a
    // block takes lost digits (16 steps, 4096 sequences: grad A 4.2e-7 from 64 bits, now 2.1e-7)
    __align__(16) double2 sum_a[C * S / 2][NT], sum_d[2][NT];
    int place, ready;
};

template <int S>
__device__ __forceinline__ void load_states(float2 (&v)[S / 2], const float* q) {
    if constexpr (S == 4) {
        const float4 f = *reinterpret_cast<const float4*>(q);
        v[0] = make_float2(f.x, f.y);
        v[1] = make_float2(f.z, f.w);
    } else {
        v[0] = *reinterpret_cast<const float2*>(q);
    }
}
template <int S, int Q>
__device__ __forceinline__ void store_states(float* q, const float (&v)[S][Q], int i) {
    if constexpr (S == 4) *reinterpret_cast<float4*>(q) = make_float4(v[0][i], v[1][i], v[2][i], v[3][i]);
    else *reinterpret_cast<float2*>(q) = make_float2(v[0][i], v[1][i]);
}
__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }
__device__ __forceinline__ void add_to(double2& sum, float2 v) {
    sum = make_double2(sum.x + v.x, sum.y + v.y);
}

// V neighbouring elements of a sequence
template <typename IO, int V>
struct __align__(sizeof(IO) * V) Pack {
    IO v[V];
};
template <typename IO, int V>
__device__ __forceinline__ float2 unpack(const IO* q) {
    const Pack<IO, V> p = *reinterpret_cast<const Pack<IO, V>*>(q);
    return make_float2(to_f(p.v[0]), to_f(p.v[V - 1]));
}
template <typename IO, int V>
__device__ __forceinline__ void store(IO* q, float2 f) {
    Pack<IO, V> p;
    p.v[0] = from_f<IO>(f.x);
    if (V == 2) p.v[V - 1] = from_f<IO>(f.y);
    *reinterpret_cast<Pack<IO, V>*>(q) = p;
}

// The flag of a chain counts its finished parts.  A part can take as long as the `steps` behind it
// together (0.4 us a step); a poll takes 0.5 us at least, and a wait has 2^21 polls and 16 for each step.
// A wait that runs out all the same is counted, and the caller goes on with NaN, which reaches all that
// depends on it.
__device__ unsigned long long expired_waits;
__device__ __forceinline__ bool wait_at_least(const int* flag, int count, long long steps, int patience) {
    const long long polls = patience * ((1LL << 21) + 16 * steps);
    for (long long i = 0; i < polls; ++i) {
        int v;
        asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
        if (v >= count) return true;
        __nanosleep(200);
    }
    atomicAdd(&expired_waits, 1ULL);
    return false;
}
__device__ __forceinline__ void publish(int* flag, int count) {
    asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(flag), "r"(count) : "memory");
}

template <typename IO, int S, int SL, int C, bool WIDE>
__global__ void __launch_bounds__(NT, 3) scan_bwd(const ScanParams p) {
    using Tl = Tile<IO, S, SL, C>;
    constexpr int CL = Tl::CL, CW = Tl::CW, BC = Tl::BC, NS = Tl::NS, J = S / 2;
    constexpr int V = WIDE ? 2 : 1;                             // channels of a pack
    constexpr int ROW = BC / V;                                 // threads along a step's channels
    constexpr int E = TT * ROW > NT ? TT * ROW / NT : 1;        // packs of a thread,
    constexpr int TS = TT / E;                                  // this many steps apart
    extern __shared__ __align__(16) unsigned char smem[];
    Tl& sh = *reinterpret_cast<Tl*>(smem);
    const dfsnn_state_scan_args& a = p.a;
    const dfsnn_state_scan_grads& g = p.g;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned bid = blockIdx.x;
    unsigned chain = 0;                                         // (tile, group, sequence)
    int split = 0;
    if (p.chained) {
        // Places in the order in which the blocks start: all last parts, then all last but one, ...  A
        // part waits only for the next one of its sequence, whose place is in front of its own: that
        // block runs or has run.
        const unsigned chains = p.tiles * a.groups * p.batch_parts;
        if (tid == 0) sh.place = atomicAdd(p.places, 1);
        __syncthreads();
        bid = __reduce_max_sync(0xffffffffu, (unsigned)sh.place);      // one value for the warp, in a uniform register
        split = p.splits - 1 - (int)(bid / chains);
        bid = chain = bid % chains;
    }
    const int tile = (int)(bid % p.tiles);
    bid /= p.tiles;
    const int grp = (int)(bid % a.groups);
    bid /= a.groups;
    if (!p.chained) {
        split = (int)(bid % p.splits);
        bid /= p.splits;
    }
    const int batch_part = (int)bid;
    const int first = split * p.split_steps;                    // this part's steps: first .. stop - 1
    const int stop = p.T - first < p.split_steps ? p.T : first + p.split_steps;
    const int part = batch_part * p.splits + split, parts = p.batch_parts * p.splits;
    const int c_base = tile * BC, cols = p.group_channels - c_base;
    const long long g_base = (long long)grp * p.group_channels;

    // elementwise role: packs (step t_e + e * TS, channels ch .. ch + V - 1)
    const int ch = tid % ROW * V, t_e = tid / ROW;
    const bool ch_ok = ch < cols && t_e < TT;
    const long long chan = g_base + c_base + ch;
    float2 bias = two(0.0f), skip = two(0.0f);
    if (ch_ok && a.delta_bias) bias = make_float2(a.delta_bias[chan], a.delta_bias[chan + V - 1]);
    if (ch_ok && a.D) skip = make_float2(a.D[chan], a.D[chan + V - 1]);

    // recurrence role: states n0 .. n0 + S - 1 of channels cl + c * CL of the block
    const int sl = lane / CL, lc = lane % CL, cl = warp * CW + lc, n0 = sl * S;
    const long long crow = (long long)CL * a.states;
    // a lane's states are one access everywhere
    const bool whole = S == 4 && a.states % 4 == 0
                       && ((reinterpret_cast<uintptr_t>(a.kept) | reinterpret_cast<uintptr_t>(a.h0)) & 15) == 0;
    auto get = [&](const float* q, float2(&v)[C][J]) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float f = q && cl + c * CL < cols && n0 + s < a.states ? q[c * crow + s] : 0.0f;
                (s % 2 ? v[c][s / 2].y : v[c][s / 2].x) = f;
            }
    };
    auto put = [&](float* q, const float2(&v)[C][J]) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (cl + c * CL < cols && n0 + s < a.states) q[c * crow + s] = s % 2 ? v[c][s / 2].y : v[c][s / 2].x;
    };
    // each thread has its own; the first use by others is behind a barrier
    for (int i = 0; i < C * J; ++i) sh.sum_a[i][tid] = make_double2(0.0, 0.0);
    for (int i = 0; i < 2; ++i) sh.sum_d[i][tid] = make_double2(0.0, 0.0);
    float2 A2[C][J] = {};
    get(a.A + (g_base + c_base + cl) * a.states + n0, A2);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j) A2[c][j] = make_float2(log2_rate(A2[c][j].x), log2_rate(A2[c][j].y));

    for (long long b = batch_part; b < a.batch; b += p.batch_parts) {
        const int whole_len = seq_length(a.lengths, a.lengths64, b, p.T);
        const int len = whole_len < stop ? whole_len : stop;
        const int top = len > first ? (len - 1) / TT * TT : -1; // first step of the last tile
        IO* gu_p = static_cast<IO*>(g.grad_u) + b * g.gu_b + chan + t_e * g.gu_t;
        IO* gd_p = static_cast<IO*>(g.grad_delta) + b * g.gdelta_b + chan + t_e * g.gdelta_t;
        IO* gz_p = static_cast<IO*>(g.grad_z) + b * g.gz_b + chan + t_e * g.gz_t;
        const long long row = ((long long)b * a.channels + g_base + c_base + cl) * a.states + n0;

        // the block's sequences at the last tile
        const IO* u_p = static_cast<const IO*>(a.u) + b * a.u_b + g_base + c_base + top * a.u_t;
        const IO* d_p = static_cast<const IO*>(a.delta) + b * a.delta_b + g_base + c_base + top * a.delta_t;
        const IO* z_p = static_cast<const IO*>(a.z) + b * a.z_b + g_base + c_base + top * a.z_t;
        const IO* g_p = static_cast<const IO*>(g.grad_y) + b * a.y_b + g_base + c_base + top * a.y_t;
        const IO* B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g + top * a.B_t;
        const IO* C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g + top * a.C_t;
        using Raw = typename Tl::Raw;
        auto fill = [&](int t0) {
            const int rows = len - t0;
            Raw& r = sh.raw[t0 / TT & 1];
            fill_tile<IO, TT, BC, NT, WIDE>(r.u[0], u_p, a.u_t, rows, cols, p.words);
            fill_tile<IO, TT, BC, NT, WIDE>(r.d[0], d_p, a.delta_t, rows, cols, p.words);
            fill_tile<IO, TT, BC, NT, WIDE>(r.g[0], g_p, a.y_t, rows, cols, p.words);
            if (a.z) fill_tile<IO, TT, BC, NT, WIDE>(r.z[0], z_p, a.z_t, rows, cols, p.words);
            fill_tile<IO, TT, NS, NT, WIDE>(r.B[0], B_p, a.B_t, rows, a.states, p.words);
            fill_tile<IO, TT, NS, NT, WIDE>(r.C_[0], C_p, a.C_t, rows, a.states, p.words);
            u_p -= TT * a.u_t;
            d_p -= TT * a.delta_t;
            z_p -= TT * a.z_t;
            g_p -= TT * a.y_t;
            B_p -= TT * a.B_t;
            C_p -= TT * a.C_t;
            copy_commit();
        };
        if (top >= 0) fill(top);

        // the state in front of the 8 steps from t on
        auto state_at = [&](int t, float2(&v)[C][J]) {
            const float* q = t > 0 ? a.kept + (long long)(t / R - 1) * a.batch * a.channels * a.states + row
                                   : (a.h0 ? a.h0 + row : nullptr);
            if (whole && q) {
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (cl + c * CL < cols && n0 < a.states) load_states<S>(v[c], q + c * crow);
            } else {
                get(q, v);
            }
        };
        float2 start[C][J] = {};                                // loaded one chunk ahead
        if (top >= 0) state_at((len - 1) / R * R, start);
        float2 lam[C][J] = {};                                  // a_(t+1) l_(t+1)
        const long long rows = a.batch * a.channels;
        if (p.chained && len > first && whole_len > stop) {
            if (tid == 0) sh.ready = wait_at_least(p.flags + chain, p.splits - 1 - split, whole_len - stop, p.patience);
            __syncthreads();
            get(p.ends + split * rows * a.states + row, lam);
            if (!sh.ready) {
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < J; ++j) lam[c][j] = two(__int_as_float(0x7fc00000));
            }
        } else if (len > first || split == 0) {
            get(g.grad_h_last ? g.grad_h_last + row : nullptr, lam);
            if (!p.chained) for (int k = (whole_len - 1) / p.split_steps; k > split; --k) {
                float2 end[C][J] = {};
                get(p.ends + k * rows * a.states + row, end);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float half = cl + c * CL < cols ? 0.5f * p.end_steps[k * rows + b * a.channels + g_base + c_base + cl + c * CL] : 0.0f;
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        lam[c][j] = make_float2(carry_over(half * A2[c][j].x, lam[c][j].x, end[c][j].x),
                                                carry_over(half * A2[c][j].y, lam[c][j].y, end[c][j].y));
                }
            }
        }

        // rows behind the end
        if (ch_ok)
            for (long long t = (top < 0 ? (long long)first : (long long)top + TT) + t_e; t < stop; t += TS) {
                const float2 none = two(0.0f);
                store<IO, V>(gu_p + (t - t_e) * g.gu_t, none);
                store<IO, V>(gd_p + (t - t_e) * g.gdelta_t, none);
                if (g.grad_z) store<IO, V>(gz_p + (t - t_e) * g.gz_t, none);
            }

        for (int t0 = top; t0 >= first; t0 -= TT) {
            const Raw& raw = sh.raw[t0 / TT & 1];
            copy_wait<0>();
            __syncthreads();
            if (t0 > first) fill(t0 - TT);
            const bool tail = t0 + TT > len;
            float2 x_r[E], dt_r[E];                             // the softplus's argument and result
            if (t_e < TT) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int t = t_e + e * TS;
                    const float2 u = unpack<IO, V>(&raw.u[t][ch]);
                    float2 go = unpack<IO, V>(&raw.g[t][ch]);
                    float2 dt = __fadd2_rn(unpack<IO, V>(&raw.d[t][ch]), bias);
                    x_r[e] = dt;
                    if (a.softplus) dt = softplus_f(dt);
                    if (tail && t0 + t >= len) dt = two(0.0f);  // a step behind the end leaves the state alone
                    dt_r[e] = dt;
                    if (a.z) {
                        const float2 z = unpack<IO, V>(&raw.z[t][ch]);
                        go = __fmul2_rn(go, __fmul2_rn(z, sigmoid_f(z)));
                    }
                    sh.d[ch][t] = make_float2(dt.x, dt.x * u.x);
                    sh.g[ch][t] = go.x;
                    if (V == 2) {
                        sh.d[ch + V - 1][t] = make_float2(dt.y, dt.y * u.y);
                        sh.g[ch + V - 1][t] = go.y;
                    }
                }
            }
#pragma unroll
            for (int i = tid; i < TT * NS; i += NT) {
                sh.B[0][i] = to_f(raw.B[0][i]);
                sh.C_[0][i] = to_f(raw.C_[0][i]);
            }
            __syncthreads();

            // decays that stay near 1 for the whole tile take the polynomial (both of a pair, or none)
            bool near1[C][J];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float most = 0.0f;
#pragma unroll
                for (int t = 0; t < TT; t += SL)
                    if (SL <= TT || sl < TT) most = fmaxf(most, fabsf(sh.d[cl + c * CL][t + (SL <= TT ? sl : sl % TT)].x));
#pragma unroll
                for (int m = SL / 2; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m * CL));
#pragma unroll
                for (int j = 0; j < J; ++j)
                    near1[c][j] = most * fmaxf(fabsf(A2[c][j].x), fabsf(A2[c][j].y)) < kExp2Near;
            }

            float2 dA[C][J] = {};
#pragma unroll 1
            for (int tr = TT - R; tr >= 0; tr -= R) {
                if (t0 + tr >= len) continue;
                // the 8 steps' decays and states
                float2 da[R][C][J], hh[R + 1][C][J];
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < J; ++j) hh[0][c][j] = start[c][j];
                if (t0 + tr > first) state_at(t0 + tr - R, start);
                using OverStates = LaneSums<Q, SL, CL>;
                using OverChannels = LaneSums<Q, CL, 1>;
                auto keep = [&](float(&v)[Q], float* to) {
                    OverStates::run(v, sl);
                    if (OverStates::stores(sl)) {
#pragma unroll
                        for (int i = 0; i < OverStates::kHeld; ++i) to[OverStates::first(sl) + i] = v[i];
                    }
                };
                auto over_channels = [&](float(&v)[S][Q], float(*to)[NS], int tq) {
#pragma unroll
                    for (int s = 0; s < S; ++s) OverChannels::run(v[s], lc);
                    if (OverChannels::stores(lc)) {
#pragma unroll
                        for (int i = 0; i < OverChannels::kHeld; ++i)
                            store_states<S>(&to[tr + tq + OverChannels::first(lc) + i][n0], v, i);
                    }
                };
#pragma unroll
                for (int tq = 0; tq < R; tq += Q) {
                    float o[C][Q], dC[S][Q];
#pragma unroll
                    for (int i = 0; i < Q; ++i) {
                        const int t = tq + i;
                        float2 Bv[J], Cv[J], dCt[J];
                        load_states<S>(Bv, &sh.B[tr + t][n0]);
                        if (a.z) load_states<S>(Cv, &sh.C_[tr + t][n0]);
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            const float2 d = sh.d[cl + c * CL][tr + t], go = two(sh.g[cl + c * CL][tr + t]);
#pragma unroll
                            for (int j = 0; j < J; ++j) {
                                const float2 x = __fmul2_rn(two(d.x), A2[c][j]), q = exp2_near1(x);
                                da[t][c][j] = make_float2(near1[c][j] ? q.x : exp2_approx(x.x),
                                                          near1[c][j] ? q.y : exp2_approx(x.y));
                                hh[t + 1][c][j] = __ffma2_rn(da[t][c][j], hh[t][c][j], __fmul2_rn(two(d.y), Bv[j]));
                                dCt[j] = c == 0 ? __fmul2_rn(go, hh[t + 1][c][j]) : __ffma2_rn(go, hh[t + 1][c][j], dCt[j]);
                            }
                            if (a.z) {
                                float2 acc = __fmul2_rn(hh[t + 1][c][0], Cv[0]);
#pragma unroll
                                for (int j = 1; j < J; ++j) acc = __ffma2_rn(hh[t + 1][c][j], Cv[j], acc);
                                o[c][i] = acc.x + acc.y;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < J; ++j) {
                            dC[2 * j][i] = dCt[j].x;
                            dC[2 * j + 1][i] = dCt[j].y;
                        }
                    }
                    over_channels(dC, sh.red[warp][1], tq);
                    if (a.z) {
#pragma unroll
                        for (int c = 0; c < C; ++c) keep(o[c], &sh.o[cl + c * CL][tr + tq]);
                    }
                }
                // and backwards through them
#pragma unroll
                for (int tq = R - Q; tq >= 0; tq -= Q) {
                    float lb[C][Q], qa[C][Q], dB[S][Q];
#pragma unroll
                    for (int i = Q - 1; i >= 0; --i) {
                        const int t = tq + i;
                        float2 Bv[J], Cv[J], dBt[J];
                        load_states<S>(Bv, &sh.B[tr + t][n0]);
                        load_states<S>(Cv, &sh.C_[tr + t][n0]);
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            const float2 d = sh.d[cl + c * CL][tr + t];
                            const float2 dt = two(d.x), du = two(d.y), go = two(sh.g[cl + c * CL][tr + t]);
                            float2 r1, r2;
#pragma unroll
                            for (int j = 0; j < J; ++j) {
                                const float2 l = __ffma2_rn(Cv[j], go, lam[c][j]);
                                lam[c][j] = __fmul2_rn(l, da[t][c][j]);
                                const float2 q = __fmul2_rn(lam[c][j], hh[t][c][j]);
                                dBt[j] = c == 0 ? __fmul2_rn(l, du) : __ffma2_rn(l, du, dBt[j]);
                                r1 = j == 0 ? __fmul2_rn(l, Bv[j]) : __ffma2_rn(l, Bv[j], r1);
                                r2 = j == 0 ? __fmul2_rn(q, A2[c][j]) : __ffma2_rn(q, A2[c][j], r2);
                                dA[c][j] = __ffma2_rn(q, dt, dA[c][j]);
                            }
                            lb[c][i] = r1.x + r1.y;
                            qa[c][i] = r2.x + r2.y;
                        }
#pragma unroll
                        for (int j = 0; j < J; ++j) {
                            dB[2 * j][i] = dBt[j].x;
                            dB[2 * j + 1][i] = dBt[j].y;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        keep(lb[c], &sh.lb[cl + c * CL][tr + tq]);
                        keep(qa[c], &sh.qa[cl + c * CL][tr + tq]);
                    }
                    over_channels(dB, sh.red[warp][0], tq);
                }
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < J; ++j) add_to(sh.sum_a[c * J + j][tid], dA[c][j]);

            // elementwise gradients
            if (ch_ok) {
                float2 sum_D = two(0.0f), sum_bias = two(0.0f);
                IO *gu_t = gu_p + t0 * g.gu_t, *gd_t = gd_p + t0 * g.gdelta_t, *gz_t = gz_p + t0 * g.gz_t;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int t = t_e + e * TS;
                    if (!tail || t0 + t < stop) {
                        const float2 u = unpack<IO, V>(&raw.u[t][ch]);
                        float2 go = unpack<IO, V>(&raw.g[t][ch]), gz = two(0.0f);
                        const float2 lb = make_float2(sh.lb[ch][t], sh.lb[ch + V - 1][t]);
                        const float2 qa = make_float2(sh.qa[ch][t], sh.qa[ch + V - 1][t]);
                        if (a.z) {
                            const float2 z = unpack<IO, V>(&raw.z[t][ch]), sg = sigmoid_f(z), si = __fmul2_rn(z, sg);
                            const float2 o = __ffma2_rn(skip, u, make_float2(sh.o[ch][t], sh.o[ch + V - 1][t]));
                            // silu' = sg + si (1 - sg)
                            const float2 ds = __ffma2_rn(si, __ffma2_rn(sg, two(-1.0f), two(1.0f)), sg);
                            gz = __fmul2_rn(__fmul2_rn(go, o), ds);
                            go = __fmul2_rn(go, si);
                        }
                        // q A came with A log2 e
                        float2 gd = __ffma2_rn(u, lb, __fmul2_rn(qa, two(0.69314718055994530942f)));
                        if (a.softplus) gd = __fmul2_rn(gd, sigmoid_f(x_r[e]));
                        float2 gu = __ffma2_rn(dt_r[e], lb, __fmul2_rn(skip, go));
                        if (tail && t0 + t >= len) gd = gu = gz = go = two(0.0f);
                        store<IO, V>(gu_t + e * (TS * g.gu_t), gu);
                        store<IO, V>(gd_t + e * (TS * g.gdelta_t), gd);
                        if (g.grad_z) store<IO, V>(gz_t + e * (TS * g.gz_t), gz);
                        sum_bias = __fadd2_rn(sum_bias, gd);
                        sum_D = __ffma2_rn(go, tail && t0 + t >= len ? two(0.0f) : u, sum_D);
                    }
                }
                add_to(sh.sum_d[0][tid], sum_D);
                add_to(sh.sum_d[1][tid], sum_bias);
            }
            // this block's part of grad B and grad C
#pragma unroll
            for (int i = tid; i < 2 * TT * NS / S; i += NT) {
                const int n = i % (NS / S) * S, t = i / (NS / S) % TT, which = i / (NS / S * TT);
                if (t0 + t < len) {
                    float2 v[J];
                    load_states<S>(v, &sh.red[0][which][t][n]);
#pragma unroll
                    for (int w = 1; w < NW; ++w) {
                        float2 x[J];
                        load_states<S>(x, &sh.red[w][which][t][n]);
#pragma unroll
                        for (int j = 0; j < J; ++j) v[j] = __fadd2_rn(v[j], x[j]);
                    }
                    float* q = p.part_bc + ((((long long)which * p.tiles + tile) * p.T + t0 + t) * a.batch + b) * a.groups * a.states
                               + grp * a.states + n;
#pragma unroll
                    for (int s = 0; s < S; ++s)
                        if (n + s < a.states) q[s] = s % 2 ? v[s / 2].y : v[s / 2].x;
                }
            }
        }
        if (g.grad_h0 && split == 0) put(g.grad_h0 + row, lam);
        if (p.chained && split > 0 && len > first) {            // for the part in front
            put(p.ends + (split - 1) * rows * a.states + row, lam);
            __threadfence();
            __syncthreads();
            if (tid == 0) publish(p.flags + chain, p.splits - split);
        }
        __syncthreads();                                        // before the next sequence's copies
    }

    float2 dA[C][J];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const double2 v = sh.sum_a[c * J + j][tid];
            dA[c][j] = make_float2((float)v.x, (float)v.y);
        }
    put(p.part_a + ((long long)part * a.channels + g_base + c_base + cl) * a.states + n0, dA);
    // the threads of a pack's channels, in order
    __syncthreads();
    if (tid < ROW) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            double2 v = make_double2(0.0, 0.0);
            for (int i = tid; i < NT; i += ROW) v = make_double2(v.x + sh.sum_d[which][i].x, v.y + sh.sum_d[which][i].y);
            float* q = p.part_d + ((long long)which * parts + part) * a.channels + chan;
            if (ch < cols) q[0] = (float)v.x;
            if (V == 2 && ch + 1 < cols) q[1] = (float)v.y;
        }
    }
}

// What a part of a sequence (all but the first) adds to a_t l_t in front of it, from zero behind it,
// and its sum of d: the walk of scan_bwd without anything else, for few long sequences.
template <typename IO, int S, int SL>
struct EndTile {
    static constexpr int CL = 32 / SL, BC = NW * CL, NS = S * SL;
    struct Raw {
        IO d[TT][BC], z[TT][BC], g[TT][BC], C_[TT][NS];
    };
    __align__(16) Raw raw[2];
    __align__(16) float C_[TT][NS];
    float2 d[BC][TT + 1];                            // (d, grad o)
};

template <typename IO, int S, int SL, bool WIDE>
__global__ void __launch_bounds__(NT) scan_bwd_ends(const ScanParams p) {
    using Tl = EndTile<IO, S, SL>;
    constexpr int CL = Tl::CL, BC = Tl::BC, NS = Tl::NS, J = S / 2;
    constexpr int V = WIDE ? 2 : 1, ROW = BC / V;
    constexpr int E = TT * ROW > NT ? TT * ROW / NT : 1, TS = TT / E;
    extern __shared__ __align__(16) unsigned char smem[];
    Tl& sh = *reinterpret_cast<Tl*>(smem);
    const dfsnn_state_scan_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long bid = blockIdx.x;
    const int tile = (int)(bid % p.tiles);
    bid /= p.tiles;
    const int grp = (int)(bid % a.groups);
    bid /= a.groups;
    const int split = (int)(bid % (p.splits - 1)) + 1;
    const long long b = bid / (p.splits - 1);
    const int first = split * p.split_steps;
    const int stop = p.T - first < p.split_steps ? p.T : first + p.split_steps;
    const int whole_len = seq_length(a.lengths, a.lengths64, b, p.T);
    const int len = whole_len < stop ? whole_len : stop;
    if (len <= first) return;
    const int c_base = tile * BC, cols = p.group_channels - c_base;
    const long long g_base = (long long)grp * p.group_channels;
    const int ch = tid % ROW * V, t_e = tid / ROW;
    const long long chan = g_base + c_base + ch;
    float2 bias = two(0.0f);
    if (ch < cols && a.delta_bias) bias = make_float2(a.delta_bias[chan], a.delta_bias[chan + V - 1]);
    const int sl = lane / CL, cl = warp * CL + lane % CL, n0 = sl * S;
    const long long ch_row = g_base + c_base + cl;
    float2 A2[J], x[J] = {};
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const bool ok = cl < cols;
        A2[j].x = ok && n0 + 2 * j < a.states ? log2_rate(a.A[ch_row * a.states + n0 + 2 * j]) : 0.0f;
        A2[j].y = ok && n0 + 2 * j + 1 < a.states ? log2_rate(a.A[ch_row * a.states + n0 + 2 * j + 1]) : 0.0f;
    }
    float steps = 0.0f;
    auto fill = [&](int t0) {
        const int rows = len - t0;
        const long long c = g_base + c_base;
        typename Tl::Raw& r = sh.raw[t0 / TT & 1];
        fill_tile<IO, TT, BC, NT, WIDE>(r.d[0], static_cast<const IO*>(a.delta) + b * a.delta_b + c + t0 * a.delta_t, a.delta_t, rows, cols, p.words);
        fill_tile<IO, TT, BC, NT, WIDE>(r.g[0], static_cast<const IO*>(p.g.grad_y) + b * a.y_b + c + t0 * a.y_t, a.y_t, rows, cols, p.words);
        if (a.z)
            fill_tile<IO, TT, BC, NT, WIDE>(r.z[0], static_cast<const IO*>(a.z) + b * a.z_b + c + t0 * a.z_t, a.z_t, rows, cols, p.words);
        fill_tile<IO, TT, NS, NT, WIDE>(r.C_[0], static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g + t0 * a.C_t, a.C_t, rows, a.states, p.words);
        copy_commit();
    };
    const int top = (len - 1) / TT * TT;
    fill(top);
    for (int t0 = top; t0 >= first; t0 -= TT) {
        const typename Tl::Raw& raw = sh.raw[t0 / TT & 1];
        copy_wait<0>();
        __syncthreads();
        if (t0 > first) fill(t0 - TT);
        if (t_e < TT) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int t = t_e + e * TS;
                float2 go = unpack<IO, V>(&raw.g[t][ch]), dt = __fadd2_rn(unpack<IO, V>(&raw.d[t][ch]), bias);
                if (a.softplus) dt = softplus_f(dt);
                if (t0 + t >= len) dt = two(0.0f);
                if (a.z) {
                    const float2 z = unpack<IO, V>(&raw.z[t][ch]);
                    go = __fmul2_rn(go, __fmul2_rn(z, sigmoid_f(z)));
                }
                sh.d[ch][t] = make_float2(dt.x, go.x);
                if (V == 2) sh.d[ch + V - 1][t] = make_float2(dt.y, go.y);
            }
        }
#pragma unroll
        for (int i = tid; i < TT * NS; i += NT) sh.C_[0][i] = to_f(raw.C_[0][i]);
        __syncthreads();
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < TT; ++t) most = fmaxf(most, fabsf(sh.d[cl][t].x));
        bool near1[J];
#pragma unroll
        for (int j = 0; j < J; ++j) near1[j] = most * fmaxf(fabsf(A2[j].x), fabsf(A2[j].y)) < kExp2Near;
#pragma unroll
        for (int t = TT - 1; t >= 0; --t) {
            float2 Cv[J];
            load_states<S>(Cv, &sh.C_[t][n0]);
            const float2 d = sh.d[cl][t];
            steps += d.x;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float2 y = __fmul2_rn(two(d.x), A2[j]), q = exp2_near1(y);
                const float2 dec = make_float2(near1[j] ? q.x : exp2_approx(y.x), near1[j] ? q.y : exp2_approx(y.y));
                x[j] = __fmul2_rn(dec, __ffma2_rn(Cv[j], two(d.y), x[j]));
            }
        }
    }
    if (cl < cols) {
        const long long at = ((long long)split * a.batch + b) * a.channels + ch_row;
        if (sl == 0) p.end_steps[at] = steps;
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (n0 + s < a.states) p.ends[at * a.states + n0 + s] = s % 2 ? x[s / 2].y : x[s / 2].x;
    }
}

// Adds the blocks' parts in a fixed order.  Blocks 0 .. bc_blocks - 1: grad B and grad C over the
// channel tiles, a thread for an output.  The others: grad A, D and delta_bias over the parts of
// the batch and the sequences, 32 outputs a block; its 8 warps add every eighth part, then the
// warps' sums are added in order.
constexpr int kSumThreads = 256;
template <typename IO>
__global__ void __launch_bounds__(kSumThreads) scan_bwd_sums(const ScanParams p, int bc_blocks) {
    const dfsnn_state_scan_args& a = p.a;
    const dfsnn_state_scan_grads& g = p.g;
    const long long n_bc = (long long)p.T * a.batch * a.groups * a.states;
    const long long n_a = a.channels * a.states;
    if (blockIdx.x < bc_blocks) {
        // W neighbouring states of a (step, sequence, group) at a time
        auto add = [&](auto width) {
            constexpr int W = decltype(width)::value;
            for (long long i = (long long)blockIdx.x * kSumThreads + threadIdx.x; i < 2 * n_bc / W;
                 i += (long long)bc_blocks * kSumThreads) {
                const int which = i >= n_bc / W;
                const long long k = (i - which * (n_bc / W)) * W, row = k / (a.groups * a.states);
                float v[W] = {};
                if (row / a.batch < seq_length(a.lengths, a.lengths64, row % a.batch, p.T)) {
                    const float* q = p.part_bc + (long long)which * p.tiles * n_bc + k;
#pragma unroll 8
                    for (int j = 0; j < p.tiles; ++j, q += n_bc) {
                        if constexpr (W == 4) {
                            const float4 f = __ldcs(reinterpret_cast<const float4*>(q));
                            v[0] += f.x;
                            v[1] += f.y;
                            v[2] += f.z;
                            v[3] += f.w;
                        } else {
                            v[0] += *q;
                        }
                    }
                }
                IO* out = static_cast<IO*>(which ? g.grad_C : g.grad_B) + k;
#pragma unroll
                for (int w = 0; w < W; ++w) out[w] = from_f<IO>(v[w]);
            }
        };
        if (a.states % 4 == 0) add(std::integral_constant<int, 4>{});      // rows of parts lie on 16 bytes
        else add(std::integral_constant<int, 1>{});
        return;
    }
    __shared__ double s_sum[kSumThreads / 32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long i = (long long)(blockIdx.x - bc_blocks) * 32 + lane;
    const int parts = p.batch_parts * p.splits;
    const float* q = nullptr;
    long long stride = n_a;
    float* out = nullptr;
    if (i < n_a) {
        q = p.part_a + i;
        out = g.grad_A + i;
    } else if (i < n_a + 2 * a.channels) {
        const int which = i - n_a >= a.channels;
        const long long c = i - n_a - which * a.channels;
        stride = a.channels;
        q = p.part_d + which * parts * a.channels + c;
        out = which ? g.grad_delta_bias : g.grad_D;
        if (out) out += c;
    }
    double v = 0.0;
    if (out) {
#pragma unroll 4
        for (int j = warp; j < parts; j += kSumThreads / 32) v += q[j * stride];
    }
    s_sum[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && out) {
        v = 0.0;
        for (int w = 0; w < kSumThreads / 32; ++w) v += s_sum[w][lane];
        *out = (float)v;
    }
}

template <typename IO, int S, int SL, int C, bool WIDE>
cudaError_t launch_form(const ScanParams& p, cudaStream_t st) {
    const long long blocks = (long long)p.tiles * p.a.groups * p.batch_parts * p.splits;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (p.chained) {
        const cudaError_t e = cudaMemsetAsync(p.flags, 0, (p.tiles * p.a.groups * p.batch_parts + 1) * sizeof(int), st);
        if (e != cudaSuccess) return e;
    } else if (p.splits > 1) {
        using Ends = EndTile<IO, S, SL>;
        ScanParams q = p;
        q.tiles = (p.group_channels + Ends::BC - 1) / Ends::BC;
        const long long n = (long long)q.tiles * p.a.groups * p.a.batch * (p.splits - 1);
        if (n > 0x7fffffffLL) return cudaErrorInvalidValue;
        cudaError_t e = allow_shared<scan_bwd_ends<IO, S, SL, WIDE>>(sizeof(Ends));
        if (e != cudaSuccess) return e;
        scan_bwd_ends<IO, S, SL, WIDE><<<(unsigned)n, NT, sizeof(Ends), st>>>(q);
    }
    constexpr size_t smem = sizeof(Tile<IO, S, SL, C>);
    static_assert(S * SL > 64 || 3 * (smem + 1024) <= 228 * 1024, "three blocks an SM up to 64 states");
    cudaError_t e = allow_shared<scan_bwd<IO, S, SL, C, WIDE>>(smem);
    if (e != cudaSuccess) return e;
    scan_bwd<IO, S, SL, C, WIDE><<<(unsigned)blocks, NT, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename IO, int S, int SL, int C>
cudaError_t launch(ScanParams p, cudaStream_t st) {
    const dfsnn_state_scan_grads& g = p.g;
    p.words = rows_aligned(p, sizeof(IO), 4);
    const bool wide = p.group_channels % 2 == 0 && rows_aligned(p, sizeof(IO), 16)
                      && pairs_aligned(g.grad_u, g.gu_t, g.gu_b, sizeof(IO))
                      && pairs_aligned(g.grad_delta, g.gdelta_t, g.gdelta_b, sizeof(IO))
                      && pairs_aligned(g.grad_z, g.gz_t, g.gz_b, sizeof(IO));
    return wide ? launch_form<IO, S, SL, C, true>(p, st) : launch_form<IO, S, SL, C, false>(p, st);
}

template <typename IO>
cudaError_t pick(const ScanParams& p, cudaStream_t st) {
    const int n = p.a.states;
    cudaError_t e;
    if (n <= 4) e = launch<IO, 2, 2, 1>(p, st);
    else if (n <= 8) e = launch<IO, 2, 4, 2>(p, st);
    else if (n <= 16) e = launch<IO, 4, 4, 1>(p, st);
    else if (n <= 32) e = launch<IO, 4, 8, 1>(p, st);
    else if (n <= 64) e = launch<IO, 4, 16, 1>(p, st);
    else e = launch<IO, 4, 32, 1>(p, st);
    if (e != cudaSuccess) return e;
    const long long n_bc = (long long)p.T * p.a.batch * p.a.groups * p.a.states;
    const int bc_blocks = (int)std::min<long long>((2 * n_bc + kSumThreads - 1) / kSumThreads, 148 * 16);
    const long long params = (p.a.channels * (p.a.states + 2) + 31) / 32;
    scan_bwd_sums<IO><<<(unsigned)(bc_blocks + params), kSumThreads, 0, st>>>(p, bc_blocks);
    return cudaGetLastError();
}

// Channels of a block for a state count, as pick() has them.  N = 5 .. 8: two channels a lane, which is
// better for short sequences (fp32, 16 x 4096 x 256: 317 us against 333 with one) and few rows (bf16,
// 1000 x 4 x 1000: 143 against 154), not for long ones that fill the machine (fp32, 1024 x 8 x 2048: 477
// against 326).
int block_channels(int states) {
    if (states <= 4) return Tile<float, 2, 2, 1>::BC;
    if (states <= 8) return Tile<float, 2, 4, 2>::BC;
    if (states <= 16) return Tile<float, 4, 4, 1>::BC;
    if (states <= 32) return Tile<float, 4, 8, 1>::BC;
    if (states <= 64) return Tile<float, 4, 16, 1>::BC;
    return Tile<float, 4, 32, 1>::BC;
}

}  // namespace

int state_scan_bwd_tiles(int states, long long group_channels) {
    const int bc = block_channels(states);
    return (int)((group_channels + bc - 1) / bc);
}

// How the blocks share sequences, of which `slots` walk one at a time (three blocks on each of 148
// SMs; for N > 64 the blocks' shared memory leaves two, one in fp32, and the rule was not measured
// there).  bf16, N = 16, microseconds of the whole backward with the rule and without:
//   * few rows (two parts a sequence fit the slots): each sequence in parts side by side, at the
//     price of a second walk for their ends: 4096 x 1 x 512 91 against 940, 4096 x 1 x 4096 665
//     against 984; parts of 4 tiles at least;
//   * more blocks than slots: the last wave of blocks would leave most of the machine idle for a
//     whole walk.  The sequences are cut into parts that run one after another, a block passing its
//     a_t l_t on to the next (chained), so that the last wave is a short one: 2048 x 8 x 2048 924
//     against 1205, 512 x 8 x 2048 261 against 323;
//   * 8 blocks an SM are enough of them: beyond that a block takes several sequences and adds its
//     grad A on the way, which keeps the partial sums small.
void state_scan_bwd_plan(ScanParams& p) {
    const long long per = (long long)state_scan_bwd_tiles(p.a.states, p.group_channels) * p.a.groups;
    const long long blocks = per * p.a.batch, slots = 148 * 3;
    p.splits = 1;
    p.split_steps = p.T;
    p.chained = 0;
    p.batch_parts = (int)std::max<long long>(1, std::min(p.a.batch, (148 * 8 + per - 1) / per));
    long long splits = std::min<long long>(slots / blocks, p.T / (4 * TT));
    if (splits < 2 && blocks > slots) {
        splits = std::min<long long>(8 * slots / blocks, p.T / (8 * TT));
        p.chained = splits > 1;
    }
    if (splits < 2) return;
    const long long chunks = (p.T + TT - 1) / TT, each = (chunks + splits - 1) / splits;
    p.split_steps = (int)(each * TT);
    p.splits = (int)((chunks + each - 1) / each);
    p.batch_parts = (int)p.a.batch;
}

cudaError_t state_scan_expired_waits(unsigned long long* count, cudaStream_t st) {
    const cudaError_t e = cudaMemcpyFromSymbolAsync(count, expired_waits, sizeof(*count), 0, cudaMemcpyDeviceToHost, st);
    return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}

cudaError_t state_scan_backward_launch(const ScanParams& p, cudaStream_t st) {
    switch (p.a.dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(p, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(p, st);
        default: return pick<float>(p, st);
    }
}

}  // namespace dfsnn
