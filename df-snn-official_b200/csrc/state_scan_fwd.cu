// state_scan_fwd.cu -- forward of the selective scan.
//
//   h_t[n] = exp(d_t A[n]) h_(t-1)[n] + d_t u_t B_t[n],   o_t = sum_n C_t[n] h_t[n] + D u_t
//
// One exponential and five multiply-adds for each (step, channel, state), against 3 or 4 elements
// of traffic for all N states of a (step, channel): with N = 16 the kernel is bound by the 16
// exponentials a clock of an SM's special-function unit, not by memory.  Everything else has to
// fit beside them:
//   * a channel's states lie on SL lanes, four neighbouring states each, as two packed pairs (half
//     the issue slots), and a warp walks the sequence of its 32 / SL channels;
//   * steps are taken in tiles of 16, and the sums over a channel's lanes are formed for the 16
//     steps together (LaneSums): (1 - 1/SL) shuffles a step instead of log2 SL;
//   * the elementwise work (softplus, gate, skip) is done once per (step, channel) by all threads
//     of the block, before and after the tile, with the next tile's loads in flight meanwhile.
// States, decays and sums are fp32; y is rounded once.
//
// Few rows leave most of the machine idle, so a long sequence is then cut into `splits` parts that
// run side by side: a first launch (ENDS) walks all parts but the last from a zero state for the
// state each part adds, h_out = exp(A sum d) h_in + end, and the second folds those up to its part
// before it walks it.  That takes the exponentials twice; state_scan_splits() weighs it.
#include <algorithm>

#include "state_scan.h"

namespace dfsnn {
namespace {

constexpr int TT = kScanChunk, S = 4, NT = 128;

template <int SL>
struct Tile {
    static constexpr int CL = 32 / SL;                 // channels of a warp
    static constexpr int BC = NT / 32 * CL;            // channels of the block
    static constexpr int NS = S * SL;                  // states, padded
    static constexpr int E = CL > 1 ? CL / 2 : 1;      // (step, channel) elements of a thread,
    static constexpr int TS = TT / E;                  // this many steps apart
    static constexpr int F = (TT * NS + NT - 1) / NT;  // entries of B (and C) of a thread
    float4 d[BC][TT + 1];                              // (d, d, d u, d u): packed operands as they are
    float B[TT][NS], C[TT][NS];
    float o[BC][TT + 4];
};

template <typename IO, int SL, bool ENDS>
__global__ void __launch_bounds__(NT) scan_fwd(const ScanParams p) {
    using Tl = Tile<SL>;
    constexpr int CL = Tl::CL, BC = Tl::BC, NS = Tl::NS, E = Tl::E, F = Tl::F, TS = Tl::TS;
    extern __shared__ __align__(16) unsigned char smem[];
    Tl& sh = *reinterpret_cast<Tl*>(smem);
    const dfsnn_state_scan_args& a = p.a;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long bid = blockIdx.x;
    const int tile = (int)(bid % p.tiles);
    bid /= p.tiles;
    const int grp = (int)(bid % a.groups);
    bid /= a.groups;
    const int parts = ENDS ? p.splits - 1 : p.splits;
    const int split = (int)(bid % parts);
    const long long b = bid / parts;
    const int whole_len = seq_length(a.lengths, a.lengths64, b, p.T);
    const int first = split * p.split_steps;                    // this part's steps: first .. len - 1,
    const int stop = p.T - first < p.split_steps ? p.T : first + p.split_steps;   // its rows: .. stop - 1
    const int len = whole_len < stop ? whole_len : stop;
    if (ENDS && whole_len <= stop) return;                      // no part behind this one
    const int c_base = tile * BC;                               // within the group
    const long long g_base = (long long)grp * p.group_channels; // first channel of the group

    // elementwise role: elements (step t_e + e * TS, channel ch)
    const int ch = tid % BC, t_e = tid / BC;
    const bool ch_ok = c_base + ch < p.group_channels && t_e < TT;
    const long long chan = g_base + c_base + ch;
    const float bias = ch_ok && a.delta_bias ? a.delta_bias[chan] : 0.0f;
    const float skip = ch_ok && a.D ? a.D[chan] : 0.0f;
    const IO* u_p = static_cast<const IO*>(a.u) + b * a.u_b + chan + (first + t_e) * a.u_t;
    const IO* d_p = static_cast<const IO*>(a.delta) + b * a.delta_b + chan + (first + t_e) * a.delta_t;
    const IO* z_p = static_cast<const IO*>(a.z) + b * a.z_b + chan + (first + t_e) * a.z_t;
    IO* y_p = static_cast<IO*>(a.y) + b * a.y_b + chan + (first + t_e) * a.y_t;
    // entries of B and C: state n_f, steps t_f + f * DF
    const int n_f = tid % NS, t_f = tid / NS;
    constexpr int DF = NT / NS > 0 ? NT / NS : 1;               // steps between a thread's entries
    const IO* B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g + n_f + (first + t_f) * a.B_t;
    const IO* C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g + n_f + (first + t_f) * a.C_t;

    // recurrence role: states n0 .. n0 + 3 of channel cl of the block
    const int sl = lane % SL, cl = warp * CL + lane / SL, n0 = sl * S;
    const bool cl_ok = c_base + cl < p.group_channels;
    const long long row = ((long long)b * a.channels + g_base + c_base + cl) * a.states + n0;
    // a lane's states are one float4 everywhere
    const bool whole = a.states % S == 0
                       && ((reinterpret_cast<uintptr_t>(a.kept) | reinterpret_cast<uintptr_t>(a.h_last)) & 15) == 0;
    float2 A2[S / 2] = {}, h[S / 2] = {};
    auto get = [&](const float* q, float2(&v)[S / 2]) {
        float f[S];
#pragma unroll
        for (int s = 0; s < S; ++s) f[s] = q && cl_ok && n0 + s < a.states ? q[s] : 0.0f;
        v[0] = make_float2(f[0], f[1]);
        v[1] = make_float2(f[2], f[3]);
    };
    auto put = [&](float* q) {
        if (!cl_ok || n0 >= a.states) return;
        if (whole) {
            *reinterpret_cast<float4*>(q) = make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
        } else {
            const float f[S] = {h[0].x, h[0].y, h[1].x, h[1].y};
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (n0 + s < a.states) q[s] = f[s];
        }
    };
    get(a.A + (g_base + c_base + cl) * a.states + n0, A2);
#pragma unroll
    for (int j = 0; j < S / 2; ++j) A2[j] = make_float2(A2[j].x * kLog2e, A2[j].y * kLog2e);
    if (!ENDS && first < whole_len) {
        get(a.h0 ? a.h0 + row : nullptr, h);
        const long long rows = a.batch * a.channels;
        for (int k = 0; k < split; ++k) {
            float2 end[S / 2];
            get(p.ends + k * rows * a.states + row, end);
            const float d = cl_ok ? p.end_steps[k * rows + b * a.channels + g_base + c_base + cl] : 0.0f;
#pragma unroll
            for (int j = 0; j < S / 2; ++j)
                h[j] = make_float2(fmaf(exp2_approx(d * A2[j].x), h[j].x, end[j].x),
                                   fmaf(exp2_approx(d * A2[j].y), h[j].y, end[j].y));
        }
    } else if (!ENDS && split == 0) {
        get(a.h0 ? a.h0 + row : nullptr, h);                    // an empty sequence keeps its state
    }
    float steps = 0.0f;                                         // sum of d

    float u_r[E], d_r[E], z_r[E], B_r[F], C_r[F];
    auto load = [&](int t0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool ok = ch_ok && t0 + t_e + e * TS < len;
            u_r[e] = ok ? to_f(*u_p) : 0.0f;
            d_r[e] = ok ? to_f(*d_p) : 0.0f;
            u_p += TS * a.u_t;
            d_p += TS * a.delta_t;
            if (!ENDS) {
                z_r[e] = ok && a.z ? to_f(*z_p) : 0.0f;
                z_p += TS * a.z_t;
            }
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const bool ok = t_f + f * DF < TT && n_f < a.states && t0 + t_f + f * DF < len;
            B_r[f] = ok ? to_f(B_p[f * DF * a.B_t]) : 0.0f;
            if (!ENDS) C_r[f] = ok ? to_f(C_p[f * DF * a.C_t]) : 0.0f;
        }
        B_p += TT * a.B_t;
        C_p += TT * a.C_t;
    };

    load(first);
    for (int t0 = first; t0 < len; t0 += TT) {
        float u_c[E], z_c[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            u_c[e] = u_r[e];
            if (!ENDS) z_c[e] = z_r[e];
            const int t = t_e + e * TS;
            float dt = d_r[e] + bias;
            if (a.softplus) dt = softplus_f(dt);
            if (t0 + t >= len) dt = 0.0f;       // a step behind the end leaves the state alone
            const float du = dt * u_r[e];
            if (t < TT) sh.d[ch][t] = make_float4(dt, dt, du, du);
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            if (t_f + f * DF < TT) {
                sh.B[t_f + f * DF][n_f] = B_r[f];
                if (!ENDS) sh.C[t_f + f * DF][n_f] = C_r[f];
            }
        }
        __syncthreads();
        if (t0 + TT < len) load(t0 + TT);
        if (!ENDS && a.kept && t0 > 0)
            put(a.kept + (long long)(t0 / TT - 1) * a.batch * a.channels * a.states + row);
        // decays that stay near 1 for the whole tile take the polynomial
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < TT; ++t) most = fmaxf(most, fabsf(sh.d[cl][t].x));
        bool near1[S];
#pragma unroll
        for (int j = 0; j < S / 2; ++j) {
            near1[2 * j] = most * fabsf(A2[j].x) < kExp2Near;
            near1[2 * j + 1] = most * fabsf(A2[j].y) < kExp2Near;
        }
        float y[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const float4 d = sh.d[cl][t];
            const float4 B4 = *reinterpret_cast<const float4*>(&sh.B[t][n0]);
            const float4 C4 = ENDS ? B4 : *reinterpret_cast<const float4*>(&sh.C[t][n0]);
            const float2 dt = make_float2(d.x, d.y), du = make_float2(d.z, d.w);
            const float2 Bv[2] = {make_float2(B4.x, B4.y), make_float2(B4.z, B4.w)};
            const float2 Cv[2] = {make_float2(C4.x, C4.y), make_float2(C4.z, C4.w)};
            float2 acc;
            if (ENDS) steps += d.x;
#pragma unroll
            for (int j = 0; j < S / 2; ++j) {
                const float2 x = __fmul2_rn(dt, A2[j]), q = exp2_near1(x);
                const float2 dec = make_float2(near1[2 * j] ? q.x : exp2_approx(x.x),
                                               near1[2 * j + 1] ? q.y : exp2_approx(x.y));
                h[j] = __ffma2_rn(dec, h[j], __fmul2_rn(du, Bv[j]));
                acc = j == 0 ? __fmul2_rn(h[j], Cv[j]) : __ffma2_rn(h[j], Cv[j], acc);
            }
            y[t] = acc.x + acc.y;
        }
        if (ENDS) {
            __syncthreads();
            continue;
        }
        using Sums = LaneSums<TT, SL, 1>;
        Sums::run(y, sl);
        if (Sums::stores(sl)) {
#pragma unroll
            for (int i = 0; i < Sums::kHeld; ++i) sh.o[cl][Sums::first(sl) + i] = y[i];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = t_e + e * TS;
            if (ch_ok && t0 + t < stop) {
                float o = fmaf(skip, u_c[e], sh.o[ch][t]);
                if (a.z) o *= z_c[e] * sigmoid_f(z_c[e]);
                if (t0 + t >= len) o = 0.0f;
                *y_p = from_f<IO>(o);
            }
            y_p += TS * a.y_t;
        }
    }
    if (ENDS) {
        put(p.ends + split * a.batch * a.channels * a.states + row);
        if (cl_ok && sl == 0)
            p.end_steps[(split * a.batch + b) * a.channels + g_base + c_base + cl] = steps;
        return;
    }
    // rows behind the end (y_p is at the tile behind the last)
    if (ch_ok) {
        const int done = len > first ? first + (len - first + TT - 1) / TT * TT : first;
        for (long long t = done + t_e; t < stop; t += TS, y_p += TS * a.y_t) *y_p = from_f<IO>(0.0f);
    }
    if (a.h_last && (first < whole_len ? whole_len <= stop : split == 0 && whole_len == 0)) put(a.h_last + row);
}

template <typename IO, int SL>
cudaError_t launch(ScanParams p, cudaStream_t st) {
    constexpr int BC = Tile<SL>::BC;
    p.tiles = (p.group_channels + BC - 1) / BC;
    const long long blocks = (long long)p.tiles * p.a.groups * p.a.batch;
    if (blocks > 0x7fffffffLL / p.splits) return cudaErrorInvalidValue;
    if (p.splits > 1)
        scan_fwd<IO, SL, true><<<(unsigned)(blocks * (p.splits - 1)), NT, sizeof(Tile<SL>), st>>>(p);
    scan_fwd<IO, SL, false><<<(unsigned)(blocks * p.splits), NT, sizeof(Tile<SL>), st>>>(p);
    return cudaGetLastError();
}

template <typename IO>
cudaError_t pick(const ScanParams& p, cudaStream_t st) {
    const int n = p.a.states;
    if (n <= 4) return launch<IO, 1>(p, st);
    if (n <= 8) return launch<IO, 2>(p, st);
    if (n <= 16) return launch<IO, 4>(p, st);
    if (n <= 32) return launch<IO, 8>(p, st);
    if (n <= 64) return launch<IO, 16>(p, st);
    return launch<IO, 32>(p, st);
}

// Channels of a block
int block_channels(int states) {
    int sl = 1;
    while (sl * S < states) sl *= 2;
    return NT / 32 * (32 / sl);
}

}  // namespace

int state_scan_splits(long long T, long long batch, long long group_channels, int groups, int states) {
    const int bc = block_channels(states);
    const long long blocks = (group_channels + bc - 1) / bc * groups * batch;
    long long splits = 148 * 3 / (blocks > 0 ? blocks : 1);
    if (splits < 3) return 1;
    splits = std::min(splits, T / (8 * TT));
    return (int)std::max<long long>(1, splits);
}

cudaError_t state_scan_forward_launch(const ScanParams& p, cudaStream_t st) {
    switch (p.a.dtype) {
        case DFSNN_DTYPE_F16: return pick<__half>(p, st);
        case DFSNN_DTYPE_BF16: return pick<__nv_bfloat16>(p, st);
        default: return pick<float>(p, st);
    }
}

}  // namespace dfsnn
