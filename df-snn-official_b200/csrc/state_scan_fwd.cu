// state_scan_fwd.cu -- forward of the selective scan.
//
//   h_t[n] = exp(d_t A[n]) h_(t-1)[n] + d_t u_t B_t[n],   o_t = sum_n C_t[n] h_t[n] + D u_t
//
// One exponential and five multiply-adds for each (step, channel, state), against 3 or 4 elements
// of traffic for all N states of a (step, channel): with N = 16 the 16 exponentials a clock of an
// SM's special-function unit are the floor, not memory.  Everything else has to fit beside them:
//   * a channel's states lie on SL lanes, four neighbouring states each, as two packed pairs (half
//     the issue slots), and a warp walks the sequence of its 32 / SL channels;
//   * steps are taken in tiles of 16, fetched a tile ahead, and the sums over a channel's lanes are
//     formed for 8 steps together (LaneSums): (1 - 1/SL) shuffles a step instead of log2 SL;
//   * the elementwise work (softplus, gate, skip) is done once per (step, channel) by all threads
//     of the block, before and after the tile;
//   * the operands of a group of steps are read from shared memory while the group before runs.
// States, decays and sums are fp32; y is rounded once.
//
// T = 2048, 8 sequences, 2048 channels, bf16, N = 16, gated: 332 us, 537 M (step, channel, state) at
// 1.62 T/s (36 % of the special-function unit's rate; issue and the shared-memory pipe are 57 %
// busy at 13 warps an SM); with 32 sequences 2.05 T/s.
//
// Few rows leave most of the machine idle, so a long sequence is then cut into `splits` parts that
// run side by side: a first launch (ENDS) walks all parts but the last from a zero state for the
// state each part adds, h_out = exp(A sum d) h_in + end, and the second folds those up to its part
// before it walks it.  That takes the exponentials twice; state_scan_splits() weighs it.
#include <algorithm>

#include "state_scan.h"
#include "state_tile.cuh"

namespace dfsnn {
namespace {

constexpr int TT = kScanTile, NT = 128;

// S states on each of a channel's SL lanes
template <typename IO, int S, int SL>
struct Tile {
    static constexpr int CL = 32 / SL;                 // channels of a warp
    static constexpr int BC = NT / 32 * CL;            // channels of the block
    static constexpr int NS = S * SL;                  // states, padded
    struct Raw {                                       // as the sequences have them
        IO u[TT][BC], d[TT][BC], z[TT][BC], B[TT][NS], C_[TT][NS];
    };
    template <int K> using Pieces = TilePieces<IO, TT, NT, K>;
    template <int COLS> static constexpr int kPieces = Pieces<1>::template kPieces<COLS>;
    static constexpr bool kEights = BC * sizeof(IO) < 16 || NS * sizeof(IO) < 16;   // rows of 8 bytes
    __align__(16) Raw raw[2];                          // this tile's and the next one's
    // (d, d u) of a channel, even channels in front of odd ones: a warp then writes the pairs of a
    // step, and reads its channels, without bank conflicts
    float2 d_[BC * (TT + 1) + 4];
    __device__ __forceinline__ float2* d(int ch) {
        return d_ + (ch >> 1) * (TT + 1) + (ch & 1) * (BC / 2 * (TT + 1) + 4);
    }
    __align__(16) float B[TT][NS], C_[TT][NS];
    float o[BC][TT + 1];
};

// S neighbouring states as pairs
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

// V neighbouring elements of a sequence
template <typename IO, int V>
struct __align__(sizeof(IO) * V) Pack {
    IO v[V];
};

template <typename IO, int S, int SL, bool WIDE, bool ENDS>
__global__ void __launch_bounds__(NT, 5) scan_fwd(const ScanParams p) {
    using Tl = Tile<IO, S, SL>;
    constexpr int CL = Tl::CL, BC = Tl::BC, NS = Tl::NS, J = S / 2;
    constexpr int V = WIDE ? 2 : 1;                             // channels of a pack
    constexpr int ROW = BC / V;                                 // threads along a step's channels
    constexpr int E = TT * ROW > NT ? TT * ROW / NT : 1;        // packs of a thread,
    constexpr int TS = TT / E;                                  // this many steps apart
    using Elem = Pack<IO, V>;
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
    const long long b0 = bid / parts;                           // sequences b0, b0 + seq_blocks, ...
    const int first = split * p.split_steps;                    // this part's steps: first .. len - 1,
    const int stop = p.T - first < p.split_steps ? p.T : first + p.split_steps;   // its rows: .. stop - 1
    if (ENDS && seq_length(a.lengths, a.lengths64, b0, p.T) <= stop) return;      // no part behind this one
    const int c_base = tile * BC;                               // within the group
    const long long g_base = (long long)grp * p.group_channels; // first channel of the group

    // elementwise role: elements (step t_e + e * TS, channels ch .. ch + V - 1)
    const int ch = tid % ROW * V, t_e = tid / ROW;
    const bool ch_ok = c_base + ch < p.group_channels && t_e < TT;
    const long long chan = g_base + c_base + ch;
    float bias[V], skip[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = ch_ok && a.delta_bias ? a.delta_bias[chan + v] : 0.0f;
        skip[v] = !ENDS && ch_ok && a.D ? a.D[chan + v] : 0.0f;
    }
    const int cols = p.group_channels - c_base;
    using Raw = typename Tl::Raw;
    constexpr int K = ((ENDS ? 2 : 3) * Tl::template kPieces<BC> + (ENDS ? 1 : 2) * Tl::template kPieces<NS> + NT - 1) / NT;
    typename Tl::template Pieces<WIDE ? K : 1> pieces;
    // the sequence that is being fetched, at the next step to fetch; tiles fetched and scanned so far
    const IO *u_p = nullptr, *d_p = nullptr, *z_p = nullptr, *B_p = nullptr, *C_p = nullptr;
    int len_ahead = 0, fetched = 0, scanned = 0;
    auto fill = [&](int t0) {
        const int stage = fetched++ & 1, rows = len_ahead - t0;
        if constexpr (WIDE) {
            pieces.template issue<Tl::kEights>(stage * (unsigned)sizeof(Raw), rows);
        } else {
            Raw& r = sh.raw[stage];
            fill_tile<IO, TT, BC, NT, false>(r.u[0], u_p, a.u_t, rows, cols, p.words);
            fill_tile<IO, TT, BC, NT, false>(r.d[0], d_p, a.delta_t, rows, cols, p.words);
            fill_tile<IO, TT, NS, NT, false>(r.B[0], B_p, a.B_t, rows, a.states, p.words);
            if (!ENDS) {
                if (a.z) fill_tile<IO, TT, BC, NT, false>(r.z[0], z_p, a.z_t, rows, cols, p.words);
                fill_tile<IO, TT, NS, NT, false>(r.C_[0], C_p, a.C_t, rows, a.states, p.words);
            }
            u_p += TT * a.u_t;
            d_p += TT * a.delta_t;
            z_p += TT * a.z_t;
            B_p += TT * a.B_t;
            C_p += TT * a.C_t;
        }
        copy_commit();
    };
    auto open = [&](long long b) {
        const int n = seq_length(a.lengths, a.lengths64, b, p.T);
        len_ahead = n < stop ? n : stop;
        u_p = static_cast<const IO*>(a.u) + b * a.u_b + g_base + c_base + first * a.u_t;
        d_p = static_cast<const IO*>(a.delta) + b * a.delta_b + g_base + c_base + first * a.delta_t;
        z_p = static_cast<const IO*>(a.z) + b * a.z_b + g_base + c_base + first * a.z_t;
        B_p = static_cast<const IO*>(a.B) + b * a.B_b + grp * a.B_g + first * a.B_t;
        C_p = static_cast<const IO*>(a.C) + b * a.C_b + grp * a.C_g + first * a.C_t;
        if constexpr (WIDE) {
            Raw& r = sh.raw[0];
            pieces.clear();
            pieces.template add<BC>(r.u, u_p, a.u_t, cols);
            pieces.template add<BC>(r.d, d_p, a.delta_t, cols);
            pieces.template add<NS>(r.B, B_p, a.B_t, a.states);
            if (!ENDS) {
                pieces.template add<NS>(r.C_, C_p, a.C_t, a.states);
                if (a.z) pieces.template add<BC>(r.z, z_p, a.z_t, cols);
            }
        }
        if (first < len_ahead) fill(first);
    };
    open(b0);                                                   // in flight while the states are set up

    // recurrence role: states n0 .. n0 + S - 1 of channel cl of the block
    const int sl = lane / CL, cl = warp * CL + lane % CL, n0 = sl * S;
    auto cl_ok = [&]() { return c_base + cl < p.group_channels; };
    // a lane's states are one 16-byte access everywhere
    const bool whole = S == 4 && a.states % 4 == 0
                       && ((reinterpret_cast<uintptr_t>(a.kept) | reinterpret_cast<uintptr_t>(a.h_last)) & 15) == 0;
    float2 A2[J] = {}, h[J] = {};
    auto get = [&](const float* q, float2(&v)[J]) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const float f = q && cl_ok() && n0 + s < a.states ? q[s] : 0.0f;
            (s % 2 ? v[s / 2].y : v[s / 2].x) = f;
        }
    };
    auto put = [&](float* q) {
        if (!cl_ok() || n0 >= a.states) return;
        if (S == 4 && whole) {
            *reinterpret_cast<float4*>(q) = make_float4(h[0].x, h[0].y, h[J - 1].x, h[J - 1].y);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (n0 + s < a.states) q[s] = s % 2 ? h[s / 2].y : h[s / 2].x;
        }
    };
    get(a.A + (g_base + c_base + cl) * a.states + n0, A2);
#pragma unroll
    for (int j = 0; j < J; ++j) A2[j] = make_float2(log2_rate(A2[j].x), log2_rate(A2[j].y));

    for (long long b = b0; b < a.batch; b += p.seq_blocks) {
    const int whole_len = seq_length(a.lengths, a.lengths64, b, p.T), len = whole_len < stop ? whole_len : stop;
    const long long row = (b * a.channels + g_base + c_base + cl) * a.states + n0;
    const bool another = b + p.seq_blocks < a.batch;            // its first tile is fetched during our last
    IO* y_p = static_cast<IO*>(a.y) + b * a.y_b + chan + (first + t_e) * a.y_t;
    if constexpr (ENDS) {
    } else if (first < whole_len) {
        get(a.h0 ? a.h0 + row : nullptr, h);
        const long long rows = a.batch * a.channels;
        for (int k = 0; k != split; ++k) {
            float2 end[J] = {};
            get(p.ends + k * rows * a.states + row, end);
            const float half = cl_ok() ? 0.5f * p.end_steps[k * rows + b * a.channels + g_base + c_base + cl] : 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j)
                h[j] = make_float2(carry_over(half * A2[j].x, h[j].x, end[j].x), carry_over(half * A2[j].y, h[j].y, end[j].y));
        }
    } else if (split == 0) {
        get(a.h0 ? a.h0 + row : nullptr, h);                    // an empty sequence keeps its state
    }
    float steps = 0.0f;                                         // sum of d
    const long long all_states = a.batch * a.channels * a.states;
    float* kept = a.kept + row - all_states;                    // of step t at t / R * all_states

    for (int t0 = first; t0 < len; t0 += TT) {
        const Raw& raw = sh.raw[scanned++ & 1];
        copy_wait<0>();
        __syncthreads();
        if (t0 + TT < len) fill(t0 + TT);
        else if (another) open(b + p.seq_blocks);
        const bool tail = t0 + TT > len;
        if (t_e < TT) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int t = t_e + e * TS;
                const Elem u = *reinterpret_cast<const Elem*>(&raw.u[t][ch]);
                const Elem d = *reinterpret_cast<const Elem*>(&raw.d[t][ch]);
                float2 dt = make_float2(to_f(d.v[0]) + bias[0], to_f(d.v[V - 1]) + bias[V - 1]);
                if (a.softplus) dt = softplus_f(dt);
                if (tail && t0 + t >= len) dt = make_float2(0.0f, 0.0f);   // a step behind the end leaves the state alone
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float x = v ? dt.y : dt.x;
                    sh.d(ch + v)[t] = make_float2(x, x * to_f(u.v[v]));
                }
            }
        }
#pragma unroll
        for (int i = tid; i < TT * NS; i += NT) {
            sh.B[0][i] = to_f(raw.B[0][i]);
            if (!ENDS) sh.C_[0][i] = to_f(raw.C_[0][i]);
        }
        __syncthreads();
        // decays that stay near 1 for the whole tile take the polynomial
        bool near1[S];
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < TT; t += SL)
            if (SL <= TT || sl < TT) most = fmaxf(most, fabsf(sh.d(cl)[t + (SL <= TT ? sl : sl % TT)].x));
#pragma unroll
        for (int m = SL / 2; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m * CL));
#pragma unroll
        for (int j = 0; j < J; ++j) {
            near1[2 * j] = most * fabsf(A2[j].x) < kExp2Near;
            near1[2 * j + 1] = most * fabsf(A2[j].y) < kExp2Near;
        }
        constexpr int R = 8;                    // steps whose sums over the lanes are formed together
        constexpr int G = 2;                    // steps whose operands are read one group ahead
        static_assert(R == kScanChunk, "states are kept in front of every R steps");
        float2 d_n[G], B_n[G][J], C_n[G][J];
        auto read = [&](int t0g) {
#pragma unroll
            for (int t = 0; t < G; ++t) {
                load_states<S>(B_n[t], &sh.B[t0g + t][n0]);
                if (!ENDS) load_states<S>(C_n[t], &sh.C_[t0g + t][n0]);
                d_n[t] = sh.d(cl)[t0g + t];
            }
        };
        read(0);
#pragma unroll
        for (int tr = 0; tr < TT; tr += R) {
            if (!ENDS && a.kept && t0 + tr > 0 && t0 + tr < len)
                put(kept + (long long)((t0 + tr) / R) * all_states);
            float y[R];
#pragma unroll
            for (int tg = 0; tg < R; tg += G) {
                float2 d_c[G], B_c[G][J], C_c[G][J];
#pragma unroll
                for (int t = 0; t < G; ++t) {
                    d_c[t] = d_n[t];
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        B_c[t][j] = B_n[t][j];
                        if (!ENDS) C_c[t][j] = C_n[t][j];
                    }
                }
                if (tr + tg + G < TT) read(tr + tg + G);
                float2 dec[G][J], in[G][J];
#pragma unroll
                for (int t = 0; t < G; ++t) {
                    const float2 dt = make_float2(d_c[t].x, d_c[t].x), du = make_float2(d_c[t].y, d_c[t].y);
                    if (ENDS) steps += d_c[t].x;
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float2 x = __fmul2_rn(dt, A2[j]), q = exp2_near1(x);
                        dec[t][j] = make_float2(near1[2 * j] ? q.x : exp2_approx(x.x),
                                                near1[2 * j + 1] ? q.y : exp2_approx(x.y));
                        in[t][j] = __fmul2_rn(du, B_c[t][j]);
                    }
                }
#pragma unroll
                for (int t = 0; t < G; ++t) {
                    float2 acc;
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        h[j] = __ffma2_rn(dec[t][j], h[j], in[t][j]);
                        if (!ENDS) acc = j == 0 ? __fmul2_rn(h[j], C_c[t][j]) : __ffma2_rn(h[j], C_c[t][j], acc);
                    }
                    if (!ENDS) y[tg + t] = acc.x + acc.y;
                }
            }
            if (!ENDS) {
                using Sums = LaneSums<R, SL, CL>;
                Sums::run(y, sl);
                if (Sums::stores(sl)) {
#pragma unroll
                    for (int i = 0; i < Sums::kHeld; ++i) sh.o[cl][tr + Sums::first(sl) + i] = y[i];
                }
            }
        }
        if (ENDS) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = t_e + e * TS;
            if (ch_ok && (!tail || t0 + t < stop)) {
                const Elem u = *reinterpret_cast<const Elem*>(&raw.u[t][ch]);
                const Elem z = *reinterpret_cast<const Elem*>(&raw.z[t][ch]);
                float2 o = make_float2(fmaf(skip[0], to_f(u.v[0]), sh.o[ch][t]),
                                       fmaf(skip[V - 1], to_f(u.v[V - 1]), sh.o[ch + V - 1][t]));
                if (a.z) {
                    const float2 zf = make_float2(to_f(z.v[0]), to_f(z.v[V - 1]));
                    o = __fmul2_rn(o, __fmul2_rn(zf, sigmoid_f(zf)));
                }
                if (tail && t0 + t >= len) o = make_float2(0.0f, 0.0f);
                Elem out;
                out.v[0] = from_f<IO>(o.x);
                out.v[V - 1] = from_f<IO>(V == 1 ? o.x : o.y);
                *reinterpret_cast<Elem*>(y_p) = out;
            }
            y_p += TS * a.y_t;
        }
    }
    if (first >= len && another) open(b + p.seq_blocks);
    if (ENDS) {
        put(p.ends + split * a.batch * a.channels * a.states + row);
        if (cl_ok() && sl == 0) p.end_steps[(split * a.batch + b) * a.channels + g_base + c_base + cl] = steps;
        return;
    }
    // rows behind the end (y_p is at the tile behind the last)
    if (ch_ok) {
        Elem none;
#pragma unroll
        for (int v = 0; v < V; ++v) none.v[v] = from_f<IO>(0.0f);
        const int done = len > first ? first + (len - first + TT - 1) / TT * TT : first;
        for (long long t = done + t_e; t < stop; t += TS, y_p += TS * a.y_t)
            *reinterpret_cast<Elem*>(y_p) = none;
    }
    if (a.h_last && (first < whole_len ? whole_len <= stop : split == 0 && whole_len == 0)) put(a.h_last + row);
    }
}

template <typename IO, int S, int SL, bool WIDE>
cudaError_t launch_form(const ScanParams& p, unsigned blocks, cudaStream_t st) {
    constexpr size_t smem = sizeof(Tile<IO, S, SL>);
    cudaError_t e = allow_shared<scan_fwd<IO, S, SL, WIDE, false>>(smem);
    if (e == cudaSuccess && p.splits > 1) e = allow_shared<scan_fwd<IO, S, SL, WIDE, true>>(smem);
    if (e != cudaSuccess) return e;
    if (p.splits > 1)
        scan_fwd<IO, S, SL, WIDE, true><<<blocks * (p.splits - 1), NT, smem, st>>>(p);
    scan_fwd<IO, S, SL, WIDE, false><<<blocks * p.splits, NT, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename IO, int S, int SL>
cudaError_t launch(ScanParams p, cudaStream_t st) {
    constexpr int BC = Tile<IO, S, SL>::BC;
    p.tiles = (p.group_channels + BC - 1) / BC;
    // Short sequences: one wave of blocks (five an SM) takes them all, several a block, so that the
    // set-up is paid once and the next sequence is fetched meanwhile (16 steps, 4096 sequences, 256
    // channels, fp32: 173 us against 205 with a block for each).
    const long long per = (long long)p.tiles * p.a.groups, slots = 148 * 5;
    p.seq_blocks = p.a.batch;
    if (p.T <= 4 * TT && per * p.a.batch >= 4 * slots && per <= slots) p.seq_blocks = slots / per;
    const long long blocks = per * p.seq_blocks;
    if (blocks > 0x7fffffffLL / p.splits) return cudaErrorInvalidValue;
    const dfsnn_state_scan_args& a = p.a;
    p.words = rows_aligned(p, sizeof(IO), 4);
    return p.group_channels % 2 == 0 && pairs_aligned(a.y, a.y_t, a.y_b, sizeof(IO)) && rows_aligned(p, sizeof(IO), 16) ? launch_form<IO, S, SL, true>(p, (unsigned)blocks, st)
                                                    : launch_form<IO, S, SL, false>(p, (unsigned)blocks, st);
}

template <typename IO>
cudaError_t pick(const ScanParams& p, cudaStream_t st) {
    const int n = p.a.states;
    if (n <= 4) return launch<IO, 2, 2>(p, st);
    if (n <= 8) return launch<IO, 2, 4>(p, st);
    if (n <= 16) return launch<IO, 4, 4>(p, st);
    if (n <= 32) return launch<IO, 4, 8>(p, st);
    if (n <= 64) return launch<IO, 4, 16>(p, st);
    return launch<IO, 4, 32>(p, st);
}

// Channels of a block, as pick() has them
int block_channels(int states) {
    if (states <= 4) return Tile<float, 2, 2>::BC;
    if (states <= 8) return Tile<float, 2, 4>::BC;
    if (states <= 16) return Tile<float, 4, 4>::BC;
    if (states <= 32) return Tile<float, 4, 8>::BC;
    if (states <= 64) return Tile<float, 4, 16>::BC;
    return Tile<float, 4, 32>::BC;
}

}  // namespace

// Parts of a sequence.  Five blocks run on an SM at a time; while a whole walk of each sequence
// would leave room for three times the blocks, parts pay for their second walk: 4096 steps, bf16,
// N = 16, microseconds in parts and whole: 512 channels 51 and 319, 2048 channels 135 and 322, 5888
// channels (184 blocks) 322 and 426.  Parts are 4 tiles at least.
int state_scan_splits(long long T, long long batch, long long group_channels, int groups, int states) {
    const int bc = block_channels(states);
    const long long blocks = (group_channels + bc - 1) / bc * groups * batch;
    long long splits = 148 * 5 / (blocks > 0 ? blocks : 1);
    if (splits < 3) return 1;
    splits = std::min(splits, T / (4 * TT));
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
