// state_scan.h -- arguments of the selective-scan kernels, as the launchers hand them over.
#pragma once
#include "state_space.cuh"

namespace dfsnn {

constexpr int kScanTile = 16;                  // steps of a tile
constexpr int kScanChunk = DFSNN_SCAN_CHUNK;   // steps between kept states

struct ScanParams {
    dfsnn_state_scan_args a;
    dfsnn_state_scan_grads g;
    int T, group_channels;
    int tiles;                                 // channel tiles of a group
    bool words;                                // rows_aligned(4), for rows that are not on 16 bytes
    long long seq_blocks;                      // forward: blocks that share the batch
    // a sequence in parts (splits > 1): `split_steps` steps each, a multiple of the chunk
    int splits, split_steps;
    float* ends;                               // [splits][batch][channels][states] (forward: all but
    float* end_steps;                          // the last, backward: the first unused) and sums of d
    int chained;                               // backward: the parts run in order, `ends` passed on
    int* flags;                                // [tiles * groups * batch] finished parts, zeroed first
    int* places;                               // behind them: places given to blocks so far
    int patience;                              // 1; 0: every wait runs out at once (self-check)
    // backward
    int batch_parts;                           // blocks that share the batch (part q: b = q, q + parts, ...)
    float* part_bc;                            // [2][tiles][T][batch][groups][states]
    float* part_a;                             // [batch_parts * splits][channels][states]
    float* part_d;                             // [2][batch_parts * splits][channels] (D, delta_bias)
};

// Whether every row (a step's channels of a group, a step's states) of the inputs starts on a
// multiple of `bytes`.  Channel tiles start on multiples of 4 channels, whole rows of a tile.
inline bool rows_aligned(const ScanParams& p, size_t elem, size_t bytes) {
    const dfsnn_state_scan_args& a = p.a;
    auto ok = [&](const void* q, long long t, long long b, long long g) {
        return reinterpret_cast<uintptr_t>(q) % bytes == 0 && t * (long long)elem % (long long)bytes == 0
               && b * (long long)elem % (long long)bytes == 0 && g * (long long)elem % (long long)bytes == 0;
    };
    return ok(a.u, a.u_t, a.u_b, a.groups > 1 ? p.group_channels : 0) && ok(a.delta, a.delta_t, a.delta_b, 0)
           && ok(a.z, a.z_t, a.z_b, 0) && ok(a.B, a.B_t, a.B_b, a.B_g) && ok(a.C, a.C_t, a.C_b, a.C_g)
           && ok(p.g.grad_y, a.y_t, a.y_b, 0);
}

// Whether pairs of neighbouring channels of an output start on a multiple of two elements
inline bool pairs_aligned(const void* q, long long t, long long b, size_t elem) {
    return reinterpret_cast<uintptr_t>(q) % (2 * elem) == 0 && t % 2 == 0 && b % 2 == 0;
}

int state_scan_splits(long long T, long long batch, long long group_channels, int groups, int states);
cudaError_t state_scan_forward_launch(const ScanParams& p, cudaStream_t st);
int state_scan_bwd_tiles(int states, long long group_channels);
void state_scan_bwd_plan(ScanParams& p);       // sets splits, split_steps and batch_parts
cudaError_t state_scan_backward_launch(const ScanParams& p, cudaStream_t st);
cudaError_t state_scan_expired_waits(unsigned long long* count, cudaStream_t st);

}  // namespace dfsnn
