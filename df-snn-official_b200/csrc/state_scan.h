// state_scan.h -- arguments of the selective-scan kernels, as the launchers hand them over.
#pragma once
#include "state_space.cuh"

namespace dfsnn {

constexpr int kScanChunk = DFSNN_SCAN_CHUNK;   // steps of a tile
constexpr int kScanPitch = kScanChunk + 4;     // floats of a row in shared memory: 16-byte rows,
                                               // eight of which start on different banks

struct ScanParams {
    dfsnn_state_scan_args a;
    dfsnn_state_scan_grads g;
    int T, group_channels;
    int tiles;                                 // channel tiles of a group
    // a sequence in parts (splits > 1): `split_steps` steps each, a multiple of the chunk
    int splits, split_steps;
    float* ends;                               // [splits - 1][batch][channels][states]
    float* end_steps;                          // [splits - 1][batch][channels] sums of d
    // backward
    int batch_parts;                           // blocks that share the batch (part q: b = q, q + parts, ...)
    float* part_bc;                            // [2][tiles][T][batch][groups][states]
    float* part_a;                             // [batch_parts][channels][states]
    float* part_d;                             // [2][batch_parts][channels] (D, delta_bias)
};

int state_scan_splits(long long T, long long batch, long long group_channels, int groups, int states);
cudaError_t state_scan_forward_launch(const ScanParams& p, cudaStream_t st);
int state_scan_bwd_tiles(int states, long long group_channels);
int state_scan_bwd_batch_parts(int states, long long batch, long long group_channels, int groups);
cudaError_t state_scan_backward_launch(const ScanParams& p, cudaStream_t st);

}  // namespace dfsnn
