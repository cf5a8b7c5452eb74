// short_conv.h -- arguments of the short-convolution kernels, as the launchers hand them over.
#pragma once
#include "state_space.cuh"

namespace dfsnn {

struct ConvParams {
    dfsnn_short_conv_args a;
    dfsnn_short_conv_grads g;
    long long run, runs, items;     // steps of a run, runs of a sequence, runs of the batch
    int channel_blocks, parts;      // blocks along the channels; blocks that share the items (backward)
    float* part;                    // [parts][taps + 1][channels]
};

cudaError_t short_conv_forward_launch(const dfsnn_short_conv_args& a, cudaStream_t st);
int short_conv_parts(long long T, long long batch, long long channels);
cudaError_t short_conv_backward_launch(const dfsnn_short_conv_args& a, const dfsnn_short_conv_grads& g,
                                       float* part, cudaStream_t st);
cudaError_t short_conv_step_launch(const dfsnn_short_conv_step_args& a, cudaStream_t st);

}  // namespace dfsnn
