// state_capi.cu -- extern "C" entry points of the state-space layer (include/dfsnn_b200.h):
// argument checks (nothing is launched on a bad call), workspace layout, launches.
#include <climits>

#include "kernels.h"
#include "short_conv.h"
#include "state_scan.h"

namespace dfsnn {
cudaError_t state_scan_step_launch(const dfsnn_state_scan_step_args& a, cudaStream_t st);
}

namespace {

constexpr long long kMaxSteps = INT_MAX - 1024;     // tile arithmetic stays in 32 bits

int status(cudaError_t e) { return e == cudaSuccess ? DFSNN_OK : dfsnn::record_cuda_error(e); }

bool known_dtype(int d) {
    return d == DFSNN_DTYPE_F32 || d == DFSNN_DTYPE_F16 || d == DFSNN_DTYPE_BF16;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool flag(int v) { return v == 0 || v == 1; }

int check_scan_sizes(long long T, long long batch, long long channels, int states, int groups) {
    if (T < 1 || batch < 0 || channels < 0 || states < 1 || groups < 1) return DFSNN_ERR_SHAPE;
    if (channels > INT_MAX - 1024 || channels % groups) return DFSNN_ERR_SHAPE;
    if (T > kMaxSteps || states > DFSNN_SCAN_MAX_STATES) return DFSNN_ERR_T_LIMIT;
    return DFSNN_OK;
}

int check_scan(const dfsnn_state_scan_args* a) {
    if (!a) return DFSNN_ERR_NULL;
    if (int s = check_scan_sizes(a->T, a->batch, a->channels, a->states, a->groups)) return s;
    if (!known_dtype(a->dtype) || !flag(a->softplus) || !flag(a->lengths64)) return DFSNN_ERR_PARAM;
    return DFSNN_OK;
}

// Parts of the forward, and their floats in the workspace: [splits - 1] states and sums of d
int forward_splits(const dfsnn_state_scan_args& a) {
    return dfsnn::state_scan_splits(a.T, a.batch, a.channels / a.groups, a.groups, a.states);
}
size_t forward_floats(int splits, long long batch, long long channels, int states) {
    return (size_t)(splits - 1) * batch * channels * (states + 1);
}

dfsnn::ScanParams scan_params(const dfsnn_state_scan_args& a) {
    dfsnn::ScanParams p{};
    p.a = a;
    p.T = (int)a.T;
    p.group_channels = (int)(a.channels / a.groups);
    p.splits = 1;
    p.split_steps = p.T;
    p.patience = 1;
    return p;
}

struct ScanWorkspace {
    size_t bc, a, d, ends, end_steps, flags;       // 4-byte words
    size_t bytes() const { return (bc + a + d + ends + end_steps + flags) * sizeof(float); }
};

ScanWorkspace backward_plan(dfsnn::ScanParams& p) {
    p.tiles = dfsnn::state_scan_bwd_tiles(p.a.states, p.group_channels);
    dfsnn::state_scan_bwd_plan(p);
    const size_t rows = (size_t)p.a.batch * p.a.channels, parts = (size_t)p.batch_parts * p.splits;
    ScanWorkspace w;
    w.bc = (size_t)2 * p.tiles * p.a.T * p.a.batch * p.a.groups * p.a.states;
    w.a = parts * p.a.channels * p.a.states;
    w.d = 2 * parts * p.a.channels;
    w.ends = p.splits > 1 ? p.splits * rows * p.a.states : 0;
    w.end_steps = p.splits > 1 && !p.chained ? p.splits * rows : 0;
    w.flags = p.chained ? (size_t)p.tiles * p.a.groups * p.batch_parts + 1 : 0;
    return w;
}

int backward(const dfsnn_state_scan_args* a, const dfsnn_state_scan_grads* g, void* workspace,
             size_t workspace_bytes, int patience, void* stream) {
    if (int s = check_scan(a)) return s;
    if (!g) return DFSNN_ERR_NULL;
    if (a->batch == 0 || a->channels == 0) return DFSNN_OK;
    if (!a->u || !a->delta || !a->A || !a->B || !a->C || !g->grad_y || !g->grad_u || !g->grad_delta
        || !g->grad_B || !g->grad_C || !g->grad_A)
        return DFSNN_ERR_NULL;
    if (!a->kept && a->T > DFSNN_SCAN_CHUNK) return DFSNN_ERR_NULL;
    dfsnn::ScanParams p = scan_params(*a);
    p.g = *g;
    p.patience = patience;
    const ScanWorkspace w = backward_plan(p);
    if (!workspace || !aligned16(workspace) || workspace_bytes < w.bytes()) return DFSNN_ERR_WORKSPACE;
    p.part_bc = static_cast<float*>(workspace);
    p.part_a = p.part_bc + w.bc;
    p.part_d = p.part_a + w.a;
    p.ends = p.part_d + w.d;
    p.end_steps = p.ends + w.ends;
    p.flags = reinterpret_cast<int*>(p.end_steps + w.end_steps);
    p.places = p.flags + (w.flags ? w.flags - 1 : 0);
    return status(dfsnn::state_scan_backward_launch(p, (cudaStream_t)stream));
}

}  // namespace

extern "C" {

size_t dfsnn_state_scan_kept_floats(long long T, long long batch, long long channels, int states) {
    if (check_scan_sizes(T, batch, channels, states, 1)) return 0;
    return (size_t)((T - 1) / DFSNN_SCAN_CHUNK) * batch * channels * states;
}

size_t dfsnn_state_scan_forward_workspace_size(long long T, long long batch, long long channels,
                                               int states, int groups) {
    if (check_scan_sizes(T, batch, channels, states, groups) || batch == 0 || channels == 0) return 0;
    const int splits = dfsnn::state_scan_splits(T, batch, channels / groups, groups, states);
    return forward_floats(splits, batch, channels, states) * sizeof(float);
}

int dfsnn_state_scan_forward(const dfsnn_state_scan_args* a, void* workspace, size_t workspace_bytes,
                             void* stream) {
    if (int s = check_scan(a)) return s;
    if (a->batch == 0 || a->channels == 0) return DFSNN_OK;
    if (!a->u || !a->delta || !a->A || !a->B || !a->C || !a->y) return DFSNN_ERR_NULL;
    dfsnn::ScanParams p = scan_params(*a);
    p.splits = forward_splits(*a);
    if (p.splits > 1) {
        const size_t need = forward_floats(p.splits, a->batch, a->channels, a->states) * sizeof(float);
        if (!workspace || !aligned16(workspace) || workspace_bytes < need) return DFSNN_ERR_WORKSPACE;
        const long long chunks = (a->T + DFSNN_SCAN_CHUNK - 1) / DFSNN_SCAN_CHUNK;
        const long long per = (chunks + p.splits - 1) / p.splits;
        p.split_steps = (int)(per * DFSNN_SCAN_CHUNK);
        p.ends = static_cast<float*>(workspace);
        p.end_steps = p.ends + (size_t)(p.splits - 1) * a->batch * a->channels * a->states;
        p.splits = (int)((chunks + per - 1) / per);
    }
    return status(dfsnn::state_scan_forward_launch(p, (cudaStream_t)stream));
}

size_t dfsnn_state_scan_backward_workspace_size(long long T, long long batch, long long channels,
                                                int states, int groups) {
    if (check_scan_sizes(T, batch, channels, states, groups) || batch == 0 || channels == 0) return 0;
    dfsnn_state_scan_args a{};
    a.T = T;
    a.batch = batch;
    a.channels = channels;
    a.states = states;
    a.groups = groups;
    dfsnn::ScanParams p = scan_params(a);
    return backward_plan(p).bytes();
}

int dfsnn_state_scan_backward_launches(long long T, long long batch, long long channels, int states,
                                       int groups) {
    if (check_scan_sizes(T, batch, channels, states, groups) || batch == 0 || channels == 0) return 0;
    dfsnn_state_scan_args a{};
    a.T = T;
    a.batch = batch;
    a.channels = channels;
    a.states = states;
    a.groups = groups;
    dfsnn::ScanParams p = scan_params(a);
    backward_plan(p);
    return p.splits > 1 && !p.chained ? 3 : 2;
}

int dfsnn_state_scan_backward(const dfsnn_state_scan_args* a, const dfsnn_state_scan_grads* g,
                              void* workspace, size_t workspace_bytes, void* stream) {
    return backward(a, g, workspace, workspace_bytes, 1, stream);
}

int dfsnn_check_state_scan_waits(const dfsnn_state_scan_args* a, const dfsnn_state_scan_grads* g,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    return backward(a, g, workspace, workspace_bytes, 0, stream);
}

int dfsnn_state_scan_expired_waits(unsigned long long* count, void* stream) {
    if (!count) return DFSNN_ERR_NULL;
    return status(dfsnn::state_scan_expired_waits(count, (cudaStream_t)stream));
}

int dfsnn_state_scan_step(const dfsnn_state_scan_step_args* a, void* stream) {
    if (!a) return DFSNN_ERR_NULL;
    if (int s = check_scan_sizes(1, a->batch, a->channels, a->states, a->groups)) return s;
    if (a->slots < 0 || (!a->index && a->slots < a->batch)) return DFSNN_ERR_SHAPE;
    if (!known_dtype(a->dtype) || !flag(a->softplus) || !flag(a->index64)) return DFSNN_ERR_PARAM;
    if (a->batch == 0 || a->channels == 0) return DFSNN_OK;
    if (!a->u || !a->delta || !a->A || !a->B || !a->C || !a->state || !a->state_out || !a->y)
        return DFSNN_ERR_NULL;
    return status(dfsnn::state_scan_step_launch(*a, (cudaStream_t)stream));
}

static int check_conv_sizes(long long T, long long batch, long long channels, int taps) {
    if (T < 1 || batch < 0 || channels < 0 || channels > INT_MAX - 1024) return DFSNN_ERR_SHAPE;
    if (T > kMaxSteps || taps < 1 || taps > DFSNN_CONV_MAX_TAPS) return DFSNN_ERR_T_LIMIT;
    return DFSNN_OK;
}

static int check_conv(const dfsnn_short_conv_args* a) {
    if (!a) return DFSNN_ERR_NULL;
    if (int s = check_conv_sizes(a->T, a->batch, a->channels, a->taps)) return s;
    if (!known_dtype(a->dtype) || !flag(a->silu) || !flag(a->lengths64)) return DFSNN_ERR_PARAM;
    return DFSNN_OK;
}

int dfsnn_short_conv_forward(const dfsnn_short_conv_args* a, void* stream) {
    if (int s = check_conv(a)) return s;
    if (a->batch == 0 || a->channels == 0) return DFSNN_OK;
    if (!a->x || !a->weight || !a->y) return DFSNN_ERR_NULL;
    return status(dfsnn::short_conv_forward_launch(*a, (cudaStream_t)stream));
}

size_t dfsnn_short_conv_backward_workspace_size(long long T, long long batch, long long channels,
                                                int taps) {
    if (check_conv_sizes(T, batch, channels, taps) || batch == 0 || channels == 0) return 0;
    return (size_t)dfsnn::short_conv_parts(T, batch, channels) * (taps + 1) * channels * sizeof(float);
}

int dfsnn_short_conv_backward(const dfsnn_short_conv_args* a, const dfsnn_short_conv_grads* g,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if (int s = check_conv(a)) return s;
    if (!g) return DFSNN_ERR_NULL;
    if (a->batch == 0 || a->channels == 0) return DFSNN_OK;
    if (!a->x || !a->weight || !g->grad_y || !g->grad_x || !g->grad_weight) return DFSNN_ERR_NULL;
    const size_t need = dfsnn_short_conv_backward_workspace_size(a->T, a->batch, a->channels, a->taps);
    if (!workspace || !aligned16(workspace) || workspace_bytes < need) return DFSNN_ERR_WORKSPACE;
    return status(dfsnn::short_conv_backward_launch(*a, *g, static_cast<float*>(workspace),
                                                    (cudaStream_t)stream));
}

int dfsnn_short_conv_step(const dfsnn_short_conv_step_args* a, void* stream) {
    if (!a) return DFSNN_ERR_NULL;
    if (int s = check_conv_sizes(1, a->batch, a->channels, a->taps)) return s;
    if (a->slots < 0 || (!a->index && a->slots < a->batch)) return DFSNN_ERR_SHAPE;
    if (!known_dtype(a->dtype) || !flag(a->silu) || !flag(a->index64)) return DFSNN_ERR_PARAM;
    if (a->batch == 0 || a->channels == 0) return DFSNN_OK;
    if (!a->x || !a->weight || !a->y) return DFSNN_ERR_NULL;
    if (a->taps > 1 && (!a->state || !a->state_out)) return DFSNN_ERR_NULL;
    return status(dfsnn::short_conv_step_launch(*a, (cudaStream_t)stream));
}

}  // extern "C"
