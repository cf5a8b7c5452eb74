"""State-space layer on B200: selective scan, short causal convolution and their step forms.

The linear recurrence of state-space sequence models, beside this package's neuron
recurrences and over the same time-major sequences, [T, B, D] (T steps, B sequences, D
channels):

  short_conv       p_t = bias + sum_j weight[:, j] x_(t-W+1+j);  y = p or silu(p)
  state_scan       d_t = softplus(delta_t + delta_bias)
                   h_t = exp(d_t A) h_(t-1) + d_t u_t B_t        (N states for each channel)
                   y_t = (C_t . h_t + D u_t) silu(z_t)
  short_conv_step, state_scan_step: one token for each row of a batch, on states that the
                   caller keeps (one for each row, or a pool with an index)
  StateSpaceLayer  the module around them: projections, convolution, scan

The sequence forms are differentiable in every floating-point input (backwards; forward-mode
tangents are refused).  Sequences are float32, float16 or bfloat16 (one type a call) with any
strides over T and B, so halves of a projection and transposed batch-first tensors are read in
place; outputs and gradients are dense in the order of the tensor they belong to.  Parameters,
states and sums are float32.  There is no CPU path.

All calls launch on the current stream of their tensors' device, wait for nothing and can be
captured into a CUDA graph.  As with any torch operation, a backward can be captured only while
no eager graph of the same leaves is alive (torch makes the leaves' gradient nodes wait for the
stream of that graph, which a capture refuses): drop such outputs first.
"""
import ctypes
import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad as _fw
from torch.autograd.function import once_differentiable

from . import _capi
from . import profiling as _prof

_DTYPES = {torch.float32: _capi.DTYPE_F32, torch.float16: _capi.DTYPE_F16,
           torch.bfloat16: _capi.DTYPE_BF16}
_ACTIVATIONS = (None, "silu")


# ---------------------------------------------------------------------------------------
# argument checks.  They run on every call of a token loop, so each is one comparison for a good
# argument; what is wrong with a bad one is worked out afterwards.
# ---------------------------------------------------------------------------------------
def _lead(x, name, dims):
    """The sequence that sets a call's shape, type and device."""
    if not x.is_cuda:
        raise RuntimeError(f"{name} requires CUDA tensors")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: float32, float16 or bfloat16 sequences, got {x.dtype}")
    if x.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got {tuple(x.shape)}")
    return x if x.stride(-1) == 1 else _rows(x)


def _rows(x):
    return x if x.stride(-1) == 1 or x.size(-1) == 1 else x.contiguous()


def _seq(x, dtype, dev, shape, name, what):
    """A further sequence of the call: same type and device, given shape, unit last stride."""
    if x.dtype is not dtype or x.get_device() != dev or x.shape != shape:
        raise ValueError(f"{name}: {what} must be {dtype} {tuple(shape)} on cuda:{dev}, got {x.dtype} "
                         f"{tuple(x.shape)} on {x.device}")
    return x if x.stride(-1) == 1 else _rows(x)


def _param(x, dev, shape, name, what):
    """A float32 parameter or state (converted if need be), dense."""
    if x is None:
        return None
    if x.get_device() != dev or x.shape != shape or not x.dtype.is_floating_point:
        raise ValueError(f"{name}: {what} must be floating-point {tuple(shape)} on cuda:{dev}, got "
                         f"{x.dtype} {tuple(x.shape)} on {x.device}")
    if x.dtype is not torch.float32:
        x = x.float()
    return x if x.is_contiguous() else x.contiguous()


def _integers(x, dev, count, name, what):
    if x is None:
        return None
    if x.dtype not in (torch.int32, torch.int64) or x.shape != (count,) or x.get_device() != dev:
        raise ValueError(f"{name}: {what} must be int32 or int64 [{count}] on cuda:{dev}, got "
                         f"{x.dtype} {tuple(x.shape)} on {x.device}")
    return x if x.is_contiguous() else x.contiguous()


def _groups(x, dtype, dev, lead, name, what):
    """B or C as [..., G, N]; [..., N] is one group."""
    if x.dim() == len(lead) + 1:
        x = x.unsqueeze(-2)
    if x.dim() != len(lead) + 2:
        raise ValueError(f"{name}: {what} must be {tuple(lead)} + ([groups,] states), got {tuple(x.shape)}")
    return _seq(x, dtype, dev, (*lead, *x.shape[-2:]), name, what)


def _scan_sizes(D, A, B, C, name):
    if A.dim() != 2 or A.shape[0] != D:
        raise ValueError(f"{name}: A must have shape ({D}, states), got {tuple(A.shape)}")
    N, G = A.shape[1], B.shape[-2]
    if B.shape[-1] != N or C.shape != B.shape:
        raise ValueError(f"{name}: B and C must agree and have {N} states, got {tuple(B.shape)} and "
                         f"{tuple(C.shape)}")
    if not 1 <= N <= _capi.SCAN_MAX_STATES:
        raise ValueError(f"{name}: 1 to {_capi.SCAN_MAX_STATES} states, got {N}")
    if G < 1 or D % G:
        raise ValueError(f"{name}: {D} channels do not divide into {G} groups")
    return N, G


def _taps(weight, D, name):
    if weight.dim() != 2 or weight.shape[0] != D:
        raise ValueError(f"{name}: weight must have shape ({D}, taps), got {tuple(weight.shape)}")
    W = weight.shape[1]
    if not 1 <= W <= _capi.CONV_MAX_TAPS:
        raise ValueError(f"{name}: 1 to {_capi.CONV_MAX_TAPS} taps, got {W}")
    return W


def _silu_flag(activation, name):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{name}: activation must be None or 'silu', got {activation!r}")
    return int(activation == "silu")


def _slots(x, dtype, dev, inner, name, what):
    """Checks a pool of states [slots, *inner] and returns (slots, stride).  Slots may lie anywhere
    along dimension 0 (one layer of a pool for several), but each is dense: they are written in
    place."""
    if x.dtype is not dtype or x.get_device() != dev or x.dim() != 3 or x.shape[1:] != inner:
        raise ValueError(f"{name}: {what} must be {dtype} [slots, {inner[0]}, {inner[1]}] on cuda:{dev}, "
                         f"got {x.dtype} {tuple(x.shape)} on {x.device}")
    stride = x.stride()
    if stride[1:] != (inner[1], 1) and x.numel() and x.shape[1:] != (1, 1):
        raise ValueError(f"{name}: each slot of {what} must be contiguous")
    if stride[0] < inner[0] * inner[1] and x.shape[0] > 1:
        raise ValueError(f"{name}: the slots of {what} overlap")
    if x.requires_grad:
        raise ValueError(f"{name}: {what} is written in place and cannot require a gradient")
    return x.shape[0], stride[0]


def _pool(state, state_out, dtype, dev, inner, rows, index, name):
    """(state_out, slots, strides) of a step call."""
    slots, stride = _slots(state, dtype, dev, inner, name, "state")
    if state_out is None or state_out is state:
        state_out, out_stride = state, stride
    else:
        out_slots, out_stride = _slots(state_out, dtype, dev, inner, name, "state_out")
        if out_slots != slots:
            raise ValueError(f"{name}: state_out must have {slots} slots, got {out_slots}")
    if index is None and slots < rows:
        raise ValueError(f"{name}: {rows} rows need as many slots, got {slots}")
    # as torch's in-place operations do, with or without gradients: a sequence call that saved these
    # states (h0, the convolution's inputs) then refuses its backward
    if not state_out.is_inference():
        torch.autograd.graph.increment_version(state_out)
    return state_out, slots, stride, out_stride


def _no_tangents(name, tensors):
    """Refuses inputs with forward-mode tangents: they do not require a gradient, so a call would
    pass them by and return a zero derivative."""
    if _fw._current_level >= 0 and any(t is not None and _fw.unpack_dual(t).tangent is not None
                                       for t in tensors):
        raise NotImplementedError(f"{name}: forward-mode differentiation is not supported")


def _no_gradients(name, tensors):
    """Refuses what a step form could only cut off from its graph, as torch does for `out=`."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} is not differentiable, but an input requires a gradient: call it "
                                   "under torch.no_grad(), or the sequence form with one step")


# ---------------------------------------------------------------------------------------
# calls
# ---------------------------------------------------------------------------------------
def _call(fn, name, launches, nbytes, dev, *args):
    """One native call on the current stream of device number `dev`."""
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _call(fn, name, launches, nbytes, dev, *args)
    if _prof._ACTIVE is None:
        code = fn(*args, _raw_stream(dev))
    else:
        with _prof.native_call(name, launches, nbytes(), torch.device("cuda", dev)):
            code = fn(*args, _raw_stream(dev))
    if code:
        _capi.check(code, name)


def _raw_stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream = torch._C._cuda_getCurrentRawStream    # the same number without a Stream object


def _p(t):
    return 0 if t is None else t.data_ptr()


def _tb(t):
    return (0, 0) if t is None else t.stride()[:2]


def _empty_like(x):
    """Dense, in the order of x (batch-first in memory where x is), with unit last stride."""
    y = torch.empty_like(x)
    if y.stride(-1) != 1 and y.size(-1) != 1:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    return y


def _scan_args(u, delta, A, B, C, D, z, bias, h0, lengths, softplus, y, y_strides, h_last, kept):
    T, Bn, Dn = u.shape
    return _capi.STATE_SCAN_ARGS.pack(
        u.data_ptr(), delta.data_ptr(), _p(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), _p(D), _p(bias),
        _p(h0), _p(lengths), _p(y), _p(h_last), _p(kept), *u.stride()[:2], *delta.stride()[:2], *_tb(z),
        *B.stride()[:3], *C.stride()[:3], *y_strides, T, Bn, Dn, A.shape[1], B.shape[2], _DTYPES[u.dtype],
        int(softplus), int(lengths is not None and lengths.dtype is torch.int64), 0)


def _scan_forward(u, delta, A, B, C, D, z, bias, h0, lengths, softplus, want_last, keep):
    T, Bn, Dn = u.shape
    N, dev = A.shape[1], u.get_device()
    lib = _capi.lib()
    y = _empty_like(u)
    h_last = A.new_empty((Bn, Dn, N)) if want_last else None
    kept = A.new_empty(lib.dfsnn_state_scan_kept_floats(T, Bn, Dn, N)) if keep else None
    args = _scan_args(u, delta, A, B, C, D, z, bias, h0, lengths, softplus, y, y.stride()[:2], h_last, kept)
    size = lib.dfsnn_state_scan_forward_workspace_size(T, Bn, Dn, N, B.shape[2])
    ws = A.new_empty(size // 4) if size else None
    _call(lib.dfsnn_state_scan_forward, "state_scan_forward", 2 if size else 1,
          lambda: _prof.state_scan_bytes(T, Bn, Dn, N, B.shape[2], u.element_size(), z is not None, False),
          dev, args, _p(ws), size)
    return y, h_last, kept


class StateScanFunction(torch.autograd.Function):
    """apply(u, delta, A, B, C, D, z, delta_bias, h0, lengths, softplus, return_state)
    -> (y, last states or None); the arguments checked as by state_scan."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, h0, lengths, softplus, want_last):
        y, h_last, kept = _scan_forward(u, delta, A, B, C, D, z, bias, h0, lengths, softplus,
                                        want_last, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, h0, lengths, kept)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, h_last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_last):
        u, delta, A, B, C, D, z, bias, h0, lengths, kept = ctx.saved_tensors
        T, Bn, Dn = u.shape
        N, G = A.shape[1], B.shape[2]
        gy = torch.zeros_like(u) if grad_y is None else grad_y
        gy = gy if gy.stride(-1) == 1 else _rows(gy)
        gl = None if grad_last is None else grad_last.contiguous()
        gu, gdelta = _empty_like(u), _empty_like(delta)
        gz = None if z is None else _empty_like(z)
        gB, gC = u.new_empty((T, Bn, G, N)), u.new_empty((T, Bn, G, N))
        make = torch.zeros_like if Bn == 0 or Dn == 0 else torch.empty_like
        gA = make(A)
        gD, gbias, gh0 = (None if x is None else make(x) for x in (D, bias, h0))
        lib = _capi.lib()
        args = _scan_args(u, delta, A, B, C, D, z, bias, h0, lengths, ctx.softplus, None, gy.stride()[:2],
                          None, kept)
        grads = _capi.STATE_SCAN_GRADS.pack(
            gy.data_ptr(), _p(gl), gu.data_ptr(), gdelta.data_ptr(), _p(gz), gB.data_ptr(), gC.data_ptr(),
            gA.data_ptr(), _p(gD), _p(gbias), _p(gh0), *gu.stride()[:2], *gdelta.stride()[:2], *_tb(gz))
        size = lib.dfsnn_state_scan_backward_workspace_size(T, Bn, Dn, N, G)
        ws = A.new_empty(size // 4)
        _call(lib.dfsnn_state_scan_backward, "state_scan_backward",
              2 if _prof._ACTIVE is None else lib.dfsnn_state_scan_backward_launches(T, Bn, Dn, N, G),
              lambda: _prof.state_scan_bytes(T, Bn, Dn, N, G, u.element_size(), z is not None, True),
              u.get_device(), args, grads, ws.data_ptr(), size)
        return gu, gdelta, gA, gB, gC, gD, gz, gbias, gh0, None, None, None


def state_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, h0=None,
               lengths=None, return_state=False):
    """Selective scan over sequences.

    u, delta, z [T, B, D]; A [D, N] (N <= 128); B, C [T, B, N] or, for G groups of D / G
    neighbouring channels, [T, B, G, N]; D, delta_bias [D]; h0 [B, D, N] states in front of
    step 0 (default zero).  d = delta (+ delta_bias), through softplus if asked; the gate
    silu(z) multiplies the output where z is given.  lengths (int32 / int64 [B], on the
    device): sequence b ends after lengths[b] steps; what its tensors hold behind is not
    read, and outputs and gradients there are zero.  Returns y [T, B, D], with return_state
    also the states after each sequence's last step, float32 [B, D, N]."""
    name = "state_scan"
    u = _lead(u, name, 3)
    shape, dtype, dev = u.shape, u.dtype, u.get_device()
    T, Bn, Dn = shape
    if T < 1:
        raise ValueError(f"{name}: at least one step, got T = {T}")
    delta = _seq(delta, dtype, dev, shape, name, "delta")
    if z is not None:
        z = _seq(z, dtype, dev, shape, name, "z")
    B, C = _groups(B, dtype, dev, (T, Bn), name, "B"), _groups(C, dtype, dev, (T, Bn), name, "C")
    N, _ = _scan_sizes(Dn, A, B, C, name)
    A = _param(A, dev, (Dn, N), name, "A")
    D = _param(D, dev, (Dn,), name, "D")
    bias = _param(delta_bias, dev, (Dn,), name, "delta_bias")
    h0 = _param(h0, dev, (Bn, Dn, N), name, "h0")
    lengths = _integers(lengths, dev, Bn, name, "lengths")
    tensors = (u, delta, A, B, C, D, z, bias, h0)
    _no_tangents(name, tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        y, last = StateScanFunction.apply(*tensors, lengths, bool(softplus), bool(return_state))
    else:
        y, last, _ = _scan_forward(*tensors, lengths, softplus, return_state, False)
    return (y, last) if return_state else y


def expired_waits(device=None):
    """Waits of state_scan's backward that ran out on this device since the start of the process.

    For some sizes blocks of the backward wait for one another, within bounds; gradients that depend on a
    wait that ran out are NaN.  0 unless the device stalls.  Synchronises the current stream."""
    count = ctypes.c_ulonglong()
    with torch.cuda.device(device):
        _capi.check(_capi.lib().dfsnn_state_scan_expired_waits(
            ctypes.byref(count), torch.cuda.current_stream().cuda_stream), "expired_waits")
    return count.value


def state_scan_step(u, delta, state, A, B, C, D=None, z=None, delta_bias=None, softplus=False,
                    index=None, state_out=None):
    """One step of the selective scan for each of B rows; not differentiable (refused where an input
    requires a gradient and gradients are enabled).

    u, delta, z [B, D]; B, C [B, N] or [B, G, N]; state float32 [S, D, N], a slot for each row
    or, with index (int32 / int64 [B], on the device), a pool of S slots of which row b uses
    index[b].  The new states replace the old ones, or go to the same slots of state_out
    (memory of its own, or state itself).
    A negative index marks an idle row: its y is zero and no state changes.  An index past
    the pool, or one that an earlier row has, gives NaN and changes no state.  Returns
    y [B, D]."""
    name = "state_scan_step"
    u = _lead(u, name, 2)
    shape, dtype, dev = u.shape, u.dtype, u.get_device()
    Bn, Dn = shape
    delta = _seq(delta, dtype, dev, shape, name, "delta")
    if z is not None:
        z = _seq(z, dtype, dev, shape, name, "z")
    B, C = _groups(B, dtype, dev, (Bn,), name, "B"), _groups(C, dtype, dev, (Bn,), name, "C")
    N, G = _scan_sizes(Dn, A, B, C, name)
    A = _param(A, dev, (Dn, N), name, "A")
    D = _param(D, dev, (Dn,), name, "D")
    bias = _param(delta_bias, dev, (Dn,), name, "delta_bias")
    index = _integers(index, dev, Bn, name, "index")
    _no_gradients(name, (u, delta, A, B, C, D, z, bias))
    if _fw._current_level >= 0:
        _no_tangents(name, (u, delta, A, B, C, D, z, bias, state))
    state_out, slots, s_in, s_out = _pool(state, state_out, torch.float32, dev, (Dn, N), Bn, index, name)
    y = u.new_empty(shape)
    args = _capi.STATE_SCAN_STEP_ARGS.pack(
        u.data_ptr(), delta.data_ptr(), _p(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), _p(D), _p(bias),
        state.data_ptr(), state_out.data_ptr(), _p(index), y.data_ptr(), u.stride(0), delta.stride(0),
        0 if z is None else z.stride(0), *B.stride()[:2], *C.stride()[:2], Dn, s_in, s_out, Bn, Dn, slots,
        N, G, _DTYPES[dtype], int(softplus), int(index is not None and index.dtype is torch.int64), 0)
    _call(_capi.lib().dfsnn_state_scan_step, name, 1,
          lambda: _prof.state_scan_step_bytes(Bn, Dn, N, G, u.element_size(), z is not None), dev, args)
    return y


def _conv_args(x, weight, bias, state, lengths, silu, y, y_strides, last):
    T, Bn, Dn = x.shape
    return _capi.SHORT_CONV_ARGS.pack(
        x.data_ptr(), weight.data_ptr(), _p(bias), _p(state), _p(lengths), _p(y), _p(last), *x.stride()[:2],
        *y_strides, T, Bn, Dn, weight.shape[1], _DTYPES[x.dtype], silu,
        int(lengths is not None and lengths.dtype is torch.int64))


def _conv_forward(x, weight, bias, state, lengths, silu, want_last):
    T, Bn, Dn = x.shape
    W = weight.shape[1]
    y = _empty_like(x)
    last = x.new_empty((Bn, W - 1, Dn)) if want_last else None
    args = _conv_args(x, weight, bias, state, lengths, silu, y, y.stride()[:2], last)
    _call(_capi.lib().dfsnn_short_conv_forward, "short_conv_forward", 1,
          lambda: _prof.short_conv_bytes(T, Bn, Dn, W, x.element_size(), False), x.get_device(), args)
    return y, last


class ShortConvFunction(torch.autograd.Function):
    """apply(x, weight, bias, state, lengths, silu, return_state) -> (y, last inputs or None);
    the arguments checked as by short_conv."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_last):
        y, last = _conv_forward(x, weight, bias, state, lengths, silu, want_last)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_last):
        x, weight, bias, state, lengths = ctx.saved_tensors
        T, Bn, Dn = x.shape
        W = weight.shape[1]
        gy = torch.zeros_like(x) if grad_y is None else grad_y
        gy = gy if gy.stride(-1) == 1 else _rows(gy)
        gl = None if grad_last is None else grad_last.contiguous()
        gx = _empty_like(x)
        make = torch.zeros_like if Bn == 0 or Dn == 0 else torch.empty_like
        gw = make(weight)
        gb, gs = (None if t is None else make(t) for t in (bias, state))
        lib = _capi.lib()
        args = _conv_args(x, weight, bias, state, lengths, ctx.silu, None, gy.stride()[:2], None)
        grads = _capi.SHORT_CONV_GRADS.pack(gy.data_ptr(), _p(gl), gx.data_ptr(), _p(gs), gw.data_ptr(),
                                            _p(gb), *gx.stride()[:2])
        size = lib.dfsnn_short_conv_backward_workspace_size(T, Bn, Dn, W)
        ws = weight.new_empty(size // 4)
        _call(lib.dfsnn_short_conv_backward, "short_conv_backward", 2,
              lambda: _prof.short_conv_bytes(T, Bn, Dn, W, x.element_size(), True), x.get_device(), args,
              grads, ws.data_ptr(), size)
        return gx, gw, gb, gs, None, None, None


def short_conv(x, weight, bias=None, activation=None, state=None, lengths=None, return_state=False):
    """Causal convolution of each channel with a few taps.

    x [T, B, D]; weight [D, W] (W <= 8; the last tap meets the current step); bias [D];
    activation None or "silu"; state [B, W - 1, D], x's type: the inputs in front of step 0,
    oldest first (default zero); lengths as in state_scan.  Returns y [T, B, D], with
    return_state also the last W - 1 inputs of each sequence, for the tokens that follow."""
    name = "short_conv"
    silu = _silu_flag(activation, name)
    x = _lead(x, name, 3)
    T, Bn, Dn = x.shape
    dev = x.get_device()
    if T < 1:
        raise ValueError(f"{name}: at least one step, got T = {T}")
    W = _taps(weight, Dn, name)
    weight = _param(weight, dev, (Dn, W), name, "weight")
    bias = _param(bias, dev, (Dn,), name, "bias")
    if state is not None:
        state = _seq(state, x.dtype, dev, (Bn, W - 1, Dn), name, "state").contiguous()
    lengths = _integers(lengths, dev, Bn, name, "lengths")
    tensors = (x, weight, bias, state)
    _no_tangents(name, tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        y, last = ShortConvFunction.apply(*tensors, lengths, silu, bool(return_state))
    else:
        y, last = _conv_forward(*tensors, lengths, silu, return_state)
    return (y, last) if return_state else y


def short_conv_step(x, state, weight, bias=None, activation=None, index=None, state_out=None):
    """One step of the short convolution for each of B rows; not differentiable (as state_scan_step).

    x [B, D]; state [S, W - 1, D], x's type: the last inputs of each slot, oldest first, as
    short_conv returns them; index and state_out as in state_scan_step.  Returns y [B, D]."""
    name = "short_conv_step"
    silu = _silu_flag(activation, name)
    x = _lead(x, name, 2)
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    Bn, Dn = shape
    W = _taps(weight, Dn, name)
    weight = _param(weight, dev, (Dn, W), name, "weight")
    bias = _param(bias, dev, (Dn,), name, "bias")
    index = _integers(index, dev, Bn, name, "index")
    _no_gradients(name, (x, weight, bias))
    if _fw._current_level >= 0:
        _no_tangents(name, (x, weight, bias, state))
    state_out, slots, s_in, s_out = _pool(state, state_out, dtype, dev, (W - 1, Dn), Bn, index, name)
    y = x.new_empty(shape)
    args = _capi.SHORT_CONV_STEP_ARGS.pack(
        x.data_ptr(), weight.data_ptr(), _p(bias), state.data_ptr(), state_out.data_ptr(), _p(index),
        y.data_ptr(), x.stride(0), Dn, s_in, s_out, Bn, Dn, slots, W, _DTYPES[dtype], silu,
        int(index is not None and index.dtype is torch.int64))
    _call(_capi.lib().dfsnn_short_conv_step, name, 1,
          lambda: _prof.short_conv_step_bytes(Bn, Dn, W, x.element_size()), dev, args)
    return y


# ---------------------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------------------
class StateSpaceLayer(nn.Module):
    """Projections, short convolution and gated selective scan: [T, B, d_model] -> the same.

    step_mode 'm' takes a whole sequence a call, 's' one step [B, d_model] a call, carrying its
    states until reset().  Where gradients are enabled and asked for, the steps are differentiable:
    the carried states are part of the graph, which goes back to the last reset() (or to the last
    step without gradients).  Serving code that keeps its own states uses
    forward(..., state=, return_state=True) for prompts and step() for tokens: a state is the pair
    (convolution inputs [S, taps - 1, d_inner], scan states [S, d_inner, d_state])."""

    def __init__(self, d_model, d_state=16, taps=4, expand=2, groups=1, rank=None, step_mode="m",
                 step_range=(1e-3, 1e-1)):
        super().__init__()
        if step_mode not in ("s", "m"):
            raise ValueError(f"step_mode must be 's' or 'm', got {step_mode!r}")
        self.d_model, self.d_inner = int(d_model), int(expand * d_model)
        self.d_state, self.groups, self.step_mode = int(d_state), int(groups), step_mode
        if self.d_inner % self.groups:
            raise ValueError(f"{self.d_inner} channels do not divide into {groups} groups")
        self.rank = max(1, -(-self.d_model // 16)) if rank is None else int(rank)
        self.in_proj = nn.Linear(self.d_model, 2 * self.d_inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(self.d_inner, taps).uniform_(-1, 1) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(self.d_inner))
        self.x_proj = nn.Linear(self.d_inner, self.rank + 2 * self.groups * self.d_state, bias=False)
        self.dt_proj = nn.Linear(self.rank, self.d_inner, bias=False)
        # softplus(delta_bias) is spread over step_range on a logarithmic scale
        lo, hi = (math.log(v) for v in step_range)
        step = torch.exp(torch.rand(self.d_inner) * (hi - lo) + lo)
        self.delta_bias = nn.Parameter(torch.log(torch.expm1(step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, self.d_state + 1, dtype=torch.float32))
                                  .repeat(self.d_inner, 1))
        self.D = nn.Parameter(torch.ones(self.d_inner))
        self.out_proj = nn.Linear(self.d_inner, self.d_model, bias=False)
        self.reset()

    def reset(self):
        self._state = None

    def initial_state(self, slots, dtype=None, device=None):
        w = self.in_proj.weight
        dtype, device = dtype or w.dtype, device or w.device
        return (torch.zeros(slots, self.conv_weight.shape[1] - 1, self.d_inner, dtype=dtype, device=device),
                torch.zeros(slots, self.d_inner, self.d_state, device=device))

    def _split(self, x):
        dt, B, C = torch.split(self.x_proj(x), [self.rank, self.groups * self.d_state,
                                                self.groups * self.d_state], dim=-1)
        shape = (self.groups, self.d_state)
        return self.dt_proj(dt), B.unflatten(-1, shape), C.unflatten(-1, shape)

    def forward(self, x, lengths=None, state=None, return_state=False):
        if self.step_mode == "s":
            if lengths is not None or state is not None or return_state:
                raise ValueError("step_mode 's' carries its own state: use step()")
            return self._carried_step(x)
        return self._sequence(x, lengths, state, return_state)

    def _sequence(self, x, lengths, state, return_state):
        conv0, h0 = (None, None) if state is None else state
        x, z = self.in_proj(x).chunk(2, dim=-1)
        x = short_conv(x, self.conv_weight, self.conv_bias, "silu", conv0, lengths, return_state)
        if return_state:
            x, conv0 = x
        dt, B, C = self._split(x)
        y = state_scan(x, dt, -torch.exp(self.A_log.float()), B, C, self.D, z, self.delta_bias, True,
                       h0, lengths, return_state)
        if return_state:
            y, h0 = y
        y = self.out_proj(y)
        return (y, (conv0, h0)) if return_state else y

    def _carried_step(self, x):
        state = self._state
        if state is not None and state[1].shape[0] != x.shape[0]:
            raise ValueError(f"step_mode 's': the carried states are those of {state[1].shape[0]} rows, got "
                             f"{x.shape[0]}: call reset() before another batch")
        if torch.is_grad_enabled() and any(t.requires_grad for t in (x, *self.parameters(), *(state or ()))):
            y, self._state = self._sequence(x.unsqueeze(0), None, state, True)
            return y.squeeze(0)
        if state is not None:                   # of a step with gradients: nothing saved them yet
            state = self._state = tuple(s.detach() for s in state)
        return self.step(x, state)

    @torch.no_grad()
    def step(self, x, state, index=None):
        """One token for each row of x [B, d_model], without gradients; state is advanced in place."""
        x, z = self.in_proj(x).chunk(2, dim=-1)
        if state is None:                       # the layer's own, from zero
            state = self._state = self.initial_state(x.shape[0], x.dtype, x.device)
        x = short_conv_step(x, state[0], self.conv_weight, self.conv_bias, "silu", index)
        dt, B, C = self._split(x)
        y = state_scan_step(x, dt, state[1], -torch.exp(self.A_log.float()), B, C, self.D, z,
                            self.delta_bias, True, index)
        return self.out_proj(y)
