"""Precision of the state-space kernels: sums over many sequences, every output within its own error
bound, states that remember thousands of steps."""
import pytest
import torch

import state_bounds
from dfsnn_b200 import _capi, state_space as ss
from test_gpu_state_space import scan_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24                           # half a step of fp32, relative


@pytest.mark.parametrize("T,B,D,N", [(1, 600, 2048, 16), (3, 24000, 20, 4), (16, 5000, 100, 8), (2, 5000, 64, 100)])
@pytest.mark.parametrize("big", [0, -1])
def test_parameter_gradients_over_many_sequences(T, B, D, N, big):
    """A term of 2^24 and then ones, each of which one running fp32 sum would lose.

    With A = 0 and delta = u = 1 every product is a whole number below 2^24 and exact.  State 0 has
    B = C = 1 and no grad_h_last, so g_t = gy, l_t[0] = sum of the gy from t on and
    grad delta_t = grad u_t = l_t[0] (+ D g_t in grad u); the other states have h0 = 1, B = C = 0 and
    q = grad_h_last.  Sums over t and b: grad D = sum gy, grad A[n > 0] = T sum grad_h_last.  All terms
    are positive, so each rounding is off by at most U of the whole sum; there are few of them:
    T (<= 16) terms a tile, the block's sum, the blocks' sum."""
    gy, gh = torch.zeros(T, B, D), torch.ones(B, D, N)
    gy[0] = 1.0                                          # all of a sequence's gradient at its first step
    gy[0, big] = gh[big] = 2.0 ** 24
    gh[..., 0] = 0.0
    bc = torch.zeros(T, B, N)
    bc[..., 0] = 1.0
    h0 = torch.ones(B, D, N)
    h0[..., 0] = 0.0
    ones = torch.ones(T, B, D)
    leaves = {"u": ones, "delta": ones.clone(), "A": torch.zeros(D, N), "B": bc, "C": bc.clone(), "D": torch.zeros(D),
              "delta_bias": torch.zeros(D), "h0": h0}
    leaves = {k: v.to(DEV).requires_grad_(True) for k, v in leaves.items()}
    y, h = ss.state_scan(**leaves, return_state=True)
    got = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [gy.to(DEV), gh.to(DEV)])))
    total = 2.0 ** 24 + B - 1
    for name, want, terms in (("D", total, 1), ("delta_bias", total, 1), ("A", T * total, T)):
        v = got[name].double()
        v = v[:, 1:] if name == "A" else v
        assert float((v - want).abs().max()) <= (terms + 2) * U * want, (name, float(v.min()), float(v.max()), want)


# ---------------------------------------------------------------------------------------
# every output within its own running error bound (state_bounds.py)
# ---------------------------------------------------------------------------------------
def within_bounds(x, n, grads, softplus, what, part=0):
    gy, gh = grads
    leaves = {k: v.detach().requires_grad_(True) for k, v in x.items()}
    y, h = ss.state_scan(**leaves, softplus=softplus, lengths=n, return_state=True)
    got = {"y": y, "h": h}
    got.update(("g" + k, v) for k, v in zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [gy, gh])))
    want, bound = state_bounds.scan(**x, softplus=softplus, lengths=n, gy=gy, gh=gh, part=part)
    return {k: state_bounds.check(v, want[k], bound[k], f"{what} {k}") for k, v in got.items()}


TYPES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,D,N,G,full,scale", [
    (1, 3, 5, 16, 1, True, 1.0), (17, 2, 130, 2, 1, True, 1.0), (33, 2, 96, 12, 3, True, 0.3), (50, 3, 70, 8, 2, False, 1.0),
    (61, 2, 40, 32, 2, True, 0.1), (64, 2, 18, 64, 1, False, 0.3), (48, 2, 9, 128, 3, True, 0.1), (20, 2, 33, 16, 1, True, 300.0),
    (31, 1200, 36, 3, 1, True, 0.3), (16, 3000, 36, 16, 1, False, 1.0)])
def test_scan_within_bounds(T, B, D, N, G, full, scale, dtype):
    x, n, grads = scan_case(T, B, D, N, G, dtype, full=full, seed=T, scale=scale)
    within_bounds(x, n, grads, full, f"{T}x{B}x{D} N{N}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,D,N,G", [(300, 480, 8, 16, 1), (270, 64, 250, 12, 2), (290, 300, 33, 4, 1), (280, 160, 12, 100, 1)])
def test_scan_one_part_after_another_within_bounds(T, B, D, N, G, dtype):
    assert _capi.lib().dfsnn_state_scan_backward_launches(T, B, D, N, G) == 2
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(T)).tolist()
    x, n, grads = scan_case(T, B, D, N, G, dtype, lengths=lengths, seed=T, scale=0.1)
    within_bounds(x, n, grads, True, f"one after another {T}x{B}x{D}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,D,N,G,lengths", [
    (1000, 1, 40, 16, 1, None), (2049, 4, 36, 16, 2, [2049, 700, 0, 1]), (1500, 2, 12, 100, 1, [16, 1024]),
    (640, 1, 300, 3, 1, None), (1040, 3, 9, 33, 3, [1040, 1039, 129])])
def test_scan_parts_side_by_side_within_bounds(T, B, D, N, G, lengths, dtype):
    assert _capi.lib().dfsnn_state_scan_backward_launches(T, B, D, N, G) == 3
    x, n, grads = scan_case(T, B, D, N, G, dtype, lengths=lengths, seed=T, scale=0.1)
    within_bounds(x, n, grads, True, f"side by side {T}x{B}x{D}", part=-(-T // 10))


# ---------------------------------------------------------------------------------------
# states that remember thousands of steps
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,D,N", [(1, 48, 16), (1, 33, 3), (300, 32, 16), (150, 36, 8), (200, 5, 100)])
def test_slow_decays(B, D, N):
    """u = 0, one step size a channel: h_t = exp((t + 1) d A) h0 and grad h0 = exp(T d A) grad h_last, in
    whole walks and in parts.  A step is off by its decay's 1.4 units of 2^-24 (test_decays_near_one) and
    the product's rounding, 2.5 in all.  Parts: the sum of P <= 512 equal steps is off by P units, its
    exponent is at most P / 16, so P^2 / 16 a part, P / 16 a step; but a part has 64 steps where there
    are that few rows."""
    T = 4096
    g = torch.Generator().manual_seed(N)
    r = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    d, A = 0.05 + 0.1 * r(D), -(0.02 + 0.02 * r(D, N))
    rate = d.double()[:, None] * A.double()
    assert float(rate.abs().max()) * 1.4427 < 1 / 16
    h0, gh = 1 + r(B, D, N), 1 + r(B, D, N)
    n = int(torch.randint(N, (1,), generator=g))
    C = torch.zeros(T, B, N)
    C[..., n] = 1
    zero = torch.zeros(1, 1, D).expand(T, B, D)
    A, C, dt, u, h0, gh = (v.to(DEV) for v in (A, C, d.expand(T, B, D), zero, h0, gh))
    h0.requires_grad_(True)
    y, h = ss.state_scan(u, dt, A, C, C, h0=h0, return_state=True)
    gh0, = torch.autograd.grad(h, h0, gh)
    rate = rate.to(DEV)
    few = _capi.lib().dfsnn_state_scan_forward_workspace_size(T, B, D, N, 1) > 0
    K = (2.5 + (4.0 if few else 0.0)) * torch.arange(1, T + 1, device=DEV).double() + 2
    ratio = {}
    for k, got, want, units in (
            ("y", y, torch.exp(torch.arange(1, T + 1, device=DEV)[:, None, None] * rate[:, n]) * h0.detach()[..., n].double(), K[:, None, None]),
            ("h", h, torch.exp(T * rate) * h0.detach().double(), K[-1]), ("gh0", gh0, torch.exp(T * rate) * gh.double(), K[-1])):
        off = ((got.detach().double() - want).abs() / want / U / units).max()
        ratio[k] = float(off)
    assert all(v <= 1 for v in ratio.values()), ratio


@pytest.mark.parametrize("D,N", [(2048, 16), (700, 3), (512, 40), (200, 128), (1000, 8)])
@pytest.mark.parametrize("most", [2.0 ** -14, 2.0 ** -8, 0.0433])
def test_decays_near_one(D, N, most):
    """One step with u = 0 from h0 = 1 returns the decay itself, and its backward from 1 too.  For
    |d A log2 e| < 1/16 it is the polynomial's: fitted to 0.64 units of 2^-24, its inner roundings 0.1, the
    last one (below 1) 0.5, the argument's three 3 * 0.0433: 1.4 units.  The hardware's power, off by nearly 2
    there, would always be off to the same side: over the thousands of steps that a state remembers, that
    adds up."""
    B = 8
    g = torch.Generator().manual_seed(D)
    A = (-most * torch.rand(D, N, generator=g)).to(DEV)
    d = (0.9 + 0.1 * torch.rand(1, B, D, generator=g)).to(DEV)
    zero, z = torch.zeros_like(d), torch.zeros(1, B, N, device=DEV)
    one = torch.ones(B, D, N, device=DEV)
    h0 = one.clone().requires_grad_(True)
    _, h = ss.state_scan(zero, d, A, z, z, h0=h0, return_state=True)
    gh0, = torch.autograd.grad(h, h0, one)
    stepped = one.clone()
    ss.state_scan_step(zero[0], d[0], stepped, A, z[0], z[0])
    want = torch.exp(d[0].double()[..., None] * A.double())
    off = [float(((v.detach().double() - want).abs() / want).max()) / U for v in (h, gh0, stepped)]
    assert max(off) <= 1.4, off


# ---------------------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,B,D,W,act,lengths", [
    (1, 2, 128, 4, True, None), (65, 3, 7, 3, True, [65, 0, 31]), (200, 2, 132, 4, False, None), (33, 40, 130, 2, True, None),
    (100, 2, 40, 8, True, [100, 7]), (64, 1, 20, 1, False, None)])
def test_conv_within_bounds(T, B, D, W, act, lengths, dtype):
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(sum(s))).to(DEV)  # noqa: E731
    n = None if lengths is None else torch.tensor(lengths, device=DEV)
    args = {"x": r(T, B, D).to(dtype), "weight": r(D, W), "bias": r(D), "state": r(B, W - 1, D).to(dtype)}
    gy, gl = r(T, B, D).flip(0).to(dtype), r(B, W - 1, D).flip(0).to(dtype)
    leaves = {k: v.clone().requires_grad_(True) for k, v in args.items()}
    y, last = ss.short_conv(leaves["x"], leaves["weight"], leaves["bias"], "silu" if act else None, leaves["state"], n,
                            return_state=True)
    got = {"y": y, "last": last}
    got.update(("g" + k, v) for k, v in zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [gy, gl],
                                                                        allow_unused=True)))
    want, bound = state_bounds.conv(**args, silu_=act, lengths=n, gy=gy, glast=gl)
    for k, v in got.items():
        state_bounds.check(torch.zeros_like(args[k[1:]]) if v is None else v, want[k], bound[k], f"conv {k}")
    if dtype == torch.float32:
        assert torch.equal(last.detach().double(), want["last"])
