"""Precision of the state-space kernels where it could get lost: sums over many sequences."""
import pytest
import torch

from dfsnn_b200 import state_space as ss

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
