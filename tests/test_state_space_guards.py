"""State-space layer without a GPU: what the calls tell autograd, and what they refuse."""
import pytest
import torch
from torch.autograd import forward_ad

import state_bounds
import state_ref
from dfsnn_b200 import _capi, state_space as ss
from test_state_space import scan_autograd, scan_inputs


# ---------------------------------------------------------------------------------------
# states written in place
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_pool_written_in_place_raises_its_version(mode):
    """As torch's own in-place operations, which count with gradients off too."""
    state, out = torch.zeros(3, 4, 5), torch.zeros(3, 4, 5)
    pool = torch.zeros(3, 2, 4, 5)
    with mode():
        for s, o, written in ((state, None, state), (state, out, out), (pool[:, 1], None, pool)):
            before = written._version
            ss._pool(s, o, torch.float32, -1, (4, 5), 3, None, "test")
            assert written._version > before
    assert state._version == 1                          # state_out leaves `state` as it was


def test_pool_of_inference_tensors():
    with torch.inference_mode():
        state = torch.zeros(3, 4, 5)
        ss._pool(state, None, torch.float32, -1, (4, 5), 3, None, "test")
    ss._pool(state, None, torch.float32, -1, (4, 5), 3, None, "test")


# ---------------------------------------------------------------------------------------
# forward-mode tangents
# ---------------------------------------------------------------------------------------
def test_forward_mode_tangents_are_refused():
    x = torch.ones(3)
    ss._no_tangents("test", (x, None))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        ss._no_tangents("test", (x, None))              # a level alone harms nobody
        for tensors in ((dual,), (x, None, dual), (dual.double().contiguous(),)):
            with pytest.raises(NotImplementedError, match="test: forward-mode"):
                ss._no_tangents("test", tensors)


# ---------------------------------------------------------------------------------------
# gradients through the step forms
# ---------------------------------------------------------------------------------------
def test_steps_refuse_inputs_that_require_gradients():
    x, w = torch.ones(3), torch.ones(3, requires_grad=True)
    ss._no_gradients("test", (x, None))
    with torch.no_grad():
        ss._no_gradients("test", (x, w))
    with pytest.raises(RuntimeError, match="test is not differentiable"):
        ss._no_gradients("test", (x, None, w))


def test_expired_waits_without_a_place():
    assert _capi.lib().dfsnn_state_scan_expired_waits(None, None) == _capi.DFSNN_ERR_NULL


# ---------------------------------------------------------------------------------------
# the error bounds that the GPU tests go by
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("full", [True, False])
def test_bounds_go_with_the_formulas(full):
    """state_bounds.py has the values of state_ref.py, and fp32 evaluations of the formulas keep to its
    bounds."""
    g = torch.Generator().manual_seed(3)
    x = {k: v.float() for k, v in scan_inputs(40, 3, 8, 6, 2, full, True).items()}
    n = torch.tensor([40, 17, 0])
    gy, gh = torch.randn(40, 3, 8, generator=g), torch.randn(3, 8, 6, generator=g)
    want, bound = state_bounds.scan(**x, softplus=full, lengths=n, gy=gy, gh=gh)
    ref = state_ref.scan(**x, softplus=full, lengths=n, gy=gy, gh=gh)
    keys = ["y", "h", *("g" + k for k in x)]
    for k in keys:
        assert torch.allclose(want[k], ref[k], rtol=1e-12, atol=1e-13), k
        assert (bound[k] >= 0).all() and bound[k].max() < 1e-3 * (1 + want[k].abs().max()), k
    leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
    y, h = scan_autograd(leaves, full, n)
    got = [y, h, *torch.autograd.grad([y, h], list(leaves.values()), [gy, gh])]
    for k, v in zip(keys, got):
        state_bounds.check(v.float(), want[k], bound[k], k)     # (padding makes y 64 bits wide)
    w, b = torch.randn(8, 4, generator=g), torch.randn(8, generator=g)
    s, gl = torch.randn(3, 3, 8, generator=g), torch.randn(3, 3, 8, generator=g)
    want, bound = state_bounds.conv(x["u"], w, b, full, s, n, gy, gl)
    ref = state_ref.conv(x["u"], w, b, full, s, n, gy, gl)
    for k, v in want.items():
        assert torch.allclose(v, ref[k], rtol=1e-12, atol=1e-13), k
        assert bound[k].max() < 1e-3, k
