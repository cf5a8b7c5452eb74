"""State-space layer without a GPU: what the calls tell autograd, and what they refuse."""
import pytest
import torch
from torch.autograd import forward_ad

from dfsnn_b200 import _capi, state_space as ss


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
