"""State-space layer on the GPU: calls that must not return a wrong answer silently."""
import pytest
import torch
from torch.autograd import forward_ad

import state_ref
from dfsnn_b200 import _capi, state_space as ss
from test_gpu_state_space import close, scan_case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


# ---------------------------------------------------------------------------------------
# states written in place
# ---------------------------------------------------------------------------------------
def test_scan_state_advanced_before_the_backward_is_noticed():
    """h0 is saved by reference: a step that advances it must make the backward refuse."""
    T, B, D, N = 8, 2, 12, 4
    A, h0 = (-rand(D, N).abs()).requires_grad_(True), rand(B, D, N, seed=1)
    u, bc = rand(T, B, D, seed=2), rand(T, B, N, seed=3)
    for step in (torch.no_grad, torch.inference_mode):
        y = ss.state_scan(u, u, A, bc, bc, softplus=True, h0=h0)
        with step():
            ss.state_scan_step(u[0], u[0], h0, A, bc[0], bc[0], softplus=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), A)


def test_conv_state_advanced_before_the_backward_is_noticed():
    x, w, state = rand(8, 2, 12), rand(12, 4, seed=1).requires_grad_(True), rand(2, 3, 12, seed=2)
    y = ss.short_conv(x, w, state=state)
    with torch.no_grad():
        ss.short_conv_step(x[0], state, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), w)


def test_layer_step_on_a_saved_state_is_noticed():
    """The prompt's states advanced by a token between its forward and its backward; on copies of
    them the gradients are those without the token."""
    torch.manual_seed(0)
    layer = ss.StateSpaceLayer(16).to(DEV)
    x, token = rand(4, 2, 16), rand(2, 16, seed=1)
    conv, scan = rand(2, 3, 32, seed=2), rand(2, 32, 16, seed=3)
    params = list(layer.parameters())
    y, _ = layer(x, state=(conv, scan), return_state=True)
    want = torch.autograd.grad(y.sum(), params)
    y, _ = layer(x, state=(conv, scan), return_state=True)
    layer.step(token, (conv.clone(), scan.clone()))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum(), params), want))
    y, _ = layer(x, state=(conv, scan), return_state=True)
    layer.step(token, (conv, scan))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---------------------------------------------------------------------------------------
# forward-mode tangents
# ---------------------------------------------------------------------------------------
def test_forward_mode_tangents_are_refused():
    """Each input of each call in turn; the other inputs need gradients or not."""
    T, B, D, N = 4, 2, 8, 4
    scan = {"u": rand(T, B, D), "delta": rand(T, B, D, seed=1), "A": -rand(D, N).abs(), "B": rand(T, B, N),
            "C": rand(T, B, N, seed=2), "D": rand(D), "z": rand(T, B, D, seed=3), "delta_bias": rand(D), "h0": rand(B, D, N)}
    seqs = ("u", "delta", "B", "C", "z")
    step = {k: v[0] if k in seqs else v for k, v in scan.items() if k != "h0"}
    step["state"] = rand(B, D, N)
    conv = {"x": rand(T, B, D), "weight": rand(D, 3), "bias": rand(D), "state": rand(B, 2, D)}
    conv_step = {**conv, "x": conv["x"][0]}
    for call, args in ((ss.state_scan, scan), (ss.state_scan_step, step), (ss.short_conv, conv),
                       (ss.short_conv_step, conv_step)):
        want = call(**{k: v.clone() for k, v in args.items()})
        for k in args:
            with forward_ad.dual_level():
                got = call(**{n: v.clone() for n, v in args.items()})
                assert torch.equal(got, want)
                bad = {n: forward_ad.make_dual(v.clone(), torch.ones_like(v)) if n == k else v.clone()
                       for n, v in args.items()}
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(**bad)
                if call in (ss.state_scan, ss.short_conv):
                    other = next(n for n in args if n != k)
                    bad[other].requires_grad_(True)
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(**bad)


# ---------------------------------------------------------------------------------------
# gradients through the step forms
# ---------------------------------------------------------------------------------------
def test_steps_refuse_inputs_that_require_gradients():
    """They could only return outputs cut off from the graph.  Nothing is written before the refusal."""
    B, D, N = 2, 8, 4
    scan = {"u": rand(B, D), "delta": rand(B, D, seed=1), "A": -rand(D, N).abs(), "B": rand(B, N),
            "C": rand(B, N, seed=2), "D": rand(D), "z": rand(B, D, seed=3), "delta_bias": rand(D)}
    conv = {"x": rand(B, D), "weight": rand(D, 3), "bias": rand(D)}
    for call, args, state in ((ss.state_scan_step, scan, rand(B, D, N)), (ss.short_conv_step, conv, rand(B, 2, D))):
        want = call(**args, state=state.clone())
        for k in args:
            leaves = {n: v.detach().requires_grad_(n == k) for n, v in args.items()}
            kept = state.clone()
            with pytest.raises(RuntimeError, match="not differentiable"):
                call(**leaves, state=kept)
            assert torch.equal(kept, state) and kept._version == 0
            with torch.no_grad():
                assert torch.equal(call(**leaves, state=kept), want)


# ---------------------------------------------------------------------------------------
# the layer, step by step
# ---------------------------------------------------------------------------------------
def test_layer_in_single_steps_has_the_gradients_of_the_sequence():
    """Outputs and every gradient of T single steps against 64 bits.  Every path has a few hundred
    roundings (T steps of the scan, sums over 96 channels, T B rows) and four projections with sums of
    at most 96 terms; norm against norm, the bounds of the whole sequence's test."""
    from test_gpu_state_space import layer_64
    torch.manual_seed(0)
    T, B = 7, 3
    layer = ss.StateSpaceLayer(48, groups=2, step_mode="s").to(DEV)
    x = rand(T, B, 48).requires_grad_(True)
    gy = rand(T, B, 48, seed=1)
    rel = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    for _ in range(2):                                   # reset() starts anew
        y = torch.stack([layer(x[t]) for t in range(T)])
        x64 = x.detach().double().requires_grad_(True)
        y64, p = layer_64(layer, x64)
        got = torch.autograd.grad(y, [x, *layer.parameters()], gy)
        want = torch.autograd.grad(y64, [x64, *p.values()], gy.double())
        assert rel(y, y64) < 2000 * 2.0 ** -24
        for k, a, b in zip(("x", *p), got, want):
            assert rel(a, b) < 20000 * 2.0 ** -24, k
        layer.reset()
    # steps without gradients go on from those with, in place, and the other way round
    y = [layer(x[0])]
    with torch.no_grad():
        y += [layer(x[1])]
        carried = layer._state[1].data_ptr()
        y += [layer(x[2])]
        assert not y[-1].requires_grad and layer._state[1].data_ptr() == carried
    y += [layer(x[3])]
    assert rel(torch.stack(y), y64[:4].detach()) < 2000 * 2.0 ** -24
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y[3].sum() + y[0].sum(), list(layer.parameters())))


def test_layer_refuses_a_batch_that_is_not_the_carried_one():
    layer = ss.StateSpaceLayer(16, step_mode="s").to(DEV)
    for mode in (torch.no_grad, torch.enable_grad):
        with mode():
            layer.reset()
            layer(rand(8, 16))
            kept = [s.detach().clone() for s in layer._state]
            for x in (rand(4, 16), rand(9, 16)):
                with pytest.raises(ValueError, match="call reset"):
                    layer(x)
            with pytest.raises((ValueError, RuntimeError)):      # another type
                layer(rand(8, 16).double())
            assert all(torch.equal(a, b) for a, b in zip(kept, layer._state))
            layer.reset()
            assert layer(rand(4, 16)).shape == (4, 16)


# ---------------------------------------------------------------------------------------
# values at the ends of the range
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,B,D,N,G,lengths", [
    (17, 2, 40, 16, 1, None), (16, 3, 33, 5, 1, [16, 7, 0]), (40, 4, 24, 40, 2, [40, 1, 0, 23]), (31, 2, 9, 100, 1, None),
    (9, 2, 40, 8, 1, [3, 9]), (900, 1, 20, 16, 1, None), (901, 2, 12, 3, 1, [900, 461]), (300, 480, 8, 16, 1, None)])
def test_scan_states_that_forget_at_once(T, B, D, N, G, lengths):
    """A = -inf: the decay is 0, on a step behind a sequence's end (or in the rest of a tile) as well as
    on any other, where it must not touch the state.  The formula with -1e30 in its place has the same
    values.  A decay of 0 has no error, so the bound goes by the other states (as in test_scan_*)."""
    x, n, (gy, gh) = scan_case(T, B, D, N, G, "f32", lengths=lengths, seed=T, scale=0.1)
    x["A"][:, ::3] = -float("inf")
    leaves = {k: v.detach().requires_grad_(True) for k, v in x.items()}
    y, h = ss.state_scan(**leaves, softplus=True, lengths=n, return_state=True)
    got = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [gy, gh])))
    ref = {**x, "A": x["A"].clamp_min(-1e30)}
    want, mag = (state_ref.scan(**ref, softplus=True, lengths=n, gy=gy, gh=gh, mag=m) for m in (False, True))
    m = state_ref.scan(**{**x, "A": x["A"].nan_to_num(neginf=0.0)}, softplus=True, lengths=n)["step_decay"]
    K = 2 * T * (10 * m + 6) + N + D + T * B + 2 * float(x["z"].nan_to_num().abs().max()) + 60
    close(y, want["y"], mag["y"], K, ("y", y.dtype))
    close(h, want["h"], mag["h"], K, ("h", h.dtype))
    for k, v in got.items():
        close(v, want["g" + k], mag["g" + k], K, ("grad " + k, v.dtype))


def test_scan_parts_whose_decay_overflows():
    """A > 0 in few long sequences, walked in parts of 64 steps: over a part the decay (up to e^96, e^128)
    is more than a float holds, the states are not.  Zero states stay zero, small ones grow; and the same
    for the gradients.  Bounds as in test_gpu_state_space.py; a part's decay is off by the rounding of its
    exponent, which is less than its steps' together."""
    T, D, N = 1024, 32, 16
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(len(s))).to(DEV)  # noqa: E731
    A = (2.9 + 0.1 * torch.rand(D, N, generator=torch.Generator().manual_seed(1))).to(DEV)
    B, C, delta = r(T, 1, 1, N), r(T, 1, 1, N).flip(0), torch.full((T, 1, D), 1e-3, device=DEV)
    K = 2 * T * (10 * 1.5 + 6) + N + D + T + 60

    def check(u, delta, h0, gy):
        x = {"u": u, "delta": delta, "A": A, "B": B, "C": C, "h0": h0}
        leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
        y, h = ss.state_scan(**leaves, return_state=True)
        got = () if gy is None else torch.autograd.grad(y, list(leaves.values()), gy)
        want, mag = (state_ref.scan(**x, gy=gy, mag=m) for m in (False, True))
        names = [(y, "y"), (h, "h"), *((v, "g" + k) for k, v in zip(leaves, got))]
        assert all(float(want[k].abs().max()) < 1e30 for _, k in names)
        assert max(float(want[k].abs().max()) for _, k in names) > 0
        for v, k in names:
            close(v, want[k], mag[k], K, (k, v.dtype))

    # nothing before step 900, long steps until then (whose gradients would be infinite)
    u, d = r(T, 1, D), delta.clone()
    u[:900], d[:900] = 0, 0.5
    check(u, d, torch.zeros(1, D, N, device=DEV), None)
    # a small state that grows in the first part
    d = delta.clone()
    d[:64] = 0.5
    check(torch.zeros(T, 1, D, device=DEV), d, torch.full((1, D, N), 1e-30, device=DEV), torch.zeros(T, 1, D, device=DEV))
    # no gradient from the long steps at the end; no states either
    d, gy = delta.clone(), r(T, 1, D)
    d[100:], gy[100:] = 0.5, 0
    check(torch.zeros(T, 1, D, device=DEV), d, torch.zeros(1, D, N, device=DEV), gy)
    # a small gradient that grows in the last part
    d, gy = delta.clone(), torch.zeros(T, 1, D, device=DEV)
    d[-64:], gy[-1] = 0.5, 1e-30
    check(torch.zeros(T, 1, D, device=DEV), d, torch.zeros(1, D, N, device=DEV), gy)


# ---------------------------------------------------------------------------------------
# parts that wait for one another
# ---------------------------------------------------------------------------------------
def test_waits_that_run_out_are_counted_and_give_nan(monkeypatch):
    """The same backward with waits of no length: the last part of each sequence is whole, what comes in
    front of it NaN, the call returns, and the next one is as if nothing had been."""
    T, B, D = 300, 480, 8
    lib = _capi.lib()
    x, _, (gy, gh) = scan_case(T, B, D, 16, 1, "f32", seed=1, scale=0.1)
    assert lib.dfsnn_state_scan_backward_launches(T, B, D, 16, 1) == 2
    leaves = {k: v.detach().requires_grad_(True) for k, v in x.items()}

    def run():
        y, h = ss.state_scan(**leaves, softplus=True, return_state=True)
        return dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [gy, gh])))
    want, before = run(), ss.expired_waits()
    assert all(torch.isfinite(v).all() for v in want.values())
    with monkeypatch.context() as m:
        m.setattr(lib, "dfsnn_state_scan_backward", lib.dfsnn_check_state_scan_waits)
        got = run()
    # 480 sequences in two parts
    assert ss.expired_waits() - before == B
    last = int(torch.isnan(got["u"]).any(-1).any(-1).sum())             # steps of the first parts
    assert 0 < last < T and last % 16 == 0
    for k in ("u", "delta", "B"):
        assert torch.isnan(got[k][:last]).all() and torch.equal(got[k][last:], want[k][last:]), k
    for k in ("C", "z"):                                                # these need no later step
        assert torch.equal(got[k], want[k]), k
    for k in ("A", "delta_bias", "h0"):
        assert torch.isnan(got[k]).all(), k
    again = run()
    assert all(torch.equal(again[k], want[k]) for k in want)
    assert ss.expired_waits(DEV) - before == B
