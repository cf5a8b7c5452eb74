"""State-space layer without a GPU: the 64-bit formulas that the GPU tests compare against
(against autograd and against differences), argument refusals, argument structures."""
import ctypes
import os
import re

import pytest
import torch

import state_ref
from dfsnn_b200 import _capi, state_space as ss

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def scan_inputs(T, B, D, N, G, full, state, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = {"u": r(T, B, D), "delta": r(T, B, D) if full else r(T, B, D).abs() * 0.2,
         "A": -r(D, N).abs() - 0.2, "B": r(T, B, G, N), "C": r(T, B, G, N)}
    if full:
        x.update(D=r(D), z=r(T, B, D), delta_bias=r(D))
    if state:
        x["h0"] = r(B, D, N)
    return x


def scan_autograd(x, softplus, lengths):
    """The definition with torch's own differentiation, sequence by sequence."""
    u = x["u"]
    T, B, D = u.shape
    G, N = x["B"].shape[2:]
    dt = x["delta"] + x.get("delta_bias", 0)
    dt = torch.nn.functional.softplus(dt) if softplus else dt
    rep = lambda v: v.repeat_interleave(D // G, dim=1)  # noqa: E731
    ys, hs = [], []
    for b in range(B):
        h = x["h0"][b] if "h0" in x else torch.zeros(D, N, dtype=torch.float64)
        for t in range(T):
            if t >= int(lengths[b]):
                ys.append(torch.zeros(D, dtype=torch.float64))
                continue
            h = torch.exp(dt[t, b][:, None] * x["A"]) * h \
                + (dt[t, b] * u[t, b])[:, None] * rep(x["B"][t, b][None])[0]
            y = (rep(x["C"][t, b][None])[0] * h).sum(-1)
            if "D" in x:
                y = y + x["D"] * u[t, b]
            if "z" in x:
                y = y * torch.nn.functional.silu(x["z"][t, b])
            ys.append(y)
        hs.append(h)
    return torch.stack(ys).reshape(B, T, D).transpose(0, 1), torch.stack(hs)


@pytest.mark.parametrize("full,state", [(True, True), (False, False), (True, False)])
def test_scan_formula_against_autograd_and_differences(full, state):
    x = scan_inputs(7, 3, 4, 3, 2, full, state)
    n = torch.tensor([7, 4, 0])
    leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
    y, h = scan_autograd(leaves, full, n)
    gy, gh = torch.randn_like(y), torch.randn_like(h)
    want = torch.autograd.grad([y, h], list(leaves.values()), [gy, gh], allow_unused=True)
    got = state_ref.scan(**x, softplus=full, lengths=n, gy=gy, gh=gh)
    assert torch.allclose(got["y"], y, rtol=1e-12, atol=1e-12)
    assert torch.allclose(got["h"], h, rtol=1e-12, atol=1e-12)
    for k, w in zip(leaves, want):
        assert torch.allclose(got["g" + k], w, rtol=1e-11, atol=1e-11), k
    loss = lambda v: sum((a * b).sum() for a, b in zip(  # noqa: E731
        [state_ref.scan(**v, softplus=full, lengths=n)[k] for k in ("y", "h")], (gy, gh)))
    for k in x:
        v = torch.randn_like(x[k])
        up, down = ({**x, k: x[k] + s * 1e-6 * v} for s in (1, -1))
        slope = (loss(up) - loss(down)) / 2e-6
        assert abs(slope - (got["g" + k] * v).sum()) < 1e-6 * (1 + abs(slope)), k


@pytest.mark.parametrize("W", [1, 2, 4])
@pytest.mark.parametrize("act", [False, True])
def test_conv_formula_against_autograd(W, act):
    g = torch.Generator().manual_seed(W)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    x, w, b, s = r(6, 3, 5), r(5, W), r(5), r(3, W - 1, 5)
    n = torch.tensor([6, 2, 0])
    ys, lasts = [], []
    for k in range(3):
        e = torch.cat([s[k], x[:n[k], k]])
        p = [b + sum(w[:, j] * e[t + j] for j in range(W)) for t in range(int(n[k]))]
        p = torch.stack(p) if p else torch.zeros(0, 5, dtype=torch.float64)
        y = torch.nn.functional.silu(p) if act else p
        ys.append(torch.cat([y, torch.zeros(6 - len(y), 5, dtype=torch.float64)]))
        lasts.append(e[int(n[k]):])
    y, last = torch.stack(ys, 1), torch.stack(lasts)
    gy, gl = torch.randn_like(y), torch.randn_like(last)
    want = torch.autograd.grad([y, last], [x, w, b, s], [gy, gl], allow_unused=True)
    got = state_ref.conv(x, w, b, act, s, n, gy, gl)
    assert torch.allclose(got["y"], y) and torch.equal(got["last"], last)
    for k, v in zip(("gx", "gweight", "gbias", "gstate"), want):
        assert torch.allclose(got[k], torch.zeros_like(got[k]) if v is None else v, atol=1e-12), k


def test_no_cpu_path():
    x = torch.zeros(4, 2, 8)
    bc, A = torch.zeros(4, 2, 16), torch.zeros(8, 16)
    with pytest.raises(RuntimeError):
        ss.state_scan(x, x, A, bc, bc)
    with pytest.raises(RuntimeError):
        ss.short_conv(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError):
        ss.state_scan_step(x[0], x[0], torch.zeros(2, 8, 16), A, bc[0], bc[0])
    with pytest.raises(RuntimeError):
        ss.short_conv_step(x[0], torch.zeros(2, 3, 8), torch.zeros(8, 4))


def test_argument_structures_match_the_header():
    """The packed layouts name as many pointers, 64-bit and 32-bit fields as the header's."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "dfsnn_b200.h")).read(), flags=re.S)
    for name, packed in (("state_scan_args", _capi.STATE_SCAN_ARGS), ("state_scan_grads", _capi.STATE_SCAN_GRADS),
                         ("state_scan_step_args", _capi.STATE_SCAN_STEP_ARGS),
                         ("short_conv_args", _capi.SHORT_CONV_ARGS),
                         ("short_conv_grads", _capi.SHORT_CONV_GRADS),
                         ("short_conv_step_args", _capi.SHORT_CONV_STEP_ARGS)):
        body = re.search(r"typedef struct \{([^{}]*)\} dfsnn_%s;" % name, text).group(1)
        kinds = []
        for decl in body.split(";")[:-1]:
            kind = "P" if "*" in decl else "q" if "long long" in decl else "i"
            kinds += [kind] * len(decl.split(","))
        n = {k: kinds.count(k) for k in "Pqi"}
        assert kinds == ["P"] * n["P"] + ["q"] * n["q"] + ["i"] * n["i"], name
        assert packed.format == "<%dQ%dq" % (n["P"], n["q"]) + ("%di" % n["i"] if n["i"] else ""), name


FAKE = 0x1000                            # never dereferenced: validation fails first


def scan_pack(**k):
    v = dict(u=FAKE, delta=FAKE, z=0, B=FAKE, C=FAKE, A=FAKE, D=0, bias=0, h0=0, lengths=0, y=FAKE, h_last=0,
             kept=0, T=32, batch=2, channels=8, states=16, groups=1, dtype=0, softplus=1, lengths64=0)
    v.update(k)
    return _capi.STATE_SCAN_ARGS.pack(
        *(v[n] for n in ("u", "delta", "z", "B", "C", "A", "D", "bias", "h0", "lengths", "y", "h_last", "kept")),
        *([8] * 14), *(v[n] for n in ("T", "batch", "channels", "states", "groups", "dtype", "softplus",
                                      "lengths64")), 0)


@pytest.mark.parametrize("change,code", [
    (dict(T=0), "SHAPE"), (dict(batch=-1), "SHAPE"), (dict(channels=-1), "SHAPE"), (dict(states=0), "SHAPE"),
    (dict(groups=0), "SHAPE"), (dict(groups=3), "SHAPE"), (dict(states=129), "T_LIMIT"),
    (dict(T=1 << 31), "T_LIMIT"), (dict(channels=1 << 31), "SHAPE"), (dict(dtype=3), "PARAM"),
    (dict(softplus=2), "PARAM"), (dict(lengths64=5), "PARAM"), (dict(u=0), "NULL"), (dict(A=0), "NULL"),
    (dict(C=0), "NULL"), (dict(y=0), "NULL"), (dict(batch=0, u=0), "OK")])
def test_scan_forward_refusals(change, code):
    f = _capi.lib().dfsnn_state_scan_forward
    assert f(scan_pack(**change), None, 0, None) == getattr(_capi, "DFSNN_OK" if code == "OK" else "DFSNN_ERR_" + code)
    assert f(None, None, 0, None) == _capi.DFSNN_ERR_NULL


def test_scan_forward_workspace():
    """Few long sequences need one, and it is checked; many rows need none."""
    L = _capi.lib()
    size = L.dfsnn_state_scan_forward_workspace_size(8192, 1, 64, 16, 1)
    assert size > 0 and L.dfsnn_state_scan_forward_workspace_size(8192, 512, 2048, 16, 1) == 0
    assert L.dfsnn_state_scan_forward_workspace_size(16, 1, 64, 16, 1) == 0
    long = scan_pack(T=8192, batch=1, channels=64)
    for ws, n in ((None, size), (ctypes.c_void_p(0x1008), size), (ctypes.c_void_p(0x1000), size - 1)):
        assert L.dfsnn_state_scan_forward(long, ws, n, None) == _capi.DFSNN_ERR_WORKSPACE


def test_scan_backward_refusals():
    L = _capi.lib()
    f, size = L.dfsnn_state_scan_backward, L.dfsnn_state_scan_backward_workspace_size(32, 2, 8, 16, 1)
    assert size > 0 and L.dfsnn_state_scan_backward_workspace_size(0, 2, 8, 16, 1) == 0
    assert L.dfsnn_state_scan_backward_workspace_size(32, 2, 8, 16, 3) == 0
    assert L.dfsnn_state_scan_kept_floats(32, 2, 8, 16) == (32 // _capi.SCAN_CHUNK - 1) * 2 * 8 * 16
    assert L.dfsnn_state_scan_kept_floats(_capi.SCAN_CHUNK, 2, 8, 16) == 0
    full = [FAKE] * 11
    pack = lambda v: _capi.STATE_SCAN_GRADS.pack(*v, *([8] * 6))  # noqa: E731
    ws, E = ctypes.c_void_p(0x1000), _capi
    assert f(scan_pack(kept=FAKE), pack(full), None, size, None) == E.DFSNN_ERR_WORKSPACE
    assert f(scan_pack(kept=FAKE), pack(full), ctypes.c_void_p(0x1008), size, None) == E.DFSNN_ERR_WORKSPACE
    assert f(scan_pack(kept=FAKE), pack(full), ws, size - 1, None) == E.DFSNN_ERR_WORKSPACE
    assert f(scan_pack(kept=0), pack(full), ws, size, None) == E.DFSNN_ERR_NULL     # long T needs them
    for i in (0, 2, 3, 5, 6, 7):                                                    # the required ones
        assert f(scan_pack(kept=FAKE), pack(full[:i] + [0] + full[i + 1:]), ws, size, None) == E.DFSNN_ERR_NULL
    assert f(scan_pack(kept=FAKE), None, ws, size, None) == E.DFSNN_ERR_NULL


def test_step_refusals():
    L, E = _capi.lib(), _capi
    def scan(**k):
        v = dict(state=FAKE, index=0, batch=4, channels=8, slots=4, states=16, groups=1, dtype=0, softplus=0, i64=0)
        v.update(k)
        return L.dfsnn_state_scan_step(E.STATE_SCAN_STEP_ARGS.pack(
            FAKE, FAKE, 0, FAKE, FAKE, FAKE, 0, 0, v["state"], FAKE, v["index"], FAKE, *([8] * 10), v["batch"],
            v["channels"], v["slots"], v["states"], v["groups"], v["dtype"], v["softplus"], v["i64"], 0), None)
    assert scan(slots=3) == E.DFSNN_ERR_SHAPE and scan(slots=-1, index=FAKE) == E.DFSNN_ERR_SHAPE
    assert scan(groups=3) == E.DFSNN_ERR_SHAPE and scan(states=200) == E.DFSNN_ERR_T_LIMIT
    assert scan(state=0) == E.DFSNN_ERR_NULL and scan(dtype=9) == E.DFSNN_ERR_PARAM
    assert scan(batch=0, slots=0) == E.DFSNN_OK

    def conv(**k):
        v = dict(state=FAKE, index=0, batch=4, channels=8, slots=4, taps=4, dtype=0, silu=0, i64=0)
        v.update(k)
        return L.dfsnn_short_conv_step(E.SHORT_CONV_STEP_ARGS.pack(
            FAKE, FAKE, 0, v["state"], FAKE, v["index"], FAKE, *([8] * 4), v["batch"], v["channels"], v["slots"],
            v["taps"], v["dtype"], v["silu"], v["i64"]), None)
    assert conv(slots=3) == E.DFSNN_ERR_SHAPE and conv(taps=9) == E.DFSNN_ERR_T_LIMIT
    assert conv(taps=0) == E.DFSNN_ERR_T_LIMIT and conv(state=0) == E.DFSNN_ERR_NULL
    assert conv(silu=2) == E.DFSNN_ERR_PARAM and conv(batch=0, slots=0) == E.DFSNN_OK


def test_conv_refusals():
    L, E = _capi.lib(), _capi

    def pack(**k):
        v = dict(x=FAKE, y=FAKE, T=8, batch=2, channels=8, taps=4, dtype=0, silu=0, l64=0)
        v.update(k)
        return E.SHORT_CONV_ARGS.pack(v["x"], FAKE, 0, 0, 0, v["y"], 0, *([8] * 4), v["T"], v["batch"], v["channels"],
                                      v["taps"], v["dtype"], v["silu"], v["l64"])
    f = L.dfsnn_short_conv_forward
    assert f(pack(T=0), None) == E.DFSNN_ERR_SHAPE and f(pack(taps=9), None) == E.DFSNN_ERR_T_LIMIT
    assert f(pack(x=0), None) == E.DFSNN_ERR_NULL and f(pack(y=0), None) == E.DFSNN_ERR_NULL
    assert f(pack(dtype=-1), None) == E.DFSNN_ERR_PARAM and f(pack(channels=0, x=0), None) == E.DFSNN_OK
    b, size = L.dfsnn_short_conv_backward, L.dfsnn_short_conv_backward_workspace_size(8, 2, 8, 4)
    assert size > 0 and L.dfsnn_short_conv_backward_workspace_size(8, 2, 8, 9) == 0
    grads, ws = E.SHORT_CONV_GRADS.pack(*([FAKE] * 6), 8, 8), ctypes.c_void_p(0x1000)
    assert b(pack(), grads, ws, size - 1, None) == E.DFSNN_ERR_WORKSPACE
    assert b(pack(), grads, None, size, None) == E.DFSNN_ERR_WORKSPACE
    assert b(pack(), E.SHORT_CONV_GRADS.pack(FAKE, 0, 0, 0, FAKE, 0, 8, 8), ws, size, None) == E.DFSNN_ERR_NULL


def test_layer_states_and_modes():
    layer = ss.StateSpaceLayer(32, d_state=8, taps=3, groups=2)
    conv, scan = layer.initial_state(5)
    assert conv.shape == (5, 2, 64) and scan.shape == (5, 64, 8)
    assert torch.nn.functional.softplus(layer.delta_bias).min() > 0.9e-3
    with pytest.raises(ValueError):
        ss.StateSpaceLayer(32, step_mode="x")
    with pytest.raises(ValueError):
        ss.StateSpaceLayer(32, groups=3)
    with pytest.raises(RuntimeError):
        layer(torch.zeros(4, 2, 32))
