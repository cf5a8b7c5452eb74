"""Cases of the state-space operators: the selective scan and the short causal convolution in
front of it, each over a whole sequence (forward alone, or forward and backward) and for one
token a call.

Sequences are time-major, [T, B, D] (T steps, B sequences, D channels), as everywhere in this
package; a channel's state has N entries and G groups of channels share the scan's B and C.
"""
import math
import os
import random  # noqa: F401  (draw takes a random.Random)
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    """The listed cases.

    scan: T, B, D, N, G; `full`: with skip weight, gate, step bias and softplus (a block of a
      language model), else the bare recurrence; `state`: starts from given states and returns
      the last ones; `ragged`: a padded batch with a length per sequence; `train`: forward and
      backward, else forward alone.
    conv: W taps; `act`: with silu; the other keys as above.
    scan_step / conv_step: one token for each of B requests; `slots` > 0: their states lie in a
      pool of that many slots, found by an index, with idle rows (-1) in between."""
    return [
        # one request's next token through one layer: latency
        {"name": "scan_step_one", "op": "scan_step", "B": 1, "D": 2048, "N": 16, "G": 1,
         "dtype": "bf16", "full": True, "slots": 0},
        # the next tokens of a serving batch, states in a pool
        {"name": "scan_step_pool", "op": "scan_step", "B": 256, "D": 4096, "N": 16, "G": 1,
         "dtype": "bf16", "full": True, "slots": 384},
        # the convolution's part of those two
        {"name": "conv_step_one", "op": "conv_step", "B": 1, "D": 2048, "W": 4, "dtype": "bf16",
         "act": True, "slots": 0},
        {"name": "conv_step_pool", "op": "conv_step", "B": 256, "D": 4096, "W": 4,
         "dtype": "bf16", "act": True, "slots": 384},
        # one long prompt: few rows, a long recurrence, its last state kept for the tokens after
        {"name": "scan_prompt_long", "op": "scan", "T": 32768, "B": 1, "D": 1024, "N": 16, "G": 1,
         "dtype": "bf16", "full": True, "state": True, "ragged": False, "train": False},
        # a padded batch of prompts
        {"name": "scan_prompt_batch", "op": "scan", "T": 1024, "B": 16, "D": 2048, "N": 16, "G": 1,
         "dtype": "f16", "full": True, "state": True, "ragged": True, "train": False},
        # a training step of a layer
        {"name": "scan_train", "op": "scan", "T": 2048, "B": 8, "D": 2048, "N": 16, "G": 1,
         "dtype": "bf16", "full": True, "state": False, "ragged": False, "train": True},
        # the short sequences of spiking networks: 16 time steps, image tokens as the batch
        # (64 images of 64 tokens, width 256, fp32)
        {"name": "scan_train_steps16", "op": "scan", "T": 16, "B": 4096, "D": 256, "N": 16, "G": 1,
         "dtype": "f32", "full": False, "state": False, "ragged": False, "train": True},
        # odd sizes, two groups, a state that is no power of two, padded, with given states
        {"name": "scan_train_odd", "op": "scan", "T": 509, "B": 5, "D": 1002, "N": 12, "G": 2,
         "dtype": "f32", "full": True, "state": True, "ragged": True, "train": True},
        # a long prompt through the convolution
        {"name": "conv_prompt", "op": "conv", "T": 8192, "B": 2, "D": 4096, "W": 4,
         "dtype": "bf16", "act": True, "state": True, "ragged": False, "train": False},
        # a training step through the convolution
        {"name": "conv_train", "op": "conv", "T": 2048, "B": 8, "D": 2048, "W": 4,
         "dtype": "bf16", "act": True, "state": False, "ragged": False, "train": True},
        # odd sizes, three taps, padded, no activation
        {"name": "conv_train_odd", "op": "conv", "T": 509, "B": 5, "D": 1001, "W": 3,
         "dtype": "f32", "act": False, "state": True, "ragged": True, "train": True},
    ]


_MOST_SCAN = 2048 * 8 * 2048 * 16            # T * B * D * N of the largest listed scan
_MOST_CONV = 8192 * 2 * 4096                 # T * B * D of the largest listed convolution
_MOST_STEP = 256 * 4096 * 16                 # B * D * N of the largest listed step


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "conv", "conv", "scan_step", "conv_step"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    D = _log_int(rng, 64, 4096)
    if op in ("scan_step", "conv_step"):
        B = _log_int(rng, 1, 256)
        case = {"op": op, "B": B, "D": D, "dtype": dtype,
                "slots": rng.choice([0, B + rng.randint(0, 64)])}
        if op == "conv_step":
            return {**case, "W": rng.choice([2, 3, 4, 4]), "act": rng.random() < 0.7}
        N, G = rng.choice([8, 12, 16, 16, 16, 24, 32, 64]), rng.choice([1, 1, 2, 4])
        case["D"] = D = max(G, min(D, _MOST_STEP // (B * N)) // G * G)
        return {**case, "N": N, "G": G, "full": rng.random() < 0.7}
    flags = {"state": rng.random() < 0.5, "ragged": rng.random() < 0.4,
             "train": rng.random() < 0.5}
    if op == "conv":
        T = _log_int(rng, 1, 16384)
        B = _log_int(rng, 1, max(1, min(64, _MOST_CONV // (T * D))))
        return {"op": op, "T": T, "B": B, "D": D, "W": rng.choice([2, 3, 4, 4]), "dtype": dtype,
                "act": rng.random() < 0.7, **flags}
    N, G = rng.choice([8, 12, 16, 16, 16, 24, 32, 64]), rng.choice([1, 1, 2, 4])
    T = _log_int(rng, 1, 16384)
    # a training pass of the plain form costs more than a forward one of the same size
    most = _MOST_SCAN // 2 if flags["train"] else _MOST_SCAN
    D = max(G, min(D, most // (T * N)) // G * G)
    B = _log_int(rng, 1, max(1, min(64, most // (T * D * N))))
    return {"op": op, "T": T, "B": B, "D": D, "N": N, "G": G, "dtype": dtype,
            "full": rng.random() < 0.7, **flags}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def prepare(case, seed):
    """What a program holds before the call.  The sequences are slices of the projections that
    make them, as in a model: the convolution's input and the scan's gate are halves of one
    [T, B, 2 D] projection, B and C parts of another."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        x = torch.randn(shape, device=dev, generator=g, dtype=torch.float32)
        return (x.mul_(scale) if scale != 1.0 else x).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, device=dev, generator=g, dtype=torch.float32)

    op, B, D = case["op"], case["B"], case["D"]
    s = {"case": dict(case)}
    if op in ("conv", "conv_step"):
        W = case["W"]
        s["weight"] = normal(D, W, scale=W ** -0.5)
        s["bias"] = normal(D, scale=0.1)
        lead = (case["T"], B) if op == "conv" else (B,)
        s["x"] = normal(*lead, 2 * D, dtype=dt)[..., :D]
        if op == "conv":
            s["state"] = normal(B, W - 1, D, dtype=dt) if case["state"] else None
            s["grads"] = [normal(*lead, D, dtype=dt)] if case["train"] else []
            if case["train"] and case["state"]:
                s["grads"].append(normal(B, W - 1, D, dtype=dt))
        else:
            s["state"] = normal(case["slots"] or B, W - 1, D, dtype=dt)
    else:
        N, G, full = case["N"], case["G"], case["full"]
        lead = (case["T"], B) if op == "scan" else (B,)
        s["u"] = torch.nn.functional.silu(normal(*lead, D)).to(dt)
        # decay rates 1 .. N per channel, as the usual initialisation has them, a little apart
        s["A"] = -(torch.arange(1, N + 1, device=dev, dtype=torch.float32)
                   * (0.8 + 0.4 * uniform(D, N)))
        step = torch.exp(uniform(D) * math.log(100.0)) * 1e-3          # 0.001 .. 0.1
        if full:
            s["delta"] = normal(*lead, D, scale=0.5, dtype=dt)
            s["delta_bias"] = torch.log(torch.expm1(step))
            s["D"] = 1.0 + normal(D, scale=0.1)
            s["z"] = normal(*lead, 2 * D, dtype=dt)[..., D:]
        else:
            s["delta"] = (step * (0.5 + uniform(*lead, D))).to(dt)
            s["delta_bias"] = s["D"] = s["z"] = None
        bc = normal(*lead, 32 + 2 * G * N, dtype=dt)[..., 32:]
        s["B"] = bc[..., :G * N].unflatten(-1, (G, N))
        s["C"] = bc[..., G * N:].unflatten(-1, (G, N))
        if op == "scan":
            s["h0"] = normal(B, D, N) if case["state"] else None
            s["grads"] = [normal(*lead, D, dtype=dt)] if case["train"] else []
            if case["train"] and case["state"]:
                s["grads"].append(normal(B, D, N))
        else:
            s["state"] = normal(case["slots"] or B, D, N)
    if op in ("scan", "conv"):
        s["lengths"] = None
        if case["ragged"]:
            n = torch.randint(1, case["T"] + 1, (B,), device=dev, generator=g, dtype=torch.int32)
            if B > 2:
                n[B // 2] = 0                       # a sequence that has ended
            s["lengths"] = n
        if case["train"]:
            s["leaves"] = [k for k in (("x", "weight", "bias", "state") if op == "conv" else
                                       ("u", "delta", "A", "B", "C", "D", "z", "delta_bias",
                                        "h0")) if s[k] is not None]
            for k in s["leaves"]:
                s[k].requires_grad_(True)
    else:
        s["index"] = None
        if case["slots"]:
            i = torch.randperm(case["slots"], device=dev, generator=g)[:B].to(torch.int32)
            if B > 3:
                i[1::4] = -1                        # idle rows of a padded batch
            s["index"] = i
        s["state_out"] = s["state"].clone()         # the step leaves the state before it intact
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    with torch.no_grad():
        if op == "scan":
            return _plain_scan(state)
        if op == "conv":
            return _plain_conv(state)
        return _plain_scan_step(state) if op == "scan_step" else _plain_conv_step(state)


_module = None


def _state_space():
    global _module
    if _module is None:
        root = os.path.join(os.getcwd(), "df-snn-official_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from dfsnn_b200 import state_space
        _module = state_space
    return _module


def _run_own(op, s):
    ss, case = _state_space(), s["case"]
    if op == "scan_step":
        y = ss.state_scan_step(s["u"], s["delta"], s["state"], s["A"], s["B"], s["C"], D=s["D"],
                               z=s["z"], delta_bias=s["delta_bias"], softplus=case["full"],
                               index=s["index"], state_out=s["state_out"])
        return [y, s["state_out"]]
    if op == "conv_step":
        y = ss.short_conv_step(s["x"], s["state"], s["weight"], bias=s["bias"],
                               activation="silu" if case["act"] else None, index=s["index"],
                               state_out=s["state_out"])
        return [y, s["state_out"]]
    if op == "scan":
        out = ss.state_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                            delta_bias=s["delta_bias"], softplus=case["full"], h0=s["h0"],
                            lengths=s["lengths"], return_state=case["state"])
    else:
        out = ss.short_conv(s["x"], s["weight"], bias=s["bias"],
                            activation="silu" if case["act"] else None, state=s["state"],
                            lengths=s["lengths"], return_state=case["state"])
    out = list(out) if case["state"] else [out]
    if not case["train"]:
        return out
    grads = torch.autograd.grad(out, [s[k] for k in s["leaves"]], s["grads"])
    return [o.detach() for o in out] + list(grads)


# ---------------------------------------------------------------------------------------
# plain forms (32 bits, rounded once at the end)
# ---------------------------------------------------------------------------------------
def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _per_channel(x, D):
    """[..., G, N] -> [..., D, N]: the entries that each channel's group shares."""
    G = x.shape[-2]
    return x.float().unsqueeze(-2).expand(*x.shape[:-2], G, D // G, x.shape[-1]).flatten(-3, -2)


def _group_sum(x, G):
    return x.unflatten(-2, (G, x.shape[-2] // G)).sum(-2)


def _linear_scan(a, x, h0):
    """h_t = a_t h_(t-1) + x_t along the first axis, in place of x; chunks of about sqrt(T)
    steps run side by side and are joined afterwards.  Returns (states, last state)."""
    T = a.shape[0]
    K = max(1, int(round(math.sqrt(T))))
    nc = -(-T // K)
    if nc * K != T:
        pad = nc * K - T
        a = torch.cat([a, torch.ones_like(a[:1]).expand(pad, *a.shape[1:])])
        x = torch.cat([x, torch.zeros_like(x[:1]).expand(pad, *x.shape[1:])])
    a, x = a.unflatten(0, (nc, K)), x.unflatten(0, (nc, K))
    p = torch.empty_like(a)                      # products of the decays within each chunk
    p[:, 0] = a[:, 0]
    for k in range(1, K):
        x[:, k] += a[:, k] * x[:, k - 1]
        p[:, k] = a[:, k] * p[:, k - 1]
    start = torch.empty_like(x[:, 0])
    h = torch.zeros_like(x[0, 0]) if h0 is None else h0
    for c in range(nc):
        start[c] = h
        h = p[c, -1] * h + x[c, -1]
    x += p.mul_(start.unsqueeze(1))
    return x.flatten(0, 1)[:T], h


def _plain_scan(s):
    case = s["case"]
    T, B, D, N, G = (case[k] for k in ("T", "B", "D", "N", "G"))
    A = s["A"]
    u, raw = s["u"].float(), s["delta"].float()
    if s["delta_bias"] is not None:
        raw = raw + s["delta_bias"]
    dt = _softplus(raw) if case["full"] else raw
    live = None
    Bc, Cc = s["B"].float(), s["C"].float()
    if s["lengths"] is not None:
        live = (torch.arange(T, device=u.device)[:, None] < s["lengths"][None, :])[..., None]
        dt, u = dt * live, torch.where(live, u, 0.0)
    a = torch.exp(dt.unsqueeze(-1) * A)
    x = (dt * u).unsqueeze(-1) * _per_channel(Bc, D)
    h, last = _linear_scan(a, x, s["h0"])
    pre = (h * _per_channel(Cc, D)).sum(-1)
    if s["D"] is not None:
        pre = pre + s["D"] * u
    y = pre
    if s["z"] is not None:
        z = s["z"].float()
        sg = torch.sigmoid(z)
        y = pre * (z * sg)
    if live is not None:
        y = torch.where(live, y, 0.0)
    ot = s["u"].dtype
    out = [y.to(ot)] + ([last] if case["state"] else [])
    if not case["train"]:
        return out
    gy = s["grads"][0].float()
    if live is not None:
        gy = torch.where(live, gy, 0.0)
    got = {}
    if s["z"] is not None:
        got["z"] = gy * pre * (sg * (1 + z * (1 - sg)))
        gy = gy * (z * sg)
    del pre, y
    got["C"] = _group_sum(gy.unsqueeze(-1) * h, G)
    # g_t = C_t gy_t + a_(t+1) g_(t+1): the same scan with time reversed
    drive = gy.unsqueeze(-1) * _per_channel(Cc, D)
    if case["state"]:
        drive[-1] += s["grads"][1]
    ones = torch.ones_like(a[:1])
    g = _linear_scan(torch.cat([a[1:], ones]).flip(0), drive.flip(0), None)[0].flip(0)
    del drive
    h = torch.cat([torch.zeros_like(h[:1]) if s["h0"] is None else s["h0"][None], h[:-1]])
    if case["state"]:
        got["h0"] = a[0] * g[0]
    w = g * a * h                                # g_t times the decayed state
    del a, h
    gb = (g * _per_channel(Bc, D)).sum(-1)
    got["B"] = _group_sum(g * (dt * u).unsqueeze(-1), G)
    del g
    got["u"] = dt * gb
    gdt = u * gb + (w * A).sum(-1)
    got["A"] = (w * dt.unsqueeze(-1)).sum((0, 1))
    if live is not None:
        gdt = torch.where(live, gdt, 0.0)
        got["B"] = torch.where(live[..., None], got["B"], 0.0)
    if s["D"] is not None:
        got["u"] = got["u"] + s["D"] * gy
        got["D"] = (gy * u).sum((0, 1))
    if case["full"]:
        gdt = gdt * torch.sigmoid(raw)
    got["delta"] = gdt
    if s["delta_bias"] is not None:
        got["delta_bias"] = gdt.sum((0, 1))
    return out + [got[k].to(s[k].dtype) for k in s["leaves"]]


def _plain_conv(s):
    case = s["case"]
    T, B, D, W = (case[k] for k in ("T", "B", "D", "W"))
    x = s["x"].float()
    before = torch.zeros(W - 1, B, D, device=x.device) if s["state"] is None \
        else s["state"].float().transpose(0, 1)
    live = n = None
    if s["lengths"] is not None:
        n = s["lengths"].long()
        live = (torch.arange(T, device=x.device)[:, None] < n[None, :])[..., None]
        x = torch.where(live, x, 0.0)
    x = torch.cat([before, x])                   # [W - 1 + T, B, D]
    w = s["weight"].float()
    pre = s["bias"].float() + sum(w[:, j] * x[j:j + T] for j in range(W))
    y = pre * torch.sigmoid(pre) if case["act"] else pre
    if live is not None:
        y = torch.where(live, y, 0.0)
    out = [y.to(s["x"].dtype)]
    # the last W - 1 inputs of each sequence: rows n .. n + W - 2 of the extended one
    rows = None
    if case["state"]:
        rows = torch.arange(W - 1, device=x.device)[None, :] + (n[:, None] if n is not None else T)
        rows = rows.expand(B, W - 1)
        out.append(x[rows, torch.arange(B, device=x.device)[:, None]].to(s["x"].dtype))
    if not case["train"]:
        return out
    gp = s["grads"][0].float()
    if live is not None:
        gp = torch.where(live, gp, 0.0)
    if case["act"]:
        sg = torch.sigmoid(pre)
        gp = gp * (sg * (1 + pre * (1 - sg)))
    gx = torch.zeros_like(x)
    for j in range(W):
        gx[j:j + T] += w[:, j] * gp
    if rows is not None:
        gx[rows, torch.arange(B, device=x.device)[:, None]] += s["grads"][1].float()
    got = {"x": gx[W - 1:], "state": gx[:W - 1].transpose(0, 1), "bias": gp.sum((0, 1)),
           "weight": torch.stack([(gp * x[j:j + T]).sum((0, 1)) for j in range(W)], 1)}
    return out + [got[k].to(s[k].dtype) for k in s["leaves"]]


def _rows(s):
    """(live rows, their slots) of a step; None without an index."""
    if s["index"] is None:
        return None, None
    live = s["index"] >= 0
    return live, s["index"].clamp_min(0).long()


def _store(s, new, live, slot):
    """The new states at their slots of state_out; the other slots stay."""
    if live is None:
        s["state_out"].copy_(new)
    else:
        keep = live.reshape(-1, *([1] * (new.dim() - 1)))
        spare = torch.cat([s["state_out"], s["state_out"][:1]])
        at = torch.where(live, slot, s["state_out"].shape[0])       # idle rows to the spare slot
        spare[at] = torch.where(keep, new, 0.0).to(spare.dtype)
        s["state_out"].copy_(spare[:-1])


def _plain_scan_step(s):
    D = s["case"]["D"]
    live, slot = _rows(s)
    h = s["state"] if slot is None else s["state"][slot]
    u, dt = s["u"].float(), s["delta"].float()
    if s["delta_bias"] is not None:
        dt = dt + s["delta_bias"]
    if s["case"]["full"]:
        dt = _softplus(dt)
    h = torch.exp(dt.unsqueeze(-1) * s["A"]) * h + (dt * u).unsqueeze(-1) * _per_channel(s["B"], D)
    y = (h * _per_channel(s["C"], D)).sum(-1)
    if s["D"] is not None:
        y = y + s["D"] * u
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    if live is not None:
        y = torch.where(live[:, None], y, 0.0)
    _store(s, h, live, slot)
    return [y.to(s["u"].dtype), s["state_out"]]


def _plain_conv_step(s):
    live, slot = _rows(s)
    old = s["state"] if slot is None else s["state"][slot]
    x = torch.cat([old, s["x"].unsqueeze(1)], 1)                     # [B, W, D]
    y = s["bias"].float() + (x.float() * s["weight"].float().t()).sum(1)
    if s["case"]["act"]:
        y = y * torch.sigmoid(y)
    if live is not None:
        y = torch.where(live[:, None], y, 0.0)
    _store(s, x[:, 1:], live, slot)
    return [y.to(s["x"].dtype), s["state_out"]]


# ---------------------------------------------------------------------------------------
# the cost that no implementation avoids
# ---------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    op, B, D = case["op"], case["B"], case["D"]
    if op == "conv_step":
        rows = _live_rows(case)
        return {"bytes": rows * D * e * (2 + 2 * (case["W"] - 1)) + D * (case["W"] + 1) * 4,
                "flops": rows * D * (2 * case["W"] + (4 if case["act"] else 0))}
    if op == "scan_step":
        N, rows = case["N"], _live_rows(case)
        io = 4 if case["full"] else 3
        return {"bytes": rows * (D * e * io + 2 * case["G"] * N * e + D * N * 8)
                + D * N * 4 + (D * 8 if case["full"] else 0),
                "flops": rows * D * N * 7}
    steps = case["T"] * B * (0.5 if case["ragged"] else 1.0)    # a ragged batch is about half full
    if op == "conv":
        W = case["W"]
        seqs = 4 if case["train"] else 2                        # x, y; and grad y, grad x
        taps = 2 * W + (4 if case["act"] else 0)
        state = B * (W - 1) * D * e * (2 if case["state"] else 0)
        return {"bytes": steps * D * e * seqs + D * (W + 1) * 4 * (2 if case["train"] else 1)
                + state * (2 if case["train"] else 1),
                "flops": steps * D * taps * (3 if case["train"] else 1)}
    N = case["N"]
    seqs = 4 if case["full"] else 3                             # u, delta, y (and z)
    if case["train"]:
        seqs = 2 * seqs
    twice = 2 if case["train"] else 1
    return {"bytes": steps * D * e * seqs + twice * (steps * 2 * case["G"] * N * e + D * N * 4
                                                     + (D * 8 if case["full"] else 0)
                                                     + (B * D * N * 8 if case["state"] else 0)),
            "flops": steps * D * N * (22 if case["train"] else 7)}


def _live_rows(case):
    B = case["B"]
    return B - len(range(1, B, 4)) if case["slots"] and B > 3 else B


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "scan":
            return _exact_scan(case, s)
        if case["op"] == "conv":
            return _exact_conv(case, s)
        return _exact_scan_step(case, s) if case["op"] == "scan_step" else _exact_conv_step(case, s)


def _d(x):
    return None if x is None else x.detach().double()


def _silu64(x):
    return x / (1 + torch.exp(-x))


def _dsilu64(x):
    q = 1 / (1 + torch.exp(-x))
    return q + x * q * (1 - q)


def _log1pexp64(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def _exact_scan(case, s):
    """Sequence after sequence of equal length would be the definition; here every sequence of
    the batch takes its step t together, and those that have ended keep their state."""
    T, B, D, N, G = (case[k] for k in ("T", "B", "D", "N", "G"))
    n = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"].long()
    group = torch.arange(D, device="cuda") // (D // G)
    A = _d(s["A"])
    skip = torch.zeros(D, device="cuda", dtype=torch.float64) if s["D"] is None else _d(s["D"])
    bias = torch.zeros_like(skip) if s["delta_bias"] is None else _d(s["delta_bias"])
    keep = torch.empty(T + 1 if case["train"] else 1, B, D, N, device="cuda", dtype=torch.float64)
    h = torch.zeros(B, D, N, device="cuda", dtype=torch.float64) if s["h0"] is None else _d(s["h0"])
    keep[0] = h
    steps = int(n.max())
    y = torch.zeros(T, B, D, device="cuda", dtype=torch.float64)
    padded = bool((n < T).any())

    def at(t):
        on = (n > t)[:, None]
        raw = torch.where(on, _d(s["delta"][t]) + bias, 0.0)
        dt = _log1pexp64(raw) if case["full"] else raw
        return (on, raw, torch.where(on, dt, 0.0), torch.where(on, _d(s["u"][t]), 0.0),
                _d(s["B"][t])[:, group], _d(s["C"][t])[:, group])

    for t in range(steps):
        on, raw, dt, u, b, c = at(t)
        new = torch.exp(dt[..., None] * A) * h + (dt * u)[..., None] * b
        h = torch.where(on[..., None], new, h) if padded else new
        o = (h * c).sum(-1) + skip * u
        if s["z"] is not None:
            o = o * _silu64(_d(s["z"][t]))
        y[t] = torch.where(on, o, 0.0)
        if case["train"]:
            keep[t + 1] = h
    out = [y] + ([h] if case["state"] else [])
    if not case["train"]:
        return out
    z64 = {"dtype": torch.float64, "device": "cuda"}
    got = {"u": torch.zeros(T, B, D, **z64), "delta": torch.zeros(T, B, D, **z64),
           "z": torch.zeros(T, B, D, **z64), "B": torch.zeros(T, B, G, N, **z64),
           "C": torch.zeros(T, B, G, N, **z64), "A": torch.zeros(D, N, **z64),
           "D": torch.zeros(D, **z64), "delta_bias": torch.zeros(D, **z64)}
    lam = _d(s["grads"][1]) if case["state"] else torch.zeros(B, D, N, **z64)
    for t in range(steps - 1, -1, -1):
        on, raw, dt, u, b, c = at(t)
        gy = torch.where(on, _d(s["grads"][0][t]), 0.0)
        h, hp = keep[t + 1], keep[t]
        if s["z"] is not None:
            z = _d(s["z"][t])
            got["z"][t] = torch.where(on, gy * ((h * c).sum(-1) + skip * u) * _dsilu64(z), 0.0)
            gy = gy * _silu64(z)
        got["C"][t] = (gy[..., None] * h).reshape(B, G, D // G, N).sum(2)
        lam = lam + gy[..., None] * c
        a = torch.exp(dt[..., None] * A)
        q = lam * a * hp * on[..., None]
        lb = (lam * b).sum(-1) * on
        got["B"][t] = (lam * (dt * u * on)[..., None]).reshape(B, G, D // G, N).sum(2)
        got["u"][t] = dt * lb + skip * gy
        gd = u * lb + (q * A).sum(-1)
        got["delta"][t] = gd / (1 + torch.exp(-raw)) if case["full"] else gd
        got["A"] += (q * dt[..., None]).sum(0)
        got["D"] += (gy * u).sum(0)
        got["delta_bias"] += got["delta"][t].sum(0)
        lam = torch.where(on[..., None], a * lam, lam) if padded else a * lam
    got["h0"] = lam
    return out + [got[k] for k in s["leaves"]]


def _exact_conv(case, s):
    T, B, D, W = (case[k] for k in ("T", "B", "D", "W"))
    w, bias = _d(s["weight"]), _d(s["bias"])
    z64 = {"dtype": torch.float64, "device": "cuda"}
    y, last = torch.zeros(T, B, D, **z64), torch.zeros(B, W - 1, D, **z64)
    got = {"x": torch.zeros(T, B, D, **z64), "weight": torch.zeros(D, W, **z64),
           "bias": torch.zeros(D, **z64), "state": torch.zeros(B, W - 1, D, **z64)}
    for b in range(B):
        n = T if s["lengths"] is None else int(s["lengths"][b])
        head = torch.zeros(W - 1, D, **z64) if s["state"] is None else _d(s["state"][b])
        x = torch.cat([head, _d(s["x"][:n, b])])
        win = x.unfold(0, W, 1) if n else torch.zeros(0, D, W, **z64)      # [n, D, W]
        pre = torch.einsum("tdw,dw->td", win, w) + bias
        y[:n, b] = _silu64(pre) if case["act"] else pre
        last[b] = x[n:]
        if case["train"]:
            gp = _d(s["grads"][0][:n, b])
            if case["act"]:
                gp = gp * _dsilu64(pre)
            got["weight"] += torch.einsum("td,tdw->dw", gp, win)
            got["bias"] += gp.sum(0)
            gx = torch.zeros_like(x)
            if case["state"]:
                gx[n:] += _d(s["grads"][1][b])
            for i in range(W):                                   # x[t + i] enters y[t] by tap i
                gx[i:i + n] += gp * w[:, i]
            got["x"][:n, b], got["state"][b] = gx[W - 1:], gx[:W - 1]
    out = [y] + ([last] if case["state"] else [])
    return out + [got[k] for k in s["leaves"]] if case["train"] else out


def _exact_scan_step(case, s):
    D, G = case["D"], case["G"]
    group = torch.arange(D, device="cuda") // (D // G)
    y = torch.zeros(case["B"], D, device="cuda", dtype=torch.float64)
    pool = _d(s["state"]).clone()
    rows = list(range(case["B"])) if s["index"] is None else s["index"].tolist()
    for r, slot in enumerate(rows):
        if slot < 0:
            continue
        u, dt = _d(s["u"][r]), _d(s["delta"][r])
        if s["delta_bias"] is not None:
            dt = dt + _d(s["delta_bias"])
        if case["full"]:
            dt = _log1pexp64(dt)
        pool[slot] = (torch.exp(dt[:, None] * _d(s["A"])) * pool[slot]
                      + (dt * u)[:, None] * _d(s["B"][r])[group])
        o = (pool[slot] * _d(s["C"][r])[group]).sum(-1)
        if s["D"] is not None:
            o = o + _d(s["D"]) * u
        y[r] = o if s["z"] is None else o * _silu64(_d(s["z"][r]))
    return [y, pool]


def _exact_conv_step(case, s):
    y = torch.zeros(case["B"], case["D"], device="cuda", dtype=torch.float64)
    pool = _d(s["state"]).clone()
    rows = list(range(case["B"])) if s["index"] is None else s["index"].tolist()
    for r, slot in enumerate(rows):
        if slot < 0:
            continue
        x = torch.cat([pool[slot], _d(s["x"][r])[None]])
        pre = torch.einsum("wd,dw->d", x, _d(s["weight"])) + _d(s["bias"])
        y[r] = _silu64(pre) if case["act"] else pre
        pool[slot] = x[1:]
    return [y, pool]
