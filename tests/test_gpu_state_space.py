"""State-space layer on the GPU against the 64-bit formulas of state_ref.py.

Tolerances.  One unit is 2^-24, the largest relative error of one fp32 rounding.  With
m = max |d A| over the call, per step a state's relative error (to the sum of the absolute
values of its terms, which state_ref gives with mag=True) grows by the decay's: softplus at
most 8 units in d (2^x 4, log1p 2, sum 1, rounding 1), log2e A and its product with d 2, both
times m; 2^x itself 4, product and sum 2.  So after T steps at most T (10 m + 6) units, plus
the sum over N states, the gate (2^x 4, its argument 2 max|z|, quotient 4) and the inputs'
products, 30 in all.  A gradient holds a state and an adjoint of T steps each, and sums over
channels, or over steps and sequences: K = 2 T (10 m + 6) + N + D + T B + 2 max|z| + 60 units.
An output of a 16-bit type is rounded once more: half of eps relative to its value (a subnormal
fp16 by half of 2^-24)."""
import pytest
import torch

import state_ref
from dfsnn_b200 import _capi, profiling, state_space as ss

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def close(got, want, mag, units, what):
    got = got.double()
    tol = units * 2.0 ** -24 * mag
    if got_type(what) != torch.float32:
        tol = tol + torch.finfo(got_type(what)).eps / 2 * (want.abs() + tol) + 2.0 ** -25
    bad = ~((got - want).abs() <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], tol.expand_as(got)[bad][:3])


def got_type(what):
    return what[1]


def scan_case(T, B, D, N, G, dtype, full=True, state=True, lengths=None, batch_first=False, seed=0,
              scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    dt = TYPES[dtype]

    def seq(d):
        x = r(B, T, d) if batch_first else r(T, B, d)
        return (x.transpose(0, 1) if batch_first else x).to(dt)

    x = {"u": seq(D), "delta": seq(2 * D)[..., D:] if full else seq(D).abs() * 0.1,
         "A": -(r(D, N).abs() + 0.1) * scale}
    bc = seq(2 * G * N + 3)[..., 3:]
    x["B"], x["C"] = bc[..., :G * N].unflatten(-1, (G, N)), bc[..., G * N:].unflatten(-1, (G, N))
    if full:
        x.update(D=r(D), z=seq(2 * D)[..., :D], delta_bias=r(D))
    if state:
        x["h0"] = r(B, D, N)
    if lengths is not None:
        lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        for k in ("u", "delta", "z", "B", "C"):              # what lies behind is never read
            if k in x:
                pad = torch.arange(T, device=DEV)[:, None] >= lengths[None]
                x[k][pad] = float("nan")
    return x, lengths, (seq(D), r(B, D, N))


def check_scan(x, lengths, grads, softplus, what, use=(True, True)):
    gy, gh = (v if on else None for v, on in zip(grads, use))
    leaves = {k: v.detach().requires_grad_(True) for k, v in x.items()}
    y, h = ss.state_scan(**leaves, softplus=softplus, lengths=lengths, return_state=True)
    plain = ss.state_scan(**x, softplus=softplus, lengths=lengths)
    outs, gs = zip(*[(o, g) for o, g in ((y, gy), (h, gh)) if g is not None])
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs)))
    ref_gy = torch.zeros_like(y) if gy is None else gy
    want, mag = (state_ref.scan(**x, softplus=softplus, lengths=lengths, gy=ref_gy, gh=gh, mag=m)
                 for m in (False, True))
    T, B, D = x["u"].shape
    N = x["A"].shape[1]
    z = float(torch.nan_to_num(x["z"].float()).abs().max()) if "z" in x else 0.0
    K = 2 * T * (10 * want["step_decay"] + 6) + N + D + T * B + 2 * z + 60
    assert torch.equal(plain.detach(), y.detach())              # with and without kept states
    close(y, want["y"], mag["y"], K, (what + " y", y.dtype))
    close(h, want["h"], mag["h"], K, (what + " h", h.dtype))
    for k, v in got.items():
        assert v.dtype == x[k].dtype and v.shape == x[k].shape
        close(v, want["g" + k], mag["g" + k], K, (what + " grad " + k, v.dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,B,D,N,G", [
    (1, 1, 1, 1, 1), (1, 3, 5, 16, 1), (2, 2, 130, 2, 1), (15, 2, 33, 16, 1), (16, 2, 32, 16, 2), (17, 1, 64, 16, 1),
    (33, 2, 96, 12, 3), (50, 3, 70, 8, 2), (40, 2, 40, 4, 4), (37, 2, 24, 5, 1), (31, 2, 40, 32, 2), (20, 2, 18, 33, 1),
    (34, 2, 10, 64, 2), (18, 1, 12, 100, 1), (33, 2, 9, 128, 3), (48, 1, 300, 17, 1)])
def test_scan_against_64_bits(T, B, D, N, G, dtype):
    x, n, grads = scan_case(T, B, D, N, G, dtype, seed=T + N)
    check_scan(x, n, grads, True, f"{T}x{B}x{D} N{N} G{G}")


@pytest.mark.parametrize("lengths", [[40, 1, 0, 17], [0, 0, 0, 0], [16, 32, 15, 33]])
@pytest.mark.parametrize("full", [True, False])
def test_scan_padded(lengths, full):
    x, n, grads = scan_case(40, 4, 50, 16, 2, "bf16", full=full, lengths=lengths, seed=3)
    check_scan(x, n, grads, full, f"padded {lengths}")
    y64 = ss.state_scan(**x, softplus=full, lengths=n.long())
    assert torch.equal(y64, ss.state_scan(**x, softplus=full, lengths=n))


@pytest.mark.parametrize("full,state", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("use", [(True, True), (True, False), (False, True)])
def test_scan_options(full, state, use):
    x, n, grads = scan_case(35, 2, 40, 16, 1, "f32", full=full, state=state, seed=4)
    check_scan(x, n, grads, full, f"full {full} state {state} use {use}", use)


def test_scan_batch_first_views():
    x, n, grads = scan_case(40, 3, 48, 16, 1, "bf16", batch_first=True, lengths=[40, 9, 30], seed=5)
    check_scan(x, n, grads, True, "batch first")
    u = x["u"].nan_to_num().requires_grad_(True)
    y = ss.state_scan(**{**x, "u": u}, softplus=True, lengths=n)
    assert y.stride(1) > y.stride(0)                         # as its input lies
    assert torch.autograd.grad(y.float().sum(), u)[0].shape == u.shape


@pytest.mark.parametrize("T,B,D,N,G,lengths", [
    (300, 480, 8, 16, 1, None), (270, 64, 250, 12, 2, "ragged"), (290, 300, 33, 4, 1, "ragged")])
def test_scan_backward_in_waves(T, B, D, N, G, lengths):
    """More blocks than run at a time: the parts of a sequence run one after another."""
    if lengths:
        lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(T)).tolist()
    x, n, grads = scan_case(T, B, D, N, G, "f32", lengths=lengths, seed=T, scale=0.1)
    check_scan(x, n, grads, True, f"waves {T}x{B}x{D}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
@pytest.mark.parametrize("D,N,G", [(64, 16, 1), (66, 12, 2), (33, 7, 1), (24, 100, 1), (8, 3, 1)])
def test_scan_alignments(D, N, G, shift, dtype):
    """Rows that start on 16 bytes, on 4 and on less, widths that end inside a 16-byte piece."""
    x, n, grads = scan_case(21, 2, D, N, G, dtype, lengths=[21, 18], seed=D + shift)
    for k in ("u", "delta", "z", "B", "C"):
        v = x[k].flatten(2)
        w = torch.empty(*v.shape[:2], v.shape[2] + 8, dtype=v.dtype, device=DEV).fill_(float("nan"))
        w[..., shift:shift + v.shape[2]] = v
        x[k] = w[..., shift:shift + v.shape[2]].unflatten(2, x[k].shape[2:])
    check_scan(x, n, grads, True, f"shift {shift}")


@pytest.mark.parametrize("T,B,D,N,G,lengths", [
    (1000, 1, 40, 16, 1, None), (2049, 4, 36, 16, 2, [2049, 700, 0, 1]), (1500, 2, 12, 100, 1, [16, 1024]),
    (999, 1, 130, 3, 1, None), (1040, 3, 9, 33, 3, [1040, 1039, 129])])
def test_scan_in_parallel_parts(T, B, D, N, G, lengths):
    """Few rows, many steps: parts of a sequence side by side."""
    x, n, grads = scan_case(T, B, D, N, G, "f32", lengths=lengths, seed=T, scale=0.1)
    check_scan(x, n, grads, True, f"parts {T}x{B}x{D}")


def test_scan_large_batch_shares_blocks():
    """More sequences than the backward has blocks for: each block adds several."""
    x, n, grads = scan_case(3, 2500, 3, 4, 1, "f32", seed=6)
    check_scan(x, n, grads, True, "large batch")


@pytest.mark.parametrize("T,B,D,N,G", [(20, 3100, 5, 16, 1), (50, 1600, 42, 8, 2), (16, 3000, 36, 3, 1)])
def test_scan_short_sequences_share_blocks(T, B, D, N, G):
    """Many short sequences: the forward's blocks take several, empty ones among them."""
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(T))
    lengths[::7] = 0
    x, n, grads = scan_case(T, B, D, N, G, "f32", lengths=lengths.tolist(), seed=T)
    check_scan(x, n, grads, True, "short sequences")
    x, n, grads = scan_case(T, B, D, N, G, "bf16", full=False, state=False, seed=T)
    check_scan(x, n, grads, False, "short sequences")


def test_scan_strong_decay():
    """d A far below zero: the decay underflows to zero."""
    x, n, grads = scan_case(20, 2, 33, 16, 1, "f32", seed=7, scale=300.0)
    check_scan(x, n, grads, True, "strong decay")


def test_scan_broadcast_inputs():
    """Expanded inputs: the gradient adds over what was broadcast."""
    x, _, (gy, _) = scan_case(20, 3, 40, 16, 1, "f32", state=False, seed=8)
    B1, z1 = x["B"][:, :1].detach().clone().requires_grad_(True), x["z"][..., :1].clone().requires_grad_(True)
    d = {**x, "B": B1.expand(20, 3, 1, 16), "z": z1.expand(20, 3, 40)}
    y = ss.state_scan(**d, softplus=True)
    gB, gz = torch.autograd.grad(y, (B1, z1), gy)
    e = {k: v.detach().contiguous().requires_grad_(True) for k, v in d.items()}
    ye = ss.state_scan(**e, softplus=True)
    hB, hz = torch.autograd.grad(ye, (e["B"], e["z"]), gy)
    assert torch.equal(y, ye)
    assert torch.equal(gB, hB.sum(1, keepdim=True)) and torch.equal(gz, hz.sum(-1, keepdim=True))


def test_scan_no_wrong_spread_of_nan():
    """A NaN in one sequence or channel stays in it (and in what it feeds)."""
    x, _, _ = scan_case(20, 3, 40, 16, 2, "f32", state=False, seed=9)
    clean = ss.state_scan(**x, softplus=True)
    x["u"][5, 1, 7] = float("nan")
    y = ss.state_scan(**x, softplus=True)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[5:, 1, 7] = True
    assert torch.equal(torch.isnan(y), hit) and torch.equal(y[~hit], clean[~hit])


def test_scan_is_deterministic():
    x, n, (gy, gh) = scan_case(70, 3, 200, 16, 1, "bf16", lengths=[70, 33, 5], seed=10)
    leaves = {k: v.requires_grad_(True) for k, v in x.items()}
    runs = []
    for _ in range(2):
        y, h = ss.state_scan(**leaves, softplus=True, lengths=n, return_state=True)
        runs.append([y, h, *torch.autograd.grad([y, h], list(leaves.values()), [gy, gh])])
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(*runs))


def test_scan_in_parts_equals_whole():
    """A prompt in two calls, the second from the first one's states."""
    x, _, _ = scan_case(64, 2, 96, 16, 1, "f32", seed=11)
    seqs = ("u", "delta", "z", "B", "C")
    y, h = ss.state_scan(**x, softplus=True, return_state=True)
    y1, h1 = ss.state_scan(**{k: v[:32] if k in seqs else v for k, v in x.items()}, softplus=True, return_state=True)
    y2, h2 = ss.state_scan(**{**{k: v[32:] if k in seqs else v for k, v in x.items()}, "h0": h1}, softplus=True,
                           return_state=True)
    # cut at a tile's end: the same operations in the same order
    assert torch.equal(torch.cat([y1, y2]), y) and torch.equal(h2, h)


def test_offsets_past_32_bits():
    """Sequences of more than 2^31 elements: their last rows as in a call of their own."""
    T, B, D, N, last = 1100, 1030, 2048, 4, 160
    g = torch.Generator(device=DEV).manual_seed(1)
    u = torch.randn(T, B, D, generator=g, device=DEV, dtype=torch.bfloat16)
    dt = torch.rand(T, B, D, generator=g, device=DEV, dtype=torch.bfloat16) * 0.1
    A, bc = -torch.rand(D, N, device=DEV), torch.randn(T, B, 2, N, generator=g, device=DEV).bfloat16()
    assert u.numel() > 2 ** 31
    full, part = ((u, dt, bc), tuple(t[:, -last:].contiguous() for t in (u, dt, bc)))

    def run(u, dt, bc):
        u, dt = u.detach().requires_grad_(True), dt.detach().requires_grad_(True)
        y = ss.state_scan(u, dt, A, bc[:, :, :1], bc[:, :, 1:])
        return [y.detach()[:, -last:], *(v[:, -last:] for v in torch.autograd.grad(y, (u, dt), torch.ones_like(y)))]
    for a, b in zip(run(*full), run(*part)):
        assert torch.equal(a, b)
    w = torch.randn(D, 4, device=DEV)

    def conv(u):
        u = u.detach().requires_grad_(True)
        y = ss.short_conv(u, w, None, "silu")
        return [y.detach()[:, -last:], torch.autograd.grad(y, u, torch.ones_like(y))[0][:, -last:]]
    for a, b in zip(conv(u), conv(part[0])):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls on two streams, each with parts that wait for one another or side by side."""
    cases = [scan_case(T, B, D, 16, 1, "f32", seed=40 + T) for T, B, D in ((300, 480, 8), (260, 500, 30), (900, 1, 64))]
    leaves = [{k: v.requires_grad_(True) for k, v in x.items()} for x, _, _ in cases]

    def run(i):
        y, h = ss.state_scan(**leaves[i], softplus=True, return_state=True)
        return [y, h, *torch.autograd.grad([y, h], list(leaves[i].values()), list(cases[i][2]))]
    want = [run(i) for i in range(3)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [None] * 3
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(i)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_empty_batch_and_channels():
    for B, D in ((0, 8), (2, 0)):
        x, _, (gy, _) = scan_case(4, B, D, 16, 1, "f32", seed=12)
        leaves = {k: v.requires_grad_(True) for k, v in x.items()}
        y, h = ss.state_scan(**leaves, softplus=True, return_state=True)
        assert y.shape == (4, B, D) and h.shape == (B, D, 16)
        assert torch.autograd.grad(y, leaves["A"], gy)[0].abs().sum() == 0
        w = torch.ones(D, 4, device=DEV, requires_grad=True)
        c = ss.short_conv(x["u"].detach(), w)
        assert c.shape == (4, B, D) and torch.autograd.grad(c, w, gy)[0].abs().sum() == 0


# ---------------------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------------------
def step_case(B, D, N, G, dtype, slots, seed=0):
    x, _, _ = scan_case(1, B, D, N, G, dtype, state=False, seed=seed)
    row = {k: v[0] if k in ("u", "delta", "z", "B", "C") else v for k, v in x.items()}
    pool = torch.randn(slots, D, N, device=DEV)
    return x, row, pool


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (1, 130, 16, 1), (3, 96, 12, 3), (5, 33, 4, 1), (2, 40, 8, 2),
                                     (2, 20, 5, 1), (4, 24, 32, 2), (2, 10, 17, 1), (3, 12, 64, 1), (2, 9, 100, 3),
                                     (2, 7, 128, 1), (2, 6, 127, 2),
                                     (130, 650, 16, 1), (300, 514, 4, 2), (200, 516, 8, 3), (150, 202, 64, 1),
                                     (100, 330, 32, 2), (160, 515, 12, 1), (90, 701, 3, 1)])
def test_scan_step_against_64_bits(B, D, N, G, dtype):
    x, row, pool = step_case(B, D, N, G, dtype, B, seed=B + N)
    kw = dict(softplus=True)
    args = {**x, "h0": pool}
    want, mag = (state_ref.scan(**args, **kw, mag=m) for m in (False, True))
    K = 10 * want["step_decay"] + 6 + N + 2 * float(x["z"].float().abs().max()) + 60
    new = torch.full_like(pool, float("nan"))
    y = ss.state_scan_step(**row, state=pool, state_out=new, **kw)
    close(y, want["y"][0], mag["y"][0], K, ("step y", y.dtype))
    close(new, want["h"], mag["h"], K, ("step h", new.dtype))
    y2 = ss.state_scan_step(**row, state=pool, **kw)                   # in place
    assert torch.equal(y, y2) and torch.equal(pool, new)


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_step_index(itype):
    """A pool with idle rows, an index past the pool and a slot named twice: the live rows as
    without an index, NaN for the bad ones, and no other slot touched."""
    B, D, N, W, S = 6, 40, 16, 4, 9
    x, row, _ = step_case(B, D, N, 1, "f32", S, seed=1)
    big = torch.randn(S, 2, D, N, device=DEV)
    pool = big[:, 1]                                                    # one layer of a pool
    keep = big.clone()
    row["u"][2] = float("nan")                                          # an idle row's inputs
    index = torch.tensor([4, 0, -1, S, 4, 8], dtype=itype, device=DEV)
    live, slots = [0, 1, 5], [4, 0, 8]
    part = {k: v[live] if k in ("u", "delta", "z", "B", "C") else v for k, v in row.items()}
    ref = pool[slots].clone()
    want = ss.state_scan_step(**part, state=ref, softplus=True)
    y = ss.state_scan_step(**row, state=pool, softplus=True, index=index)
    assert torch.equal(y[live], want) and torch.equal(y[2], torch.zeros_like(y[2]))
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    keep[slots, 1] = ref
    assert torch.equal(big, keep)

    xs, w = torch.randn(B, D, device=DEV), torch.randn(D, W, device=DEV)
    cbig = torch.randn(S, 2, W - 1, D, device=DEV)
    cpool, keep = cbig[:, 0], cbig.clone()
    ref = cpool[slots].clone()
    want = ss.short_conv_step(xs[live], ref, w)
    y = ss.short_conv_step(xs, cpool, w, index=index)
    assert torch.equal(y[live], want) and not y[2].any() and torch.isnan(y[3:5]).all()
    keep[slots, 0] = ref
    assert torch.equal(cbig, keep)


def test_steps_equal_the_sequence():
    """Prompt, then token after token, against the whole sequence in one call."""
    x, _, _ = scan_case(24, 3, 40, 16, 2, "f32", seed=13)
    seqs = ("u", "delta", "z", "B", "C")
    y, h = ss.state_scan(**x, softplus=True, return_state=True)
    _, state = ss.state_scan(**{k: v[:16] if k in seqs else v for k, v in x.items()}, softplus=True,
                             return_state=True)
    args = {k: v for k, v in x.items() if k != "h0"}
    want, mag = (state_ref.scan(**x, softplus=True, mag=m) for m in (False, True))
    K = 24 * (10 * want["step_decay"] + 6) + 16 + 2 * float(x["z"].abs().max()) + 60
    for t in range(16, 24):
        row = {k: v[t] if k in seqs else v for k, v in args.items()}
        yt = ss.state_scan_step(**row, state=state, softplus=True)
        close(yt, want["y"][t], mag["y"][t], K, (f"token {t}", yt.dtype))
    close(state, want["h"], mag["h"], K, ("states", state.dtype))
    close(h, want["h"], mag["h"], K, ("states", h.dtype))
    w, b = torch.randn(40, 4, device=DEV), torch.randn(40, device=DEV)
    yc = ss.short_conv(x["u"], w, b, "silu")
    _, s = ss.short_conv(x["u"][:10], w, b, "silu", return_state=True)
    for t in range(10, 24):
        assert torch.equal(ss.short_conv_step(x["u"][t], s, w, b, "silu"), yc[t])


# ---------------------------------------------------------------------------------------
# convolution.  Units: W products and sums, bias 1, gate 10 + 2 |p|; the gradients a second time,
# with sums over T B terms.  |p| enters through the gate's argument only and is at most max |p|.
# ---------------------------------------------------------------------------------------
def check_conv(x, w, b, act, state, n, gy, gl, what):
    leaves = {k: v.detach().requires_grad_(True) for k, v in
              (("x", x), ("weight", w), ("bias", b), ("state", state)) if v is not None}
    y, last = ss.short_conv(leaves["x"], leaves["weight"], leaves.get("bias"), "silu" if act else None,
                            leaves.get("state"), n, return_state=True)
    got = dict(zip(leaves, torch.autograd.grad([y, last], list(leaves.values()), [gy, gl], allow_unused=True)))
    want, mag = (state_ref.conv(x, w, b, act, state, n, gy, gl, mag=m) for m in (False, True))
    T, B, _ = x.shape
    K = 4 * w.shape[1] + 2 * float(mag["y"].max()) + T * B + 40
    close(y, want["y"], mag["y"], K, (what + " y", y.dtype))
    assert torch.equal(last.double(), want["last"])
    for k, v in got.items():
        close(v, want["g" + k], mag["g" + k], K, (what + " grad " + k, v.dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,B,D,W,act", [
    (1, 1, 1, 1, False), (1, 2, 128, 4, True), (2, 3, 8, 4, True), (3, 2, 130, 4, False), (33, 2, 132, 4, True),
    (65, 3, 7, 3, True), (32, 2, 256, 2, True), (100, 2, 40, 5, False), (31, 2, 12, 6, True), (70, 1, 20, 7, True),
    (40, 2, 136, 8, True), (5, 300, 12, 4, True)])
def test_conv_against_64_bits(T, B, D, W, act, dtype):
    g = torch.Generator(device=DEV).manual_seed(T + W)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    dt = TYPES[dtype]
    x = r(T, B, 2 * D).to(dt)[..., D:]
    check_conv(x, r(D, W), r(D), act, r(B, W - 1, D).to(dt), None, r(T, B, D).to(dt), r(B, W - 1, D).to(dt), "conv")
    check_conv(x, r(D, W), None, act, None, None, r(T, B, D).to(dt), r(B, W - 1, D).to(dt), "conv bare")


@pytest.mark.parametrize("D", [40, 41])
@pytest.mark.parametrize("lengths", [[70, 1, 0, 33, 2], [0, 0, 0, 0, 0], [32, 64, 31, 65, 3]])
def test_conv_padded_batch_first(D, lengths):
    g = torch.Generator(device=DEV).manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    n = torch.tensor(lengths, device=DEV)
    x = r(5, 70, D).transpose(0, 1)
    x[torch.arange(70, device=DEV)[:, None] >= n[None]] = float("nan")
    check_conv(x, r(D, 4), r(D), True, r(5, 3, D), n, r(70, 5, D), r(5, 3, D), "padded")


# ---------------------------------------------------------------------------------------
# refusals, streams, graphs, the layer
# ---------------------------------------------------------------------------------------
def test_refusals():
    x, _, _ = scan_case(8, 2, 12, 16, 1, "bf16", seed=14)
    ok = lambda **k: ss.state_scan(**{**x, **k}, softplus=True)  # noqa: E731
    for bad in (dict(delta=x["delta"].float()), dict(z=x["z"][:4]), dict(A=x["A"][:4]), dict(B=x["B"][..., :8]),
                dict(B=x["B"][:, :, 0, 0]), dict(u=x["u"][0]), dict(u=x["u"].double()), dict(D=x["D"][:3]),
                dict(h0=x["h0"][:1]), dict(h0=x["h0"].cpu()), dict(D=x["D"].long()),
                dict(lengths=torch.ones(2, device=DEV)), dict(lengths=torch.ones(3, device=DEV, dtype=torch.int32)),
                dict(lengths=torch.ones(2, dtype=torch.int32)), dict(u=x["u"][:0]),
                dict(A=x["A"][:, :1].expand(12, 129).contiguous()),
                dict(B=x["B"].expand(8, 2, 5, 16), C=x["C"].expand(8, 2, 5, 16))):
        with pytest.raises(ValueError):
            ok(**bad)
    u, A = x["u"][0], x["A"]
    B, pool = x["B"][0], torch.zeros(2, 12, 16, device=DEV)
    step = lambda s=pool, **k: ss.state_scan_step(u, u, s, A, B, B, **k)  # noqa: E731
    for bad in (pool.half(), pool[:1], pool[:, :, :8], pool.transpose(1, 2).contiguous().transpose(1, 2),
                pool[:1].expand(2, 12, 16), pool.clone().requires_grad_(True)):
        with pytest.raises(ValueError):
            step(bad)
    with pytest.raises(ValueError):
        step(state_out=torch.zeros(3, 12, 16, device=DEV))
    with pytest.raises(ValueError):
        step(index=torch.zeros(3, device=DEV, dtype=torch.int32))
    w = torch.zeros(12, 4, device=DEV)
    for k in (dict(weight=w[:3]), dict(weight=torch.zeros(12, 9, device=DEV)), dict(weight=w, activation="relu"),
              dict(weight=w, state=torch.zeros(2, 3, 12, device=DEV)), dict(weight=w, bias=w)):
        with pytest.raises(ValueError):
            ss.short_conv(x["u"], **k)
    with pytest.raises(ValueError):
        ss.short_conv_step(u, torch.zeros(2, 3, 12, device=DEV), w)     # state of another type


def test_saved_input_changed_in_place_is_noticed():
    x, _, (gy, _) = scan_case(8, 2, 12, 16, 1, "f32", seed=15)
    A = x["A"].requires_grad_(True)
    y = ss.state_scan(**{**x, "A": A}, softplus=True)
    x["u"].add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, A, gy)


def test_other_stream():
    x, n, (gy, gh) = scan_case(300, 4, 256, 16, 1, "f32", seed=16)
    leaves = {k: v.requires_grad_(True) for k, v in x.items()}

    def run():
        y, h = ss.state_scan(**leaves, softplus=True, return_state=True)
        return [y, h, *torch.autograd.grad([y, h], list(leaves.values()), [gy, gh])]
    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replay():
    """Captured training passes (whole sequences, parts side by side, parts one after another) and a
    captured step, replayed in turn on new inputs.  (An eager graph of the same leaves must not live
    while a backward is captured: torch's own gradient nodes of the leaves would wait for the stream
    of that graph, and the capture fails.)"""
    graphs = []
    L = _capi.lib()
    for seed, (T, B, D) in enumerate(((40, 2, 96), (17, 2, 64), (700, 1, 64), (300, 480, 8))):
        x, _, (gy, _) = scan_case(T, B, D, 16, 1, "bf16", seed=20 + seed)
        leaves = {k: v.requires_grad_(True) for k, v in x.items()}
        w = torch.randn(D, 4, device=DEV, requires_grad=True)

        def run(leaves=leaves, w=w, gy=gy):
            u = ss.short_conv(leaves["u"], w, None, "silu")
            y = ss.state_scan(**{**leaves, "u": u}, softplus=True)
            return [y, *torch.autograd.grad(y, [*leaves.values(), w], gy)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with profiling.NativeCallTimer() as timer, torch.cuda.graph(g):
            out = run()
        # convolution 1 + 2, the scan as its plan says
        scan = 1 + (L.dfsnn_state_scan_forward_workspace_size(T, B, D, 16, 1) > 0) \
            + L.dfsnn_state_scan_backward_launches(T, B, D, 16, 1)
        assert timer.captured_launches() == 3 + scan
        graphs.append((g, out, run, leaves))
    x, row, pool = step_case(4, 64, 16, 1, "bf16", 4, seed=30)
    new, index = torch.empty_like(pool), torch.tensor([3, -1, 0, 2], dtype=torch.int32, device=DEV)
    step = lambda: ss.state_scan_step(**row, state=pool, state_out=new, softplus=True, index=index)  # noqa: E731
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ys = step()
    for trial in range(2):
        for _, _, _, leaves in graphs:
            with torch.no_grad():
                leaves["u"].normal_()
                leaves["delta"].normal_()
        row["u"].normal_()
        index.copy_(torch.roll(index, 1))
        for graph, *_ in graphs:
            graph.replay()
        g.replay()
        for _, out, run, _ in graphs:
            assert all(torch.equal(a, b) for a, b in zip([o.clone() for o in out], run()))
        a, b = ys.clone(), new.clone()
        assert torch.equal(a, step()) and torch.equal(b, new)


def layer_64(layer, x, lengths=None):
    """StateSpaceLayer.forward in 64 bits with torch operations and their differentiation."""
    p = {k: v.detach().double().requires_grad_(True) for k, v in layer.named_parameters()}
    lin = torch.nn.functional.linear
    T, Bn, _ = x.shape
    xs, z = lin(x, p["in_proj.weight"]).chunk(2, -1)
    W = p["conv_weight"].shape[1]
    e = torch.cat([xs.new_zeros(W - 1, Bn, xs.shape[-1]), xs])
    xs = torch.nn.functional.silu(p["conv_bias"] + sum(p["conv_weight"][:, j] * e[j:j + T] for j in range(W)))
    G, N = layer.groups, layer.d_state
    dt, B, C = torch.split(lin(xs, p["x_proj.weight"]), [layer.rank, G * N, G * N], -1)
    rep = lambda v: v.unflatten(-1, (G, N)).repeat_interleave(layer.d_inner // G, 2)  # noqa: E731
    dt = torch.nn.functional.softplus(lin(dt, p["dt_proj.weight"]) + p["delta_bias"])
    a = torch.exp(dt[..., None] * -torch.exp(p["A_log"]))
    h, ys = xs.new_zeros(Bn, layer.d_inner, N), []
    for t in range(T):
        h = a[t] * h + (dt[t] * xs[t])[..., None] * rep(B)[t]
        ys.append((rep(C)[t] * h).sum(-1) + p["D"] * xs[t])
    return lin(torch.stack(ys) * torch.nn.functional.silu(z), p["out_proj.weight"]), p


def test_layer_into_neuron():
    """Projections, convolution, scan and the package's spiking neuron as one network: outputs and
    every parameter gradient against 64 bits; then the same sequence as prompt and tokens."""
    from dfsnn_b200.neuron import LIFNeuronFDE
    torch.manual_seed(0)
    T, Bn = 16, 3
    layer = ss.StateSpaceLayer(48, groups=2).to(DEV)
    x = torch.randn(T, Bn, 48, device=DEV)
    y = layer(x)
    gy = torch.randn_like(y)
    got = torch.autograd.grad(y, list(layer.parameters()), gy)
    y64, p = layer_64(layer, x.double())
    want = torch.autograd.grad(y64, list(p.values()), gy.double())
    # every path has a few hundred roundings (T steps of the scan, sums over 96 channels, T B rows)
    # and four projections with sums of at most 96 terms; norm against norm
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y, y64) < 2000 * 2.0 ** -24
    for (k, _), a, b in zip(layer.named_parameters(), got, want):
        assert rel(a, b) < 20000 * 2.0 ** -24, k
    neuron = LIFNeuronFDE(tau=2.0, threshold=0.05, surrogate_function="arctan", method="gl", beta=0.5, T=T,
                          batchsize=Bn, step_mode="m", backend="cupy").to(DEV)
    s = neuron(layer(x))
    assert s.shape == y.shape and bool(((s == 0) | (s == 1)).all())
    g = torch.autograd.grad(s.sum(), layer.A_log)[0]
    assert torch.isfinite(g).all() and bool(g.abs().sum() > 0)
    with torch.no_grad():
        _, state = layer(x[:10], return_state=True)
        for t in range(10, T):
            assert rel(layer.step(x[t], state), y64[t].detach()) < 2000 * 2.0 ** -24
        layer.step_mode = "s"
        for t in range(T):
            assert rel(layer(x[t]), y64[t].detach()) < 2000 * 2.0 ** -24
        layer.reset()
        assert rel(layer(x[0]), y64[0].detach()) < 2000 * 2.0 ** -24


def test_layer_serves_from_a_pool():
    """Padded prompts, their states into a pool, then tokens of some of them with an idle row in
    between: each sequence as if it were alone, and the pool's other slots untouched."""
    torch.manual_seed(1)
    layer = ss.StateSpaceLayer(40, d_state=12, taps=3, groups=4).to(DEV)
    T, lengths, slots = 12, [9, 3, 6], [5, 0, 2]
    x = torch.randn(T, 3, 40, device=DEV)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())  # noqa: E731
    with torch.no_grad():
        alone = [layer(x[:, b:b + 1])[:, 0] for b in range(3)]
        y, (conv, scan) = layer(x, lengths=n, return_state=True)
        for b, k in enumerate(lengths):                 # the same sums in another grid: fp32 roundings
            assert rel(y[:k, b], alone[b][:k]) < 2000 * 2.0 ** -24
        pool = layer.initial_state(7)
        for p, s in zip(pool, (conv, scan)):
            p[:] = float("nan")
            p[slots] = s
        at = list(lengths)
        for order in ([2, None, 0, 1], [None, 1, 2], [0]):
            rows = torch.stack([torch.full((40,), float("nan"), device=DEV) if b is None else x[at[b], b] for b in order])
            index = torch.tensor([-1 if b is None else slots[b] for b in order], device=DEV)
            out = layer.step(rows, pool, index)
            for r, b in enumerate(order):
                if b is not None:
                    assert rel(out[r], alone[b][at[b]]) < 2000 * 2.0 ** -24
                    at[b] += 1
        assert all(torch.isnan(p[[1, 3, 4, 6]]).all() for p in pool)
