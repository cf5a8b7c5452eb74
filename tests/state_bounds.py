"""Running error bounds of the selective scan: how far fp32 kernels may be from the formulas.

scan() walks the formulas in 64 bits together with the sum of the absolute values of the terms of
each quantity (H for h, L for l = grad h, ...) and with a bound of its error, in units of
U = 2^-24, the largest relative error of one fp32 rounding.  So a state's error fades with the state
that carries it, and each output has its own bound.  Relative errors, in units:

  d = softplus(x), x = delta + bias    x itself 1, which moves d by at most max(|x|, 1) of it; e^-|x| has
      its argument's two roundings, 2 |x|, and the approximation's 4; the quotient 4, the polynomial and
      the sum 4:  Ed = 3 |x| + 14.  Without softplus 1
  decay 2^(d A log2 e)    its argument d's error and 3 more, times |d A|; the power itself 4 by the
      hardware's approximation, or 2 by the polynomial that is taken near 1 (all of a channel's |d A log2 e|
      < 1/16):  Ea = |d A| (Ed + 3) + 4 or 2.  Parts of a sequence side by side are joined by the decay
      over a part, whose exponent is a sum of P steps: P |d A| more
  h = a h + d u B         Ed + 2 for the second term, 1 for the sum
  sigmoid(x)              its argument 2 |x|, the power 4, sum 1, quotient 2:  2 |x| + 7
  silu(z), silu'(z)       2 |z| + 9; a sum of two terms, 4 |z| + 20 of their absolute values
  sums of n terms         n + 1, the terms' own products included
  grad A, D, delta_bias   16 steps of a tile in fp32, the rest in 64 bits and rounded twice: 20

What the products of errors add is less than a hundredth."""
import torch

U = 2.0 ** -24


def _d(x):
    return None if x is None else x.detach().double()


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, h0=None, lengths=None,
         gy=None, gh=None, part=0):
    """({name: value}, {name: bound}) of y, h and, given gy, the gradients gu, gdelta, ...  `part`: steps of
    the parts that a sequence is walked in side by side (0: none)."""
    u, delta, A, B, C, D, z, bias, h0, gy, gh = map(_d, (u, delta, A, B, C, D, z, delta_bias, h0, gy, gh))
    T, Bn, Dn = u.shape
    G, N = B.shape[2:]
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device=u.device)  # noqa: E731
    n = torch.full((Bn,), T, device=u.device) if lengths is None else lengths.long().clamp(0, T)
    live = (torch.arange(T, device=u.device)[:, None] < n)[..., None]
    mask = lambda x: torch.where(live, x, new(1))  # noqa: E731
    rep = lambda x: mask(x.flatten(2)).unflatten(2, (G, N)).repeat_interleave(Dn // G, 2)  # noqa: E731
    x = mask(delta if bias is None else delta + bias)
    d = mask(torch.logaddexp(x, new(1)) if softplus else x)
    Ed = 3 * x.abs() + 14 if softplus else torch.ones_like(x)
    u, Bc, Cc = mask(u), rep(B), rep(C)
    skip = new(Dn) if D is None else D
    m = (d[..., None] * A).abs()
    near = (m.amax((0, 3)) * 1.4427 < 0.0624)[..., None]              # a sequence's channel, all its states
    Ea = m * (Ed[..., None] + 3 + part) + torch.where(near, 2.0, 4.0)
    a = torch.exp(d[..., None] * A)
    if z is not None:
        z = mask(z)
        s = torch.sigmoid(z)
        gate, Eg = z * s, 2 * z.abs() + 9
        slope, slope_abs, Es = s + z * s * (1 - s), s + z.abs() * s * (1 - s), 4 * z.abs() + 20
    else:
        gate, Eg = torch.ones_like(u), torch.zeros_like(u)

    h = new(Bn, Dn, N) if h0 is None else h0
    H, E = h.abs(), torch.zeros_like(h)
    hs, Hs, Es_h, o, O, Eo = [h], [H], [E], [], [], []
    for t in range(T):
        term = (d[t] * u[t])[..., None] * Bc[t]
        E = a[t] * E + a[t] * H * Ea[t] + term.abs() * (Ed[t][..., None] + 2)
        h, H = a[t] * h + term, a[t] * H + term.abs()
        E = torch.where(live[t][..., None], E + H, E)
        c = Cc[t].abs()
        o.append((Cc[t] * h).sum(-1) + skip * u[t])
        O.append((c * H).sum(-1) + (skip * u[t]).abs())
        Eo.append((c * E).sum(-1) + (N + 3) * O[-1])
        hs.append(h), Hs.append(H), Es_h.append(E)
    o, O, Eo = map(torch.stack, (o, O, Eo))
    out = {"y": mask(o * gate), "h": h}
    err = {"y": gate.abs() * (Eo + O * (Eg + 2)), "h": E}
    if gy is not None:
        gy = mask(gy)
        if z is not None:
            out["gz"] = gy * o * slope
            err["gz"] = gy.abs() * slope_abs * (Eo + O * (Es + 3))
        g, Eg = gy * gate, (Eg + 1) * (gy * gate).abs()
        names = ("gu", "gdelta", "gB", "gC")
        out.update({k: [] for k in names}), err.update({k: [] for k in names})
        gA, eA = torch.zeros_like(A), torch.zeros_like(A)
        lam = new(Bn, Dn, N) if gh is None else gh                     # a_(t+1) l_(t+1)
        L, EL = lam.abs(), torch.zeros_like(lam)
        grp = lambda v: v.unflatten(1, (G, Dn // G)).sum(2)  # noqa: E731
        w = Dn // G + 1
        for t in range(T - 1, -1, -1):
            on = live[t][..., None]
            h, H, E, hp, Hp, Ep = hs[t + 1], Hs[t + 1], Es_h[t + 1], hs[t], Hs[t], Es_h[t]
            gt, Gt, eg, dt, du = (v[..., None] for v in (g[t], g[t].abs(), Eg[t], d[t], d[t] * u[t]))
            ed, Du = Ed[t][..., None], du.abs()
            out["gC"].append(grp(gt * h))
            err["gC"].append(grp(Gt * E + eg * H + (w + 1) * Gt * H))
            c, b = Cc[t].abs(), Bc[t].abs()
            EL = torch.where(on, EL + c * eg + 2 * c * Gt + L, EL)
            lam, L = lam + Cc[t] * gt, L + c * Gt
            out["gB"].append(grp(lam * du))
            err["gB"].append(grp(Du * EL + L * Du * (ed + 1 + w)))
            lb, LB, Elb = (lam * Bc[t]).sum(-1), (L * b).sum(-1), (b * EL + (N + 1) * b * L).sum(-1)
            dt1, u1 = d[t].abs(), u[t].abs()
            out["gu"].append(d[t] * lb + skip * g[t])
            err["gu"].append(dt1 * Elb + dt1 * LB * (Ed[t] + 2) + skip.abs() * (Eg[t] + 3 * g[t].abs()))
            q, Q = lam * a[t] * hp * on, L * a[t] * Hp * on
            Eq = a[t] * (Hp * EL + L * Ep) * on + Q * (Ea[t] + 2)
            gd = u[t] * lb + (q * A).sum(-1)
            GD = u1 * LB + (Q * A.abs()).sum(-1)
            e = u1 * (Elb + 2 * LB) + (A.abs() * (Eq + (N + 6) * Q)).sum(-1) + GD
            if softplus:
                sg = torch.sigmoid(x[t])
                gd, e, GD = gd * sg, sg * (e + GD * (3 * x[t].abs() + 9)), GD * sg
            gd, e = gd * live[t], e * live[t]
            out["gdelta"].append(gd), err["gdelta"].append(e)
            gA += (q * dt).sum(0)
            eA += (dt.abs() * (Eq + Q * (ed + 21))).sum(0)
            EL = torch.where(on, a[t] * (EL + L * (Ea[t] + 1)), EL)
            lam, L = a[t] * lam, a[t] * L
        for k in names:
            out[k], err[k] = (torch.stack(v[k][::-1]) for v in (out, err))
        out["gA"], err["gA"], out["gh0"], err["gh0"] = gA, eA, lam, EL
        out["gD"], err["gD"] = (g * u).sum((0, 1)), ((Eg + 21 * g.abs()) * u.abs()).sum((0, 1))
        out["gdelta_bias"] = out["gdelta"].sum((0, 1))
        err["gdelta_bias"] = (err["gdelta"] + 20 * out["gdelta"].abs()).sum((0, 1))
        for k in ("gB", "gC"):
            out[k], err[k] = (v[k] * live[..., None] for v in (out, err))
        for k in ("gu", "gdelta"):
            out[k], err[k] = out[k] * live, err[k] * live
    return out, {k: 1.01 * U * v for k, v in err.items()}


def conv(x, weight, bias=None, silu_=False, state=None, lengths=None, gy=None, glast=None):
    """The same for the short convolution: y, last (exact) and, given gy, gx, gweight, gbias, gstate.
    p has taps + 1 roundings; silu moves by at most 1.1 of what p does, silu' by at most 0.5; sums over
    steps and sequences are taken as one after another."""
    x, weight, bias, state, gy, glast = map(_d, (x, weight, bias, state, gy, glast))
    T, Bn, Dn = x.shape
    W = weight.shape[1]
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)  # noqa: E731
    n = torch.full((Bn,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    live = (torch.arange(T, device=x.device)[:, None] < n)[..., None]
    ext = torch.cat([new(W - 1, Bn, Dn) if state is None else state.transpose(0, 1), torch.where(live, x, new(1))])
    b = new(Dn) if bias is None else bias
    p = b + sum(weight[:, j] * ext[j:j + T] for j in range(W))
    ep = (W + 1) * (b.abs() + sum((weight[:, j] * ext[j:j + T]).abs() for j in range(W)))
    s = torch.sigmoid(p)
    y, ey = (p * s, 1.1 * ep + (p * s).abs() * (2 * p.abs() + 10)) if silu_ else (p, ep)
    rows = n[:, None] + torch.arange(W - 1, device=x.device)
    cols = torch.arange(Bn, device=x.device)[:, None]
    out, err = {"y": y * live, "last": ext[rows, cols]}, {"y": ey * live, "last": new(Bn, W - 1, Dn)}
    if gy is not None:
        gp = torch.where(live, gy, new(1))
        ap, eg = gp.abs(), torch.zeros_like(gp)
        if silu_:
            size = s + p.abs() * s * (1 - s)
            eg = ap * (0.5 * ep + size * (4 * p.abs() + 21))
            gp, ap = gp * (s + p * s * (1 - s)), ap * size
        gx, ex = torch.zeros_like(ext), torch.zeros_like(ext)
        for j in range(W):
            gx[j:j + T] += weight[:, j] * gp
            ex[j:j + T] += weight[:, j].abs() * (eg + (W + 1) * ap)
        if glast is not None:
            ex[rows, cols] += gx[rows, cols].abs() + glast.abs()
            gx[rows, cols] += glast
        out["gx"], err["gx"] = (v[W - 1:] * live for v in (gx, ex))
        out["gstate"], err["gstate"] = (v[:W - 1].transpose(0, 1) for v in (gx, ex))
        terms = T * Bn + 1
        out["gweight"] = torch.stack([(gp * ext[j:j + T]).sum((0, 1)) for j in range(W)], 1)
        err["gweight"] = torch.stack([((eg + terms * ap) * ext[j:j + T].abs()).sum((0, 1)) for j in range(W)], 1)
        out["gbias"], err["gbias"] = gp.sum((0, 1)), (eg + terms * ap).sum((0, 1))
    return out, {k: 1.01 * U * v for k, v in err.items()}


def check(got, want, bound, what):
    """A 16-bit output is rounded once more (a subnormal fp16 by half of 2^-24)."""
    got, dtype = got.detach().double(), got.dtype
    tol = bound + 1e-35                                   # fp32 below its normal range
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + 2.0 ** -25
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], tol.expand_as(got)[bad][:3])
    return float((off / tol).max()) if off.numel() else 0.0
