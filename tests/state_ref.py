"""The state-space operators in 64 bits, from their formulas, one step after another.

Every function takes mag=True to return, for each output, the sum of the absolute values of
the terms that it is made of.  An fp32 evaluation that rounds each intermediate result is off by
at most K * 2^-24 times that sum, K being the number of roundings on the longest path."""
import torch


def silu(x):
    return x * torch.sigmoid(x)


def dsilu(x):
    s = torch.sigmoid(x)
    return s + x * s * (1 - s)


def dsilu_terms(x):
    """silu'(x) = s + x s (1 - s) is a sum of two terms of opposite sign where x < 0 (it is zero
    at x = -1.28, where each is 0.22): its rounding errors are relative to |s| + |x s (1 - s)|."""
    s = torch.sigmoid(x)
    return s + x.abs() * s * (1 - s)


def _d(x):
    return None if x is None else x.detach().double()


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, h0=None, lengths=None,
         gy=None, gh=None, mag=False):
    """{'y', 'h', 'step_decay' (largest |d A|)} and, given gy, the gradients {'gu', ...}."""
    u, delta, A, B, C, D, z, bias, h0, gy, gh = map(_d, (u, delta, A, B, C, D, z, delta_bias, h0, gy, gh))
    f = torch.abs if mag else (lambda x: x)
    T, Bn, Dn = u.shape
    G, N = B.shape[2:]
    grp = torch.arange(Dn, device=u.device) // (Dn // G)
    zero = torch.zeros((), dtype=torch.float64, device=u.device)
    n = torch.full((Bn,), T, device=u.device) if lengths is None else lengths.long().clamp(0, T)
    D0 = torch.zeros(Dn, dtype=torch.float64, device=u.device) if D is None else D
    raw = delta if bias is None else delta + bias
    live = (torch.arange(T, device=u.device)[:, None] < n[None])[..., None]
    raw = torch.where(live, raw, zero)
    d = torch.where(live, torch.logaddexp(raw, zero) if softplus else raw, zero)
    u = torch.where(live, u, zero)
    Bc, Cc = (torch.where(live, x[:, :, grp].flatten(2), zero).unflatten(2, (Dn, N)) for x in (B, C))
    zz = None if z is None else torch.where(live, z, zero)
    gate = 1.0 if z is None else f(silu(zz))
    h = torch.zeros(Bn, Dn, N, dtype=torch.float64, device=u.device) if h0 is None else f(h0)
    a = torch.exp(d[..., None] * A)
    hs, o = [h], []
    for t in range(T):
        h = a[t] * h + f((d[t] * u[t])[..., None] * Bc[t])
        hs.append(h)
        o.append((f(Cc[t]) * h).sum(-1) + f(D0 * u[t]))
    o = torch.stack(o)
    r = {"y": torch.where(live, o * gate, zero), "h": h, "step_decay": (d[..., None] * A).abs().max().item()}
    if gy is None:
        return r
    gy = torch.where(live, f(gy), zero)
    if z is not None:
        r["gz"] = gy * o * (dsilu_terms(zz) if mag else dsilu(zz)) * live
    g = gy * gate
    lam = torch.zeros_like(h) if gh is None else f(gh)
    out = {k: [] for k in ("gu", "gdelta", "gB", "gC")}
    gA = torch.zeros_like(A)
    for t in range(T - 1, -1, -1):
        out["gC"].append((g[t][..., None] * hs[t + 1]).unflatten(1, (G, Dn // G)).sum(2))
        lam = lam + g[t][..., None] * f(Cc[t])
        q = lam * a[t] * hs[t] * live[t][..., None]
        lb = (lam * f(Bc[t])).sum(-1) * live[t]
        out["gB"].append((lam * f(d[t] * u[t])[..., None]).unflatten(1, (G, Dn // G)).sum(2))
        out["gu"].append(f(d[t]) * lb + f(D0) * g[t])
        gd = f(u[t]) * lb + (q * f(A)).sum(-1)
        out["gdelta"].append(gd * torch.sigmoid(raw[t]) if softplus else gd)
        gA += (q * f(d[t])[..., None]).sum(0)
        lam = a[t] * lam
    for k, v in out.items():
        r[k] = torch.stack(v[::-1])
    r["gA"], r["gh0"] = gA, lam
    r["gD"] = (g * f(u)).sum((0, 1))
    r["gdelta_bias"] = r["gdelta"].sum((0, 1))
    return r


def conv(x, weight, bias=None, silu_=False, state=None, lengths=None, gy=None, glast=None, mag=False):
    x, weight, bias, state, gy, glast = map(_d, (x, weight, bias, state, gy, glast))
    f = torch.abs if mag else (lambda v: v)
    T, Bn, Dn = x.shape
    W = weight.shape[1]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    n = torch.full((Bn,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    live = (torch.arange(T, device=x.device)[:, None] < n[None])[..., None]
    head = torch.zeros(W - 1, Bn, Dn, dtype=torch.float64, device=x.device) if state is None \
        else state.transpose(0, 1)
    ext = torch.cat([head, torch.where(live, x, zero)])
    true = sum(weight[:, j] * ext[j:j + T] for j in range(W)) + (0 if bias is None else bias)
    p = sum(f(weight[:, j] * ext[j:j + T]) for j in range(W)) + (0 if bias is None else f(bias))
    # silu(p) changes by at most 1.1 |change of p|
    y = (1.1 * p if mag else silu(true)) if silu_ else p
    rows = n[:, None] + torch.arange(W - 1, device=x.device)
    cols = torch.arange(Bn, device=x.device)[:, None]
    r = {"y": torch.where(live, y, zero), "last": ext[rows, cols]}
    if gy is None:
        return r
    gp = torch.where(live, f(gy), zero)
    if silu_:
        # silu'(p) changes by at most 0.5 |change of p|
        gp = gp * ((dsilu_terms(true) + 0.5 * p) if mag else dsilu(true))
    gx = torch.zeros_like(ext)
    for j in range(W):
        gx[j:j + T] += f(weight[:, j]) * gp
    if glast is not None:
        gx[rows, cols] += f(glast)
    r["gx"] = torch.where(live, gx[W - 1:], zero)
    r["gstate"] = gx[:W - 1].transpose(0, 1)
    r["gweight"] = torch.stack([(gp * f(ext[j:j + T])).sum((0, 1)) for j in range(W)], 1)
    r["gbias"] = gp.sum((0, 1))
    return r
