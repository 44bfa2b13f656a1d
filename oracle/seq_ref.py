"""Float64 definitions of the causal sequence operators and of their gradients, frame by frame (tests only).

Every function takes `mag`: the sum of the magnitudes of the terms that make up each output (all inputs by absolute value, every
difference a sum), the yardstick of an f32 evaluation's rounding error.
"""
import torch


def _d(t):
    return None if t is None else t.detach().double().cpu()


def sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def silu(x):
    return x * sigmoid(x)


def silu_grad(x):
    return sigmoid(x) * (1 + x * (1 - sigmoid(x)))


def _ends(lengths, B, T):
    return [T] * B if lengths is None else [min(max(int(v), 0), T) for v in lengths.tolist()]


# ------------------------------------------------------------------------------------------------ causal convolution
def conv(x, w, b=None, act="silu", state=None, lengths=None, dy=None, dstate_out=None, mag=False):
    """-> dict(y, state[, dx, dw, dbias, dstate])."""
    x, b, state, dy, dstate_out = map(_d, (x, b, state, dy, dstate_out))
    w = _d(w).reshape(w.shape[0], w.shape[-1])
    B, T, C = x.shape
    K = w.shape[1]
    ab = torch.abs if mag else lambda t: t
    out = {k: torch.zeros(s, dtype=torch.float64) for k, s in
           dict(y=(B, T, C), state=(B, K - 1, C), dx=(B, T, C), dw=(C, K), dbias=(C,), dstate=(B, K - 1, C)).items()}
    for i, n in enumerate(_ends(lengths, B, T)):
        e = torch.zeros(K - 1 + n, C, dtype=torch.float64)
        if state is not None:
            e[:K - 1] = state[i]
        e[K - 1:] = x[i, :n]
        out["state"][i] = e[n:n + K - 1]
        de = torch.zeros_like(e)
        if dstate_out is not None:
            de[n:n + K - 1] += ab(dstate_out[i])
        for t in range(n):
            true = (w * e[t:t + K].t()).sum(-1) + (b if b is not None else 0)
            pre = true if not mag else (w * e[t:t + K].t()).abs().sum(-1) + (b.abs() if b is not None else 0)
            out["y"][i, t] = pre if act is None else (silu(true) if not mag else pre)
            if dy is not None:
                g = ab(dy[i, t]) * (1.0 if act is None else silu_grad(true) if not mag else 1.1 + pre)     # |silu''| < 1: an error of pre moves silu' by less
                out["dbias"] += g
                out["dw"] += g[:, None] * ab(e[t:t + K].t())
                de[t:t + K] += g * ab(w.t())
        out["dx"][i, :n], out["dstate"][i] = de[K - 1:], de[:K - 1]
    return out


# ---------------------------------------------------------------------------------------------- selective scan
def scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None, dy=None, dstate_out=None, mag=False):
    """-> dict(y, state[, du, ddt, dA, dB, dC, dD, dz, ddt_bias, dstate]); B and C [batch, frames, groups, states]."""
    u, dt, A, B, C, D, z, dt_bias, state, dy, dstate_out = map(_d, (u, dt, A, B, C, D, z, dt_bias, state, dy, dstate_out))
    nb, T, Dm = u.shape
    N, G = A.shape[1], B.shape[2]
    ab = torch.abs if mag else lambda t: t
    share = torch.arange(Dm) // (Dm // G)
    raw = dt + (dt_bias if dt_bias is not None else 0)
    s = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    skip = ab(D) if D is not None else torch.zeros(Dm, dtype=torch.float64)
    u, B, C = ab(u), ab(B), ab(C)
    gate = torch.ones_like(u) if z is None else (silu(z) if not mag else z.abs())
    out = {k: torch.zeros(shape, dtype=torch.float64) for k, shape in
           dict(y=u.shape, state=(nb, Dm, N), du=u.shape, ddt=u.shape, dA=A.shape, dB=B.shape, dC=C.shape, dD=(Dm,), dz=u.shape, ddt_bias=(Dm,),
                dstate=(nb, Dm, N)).items()}
    for i, n in enumerate(_ends(lengths, nb, T)):
        h = [ab(state[i]) if state is not None else torch.zeros(Dm, N, dtype=torch.float64)]
        y0 = []
        sa = ab(s[i])
        for t in range(n):
            h.append(torch.exp(s[i, t][:, None] * A) * h[-1] + (sa[t] * u[i, t])[:, None] * B[i, t][share])
            y0.append((C[i, t][share] * h[-1]).sum(-1) + skip * u[i, t])
            out["y"][i, t] = y0[-1] * gate[i, t]
        out["state"][i] = h[-1]
        if dy is None and dstate_out is None:
            continue
        c = ab(dstate_out[i]) if dstate_out is not None else torch.zeros(Dm, N, dtype=torch.float64)
        for t in reversed(range(n)):
            up = ab(dy[i, t]) if dy is not None else torch.zeros(Dm, dtype=torch.float64)
            g = up * gate[i, t]
            q = C[i, t][share] * g[:, None] + c
            c = torch.exp(s[i, t][:, None] * A) * q
            k = c * h[t]
            qb = (q * B[i, t][share]).sum(-1)
            out["dC"][i, t] = (g[:, None] * h[t + 1]).reshape(G, Dm // G, N).sum(1)
            out["dB"][i, t] = (q * (sa[t] * u[i, t])[:, None]).reshape(G, Dm // G, N).sum(1)
            out["du"][i, t] = sa[t] * qb + skip * g
            ds = u[i, t] * qb + (ab(A) * k).sum(-1)
            ds = ds * sigmoid(raw[i, t]) if softplus else ds
            out["ddt"][i, t] = ds
            out["ddt_bias"] += ds
            out["dA"] += k * sa[t][:, None]
            out["dD"] += g * u[i, t]
            if z is not None:
                out["dz"][i, t] = up * y0[t] * (silu_grad(z[i, t]) if not mag else 1.1 + z[i, t].abs())
        out["dstate"][i] = c
    return out


# ---------------------------------------------------------------------------------------------- gated residual norms
def _norm(v, w, b, kind, eps, mag, true=None):
    """(normalised, scaled and shifted, 1 / std) of v; `true`: the signed values behind magnitudes."""
    t = v if true is None else true
    mean = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[..., :1])
    rstd = 1 / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + eps)
    h = (t - mean) * rstd if not mag else (v + v.mean(-1, keepdim=True)) * rstd
    y = h * (w.abs() if mag else w)
    return h, y if b is None else y + (b.abs() if mag else b), rstd


def _norm_back(v, h, rstd, kind, mag):
    m = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    q = h * (v * h).mean(-1, keepdim=True)
    return rstd * (v + m + q if mag else v - m - q)


def residual_norm(x, o, w=None, b=None, pw=None, pb=None, gate=None, scale=None, eps=1e-6, kind="layer", dr=None, dn=None, mag=False):
    """-> dict(r, n[, dx, do, dgate, dw, db, dpw, dpb, dscale])."""
    x, o, w, b, pw, pb, gate, scale, dr, dn = map(_d, (x, o, w, b, pw, pb, gate, scale, dr, dn))
    ab = torch.abs if mag else lambda t: t
    one = torch.ones((), dtype=torch.float64)
    zero = torch.zeros_like(x)
    tp = o if pw is None else _norm(o, pw, pb, kind, eps, False)[1]
    tr = x + (scale if scale is not None else one) * (gate if gate is not None else one) * tp
    oh, p, orstd = (ab(o), ab(o), None) if pw is None else _norm(ab(o), pw, pb, kind, eps, mag, o)
    g, s = (ab(gate) if gate is not None else one), (ab(scale) if scale is not None else one)
    r = ab(x) + s * g * p
    out = {"r": r}
    dR = ab(dr) if dr is not None else zero
    if w is not None:
        h, n, rstd = _norm(r, w, b, kind, eps, mag, tr)
        out["n"] = n
        if dn is not None:
            out["dw"], out["db"] = (ab(dn) * h).sum((0, 1)), ab(dn).sum((0, 1))
            dR = dR + _norm_back(ab(dn) * ab(w), h, rstd, kind, mag)
    out["dx"] = dR
    dp = dR * s * g
    dg = dR * s * p
    if gate is not None:
        out["dgate"] = dg if gate.shape[1] == x.shape[1] else dg.sum(1, keepdim=True)
    out["dscale"] = (dR * g * p).sum((0, 1))
    if pw is not None:
        out["dpw"], out["dpb"] = (dp * oh).sum((0, 1)), dp.sum((0, 1))
        out["do"] = _norm_back(dp * ab(pw), oh, orstd, kind, mag)
    else:
        out["do"] = dp
    return out
