"""Measured cases of the causal sequence operators: short causal convolution, selective state space scan, gated residual norms.

`run` is one pass of one operator over what `prepare` made: the plain torch form (own = False) or the framework's call (own = True).
Sizes are those of the framework's speech encoders: 768 and 1024 channels (1536 and 2048 inside a block), 624, 781 and 999 frames per
utterance (200 000, 250 000 and 320 000 samples at 16 kHz), batches of 8 and 16, and single frames for streaming.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one stream, one frame: the latency of the convolution's step
        dict(name="conv step 1x1536", op="conv", mode="step", dtype="bf16", batch=1, frames=1, channels=1536, taps=4, ragged=False),
        # fine-tuned model on a padded batch of 16 x 200 000 samples
        dict(name="conv prompt ragged f32", op="conv", mode="prompt", dtype="f32", batch=16, frames=624, channels=1537, taps=3, ragged=True),
        # one training step of a base-sized block, 8 x 250 000 samples
        dict(name="conv train 8x781x1536", op="conv", mode="train", dtype="bf16", batch=8, frames=781, channels=1536, taps=4, ragged=False),
        # 32 streams, one frame each
        dict(name="scan step 32x1536", op="scan", mode="step", dtype="bf16", batch=32, frames=1, channels=1536, states=16, groups=1, gated=True, ragged=False),
        # one recording of about 16 minutes, continued from a state
        dict(name="scan prompt 1x48001", op="scan", mode="prompt", dtype="bf16", batch=1, frames=48001, channels=1536, states=16, groups=1, gated=True, ragged=False),
        # a padded batch of 16 x 200 000 samples in f32 (the framework's parity mode)
        dict(name="scan prompt ragged f32", op="scan", mode="prompt", dtype="f32", batch=16, frames=624, channels=1536, states=16, groups=1, gated=False, ragged=True),
        # one training step of a base-sized block
        dict(name="scan train 8x781x1536", op="scan", mode="train", dtype="bf16", batch=8, frames=781, channels=1536, states=16, groups=1, gated=True, ragged=False),
        # odd sizes, two groups, a padded batch, f32
        dict(name="scan train odd f32", op="scan", mode="train", dtype="f32", batch=3, frames=333, channels=1002, states=11, groups=2, gated=True, ragged=True),
        # one training step of a large-sized block, 16 utterances of 320 000 samples
        dict(name="scan train 16x999x2048", op="scan", mode="train", dtype="bf16", batch=16, frames=999, channels=2048, states=16, groups=1, gated=True, ragged=False),
        # one frame of 8 streams: the norms' latency
        dict(name="norm step 8x768", op="norm", mode="prompt", dtype="bf16", batch=8, frames=1, channels=768, kind="layer", gate="row", post=True, scaled=True),
        # one training step of a base-sized block, a gate per frame
        dict(name="norm train 8x781x768", op="norm", mode="train", dtype="bf16", batch=8, frames=781, channels=768, kind="layer", gate="row", post=True, scaled=True),
        # one training step of a large-sized block, a gate per utterance, root-mean-square norms
        dict(name="norm train 32x1499x1024", op="norm", mode="train", dtype="bf16", batch=32, frames=1499, channels=1024, kind="rms", gate="utterance", post=True, scaled=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    mode = rng.choice(["prompt", "train"] if op == "norm" else ["step", "prompt", "train"])
    case = dict(op=op, mode=mode, dtype=rng.choice(["bf16", "bf16", "f32"]))
    channels = _log(rng, 32, 2048)
    if rng.random() < 0.6:
        channels = max(32, channels // 64 * 64)
    batch = _log(rng, 1, 256 if mode == "step" else 32)
    most = 16 * 999 * 2048 if op != "norm" else 32 * 1499 * 1024
    frames = 1 if mode == "step" else _log(rng, 1, max(1, min(20000, most // (batch * channels))))
    case.update(batch=batch, frames=frames)
    if op == "conv":
        case.update(channels=channels, taps=rng.choice([2, 3, 4, 4]), ragged=mode != "step" and rng.random() < 0.5)
    elif op == "scan":
        groups = rng.choice([1, 1, 2, 4])
        case.update(channels=max(8, channels // groups) * groups, states=rng.choice([4, 8, 16, 16]) if rng.random() < 0.7 else rng.randint(1, 16), groups=groups,
                    gated=rng.random() < 0.7, ragged=mode != "step" and rng.random() < 0.5)
    else:
        case.update(channels=channels, kind=rng.choice(["layer", "rms"]), gate=rng.choice(["row", "utterance", "none"]), post=rng.random() < 0.8, scaled=rng.random() < 0.7)
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, T, C = case["batch"], case["frames"], case["channels"]
    train = case["mode"] == "train"

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    def leaf(t):
        return t.detach().requires_grad_(train) if t is not None else None

    s = {"case": case, "lengths": None}
    if case.get("ragged"):
        s["lengths"] = torch.randint(1, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        s["lengths"][B // 2] = T
    if case["op"] == "conv":
        K = case["taps"]
        s["weight"] = leaf(normal(C, K, scale=1 / math.sqrt(K), dtype=torch.float32))
        s["bias"] = leaf(normal(C, scale=0.1, dtype=torch.float32))
        if case["mode"] == "step":
            s["x"], s["state"] = normal(B, C), normal(B, K - 1, C)
        else:
            s["x"] = leaf(normal(B, T, 2 * C)[:, :, :C])                    # one half of a block's input projection
            s["state"] = normal(B, K - 1, C) if case["mode"] == "prompt" else None
    elif case["op"] == "scan":
        N, G = case["states"], case["groups"]
        R = max(4, C // 16)
        s["A"] = leaf(-(torch.arange(1, N + 1, device="cuda").float() * torch.exp(0.1 * normal(C, N, dtype=torch.float32))))
        s["D"] = leaf(1 + normal(C, scale=0.1, dtype=torch.float32))
        step = torch.exp(torch.rand(C, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = leaf(step + torch.log(-torch.expm1(-step)))           # softplus(dt_bias) spread over 0.001 .. 0.1
        lead = (B,) if case["mode"] == "step" else (B, T)
        s["u"] = leaf(F.silu(normal(*lead, C, dtype=torch.float32)).to(dt))
        s["dt"] = leaf(normal(*lead, C, scale=0.5))
        proj = normal(*lead, R + 2 * G * N)                                 # (dt's low rank input, B, C): one product's output
        s["B"] = leaf(proj[..., R:R + G * N].unflatten(-1, (G, N)))
        s["C"] = leaf(proj[..., R + G * N:].unflatten(-1, (G, N)))
        s["z"] = leaf(normal(*lead, 2 * C)[..., C:]) if case["gated"] else None
        s["state"] = normal(B, C, N, dtype=torch.float32) if not train else None
    else:
        s["x"], s["o"] = leaf(normal(B, T, C)), leaf(normal(B, T, C, scale=3.0))
        s["weight"] = leaf(1 + normal(C, scale=0.1, dtype=torch.float32))
        layer = case["kind"] == "layer"
        s["bias"] = leaf(normal(C, scale=0.1, dtype=torch.float32)) if layer else None
        s["post_weight"] = leaf(1 + normal(C, scale=0.1, dtype=torch.float32)) if case["post"] else None
        s["post_bias"] = leaf(normal(C, scale=0.1, dtype=torch.float32)) if case["post"] and layer else None
        s["gate"] = leaf(normal(B, T if case["gate"] == "row" else 1, C)) if case["gate"] != "none" else None
        s["scale"] = leaf(0.5 + normal(C, scale=0.1, dtype=torch.float32)) if case["scaled"] else None
        if train:
            s["dr"], s["dn"] = normal(B, T, C), normal(B, T, C)
    if train and case["op"] != "norm":
        s["dy"] = normal(B, T, C)
    return s


def _grads(outputs, leaves, upstream):
    names = [k for k in leaves if leaves[k] is not None]
    got = torch.autograd.grad(outputs, [leaves[k] for k in names], upstream)
    return {"d" + k: g for k, g in zip(names, got)}


def run(s):
    return {"conv": _conv, "scan": _scan, "norm": _norm}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------------ short causal convolution
def _conv(s):
    mode = s["case"]["mode"]
    if own:
        from audio8_amd import ops
        if mode == "step":
            return {"y": ops.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"]), "state": s["state"]}
        if mode == "prompt":
            y, state = ops.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"], return_state=True)
            return {"y": y, "state": state}
        y = ops.causal_conv(s["x"], s["weight"], s["bias"], lengths=s["lengths"])
        return {"y": y, **_grads([y], {k: s[k] for k in ("x", "weight", "bias")}, [s["dy"]])}
    with torch.no_grad():
        return _conv_plain(s, mode)


def _valid(lengths, T):
    return (torch.arange(T, device="cuda")[None, :] < lengths[:, None])[..., None]


def _conv_plain(s, mode):
    w, b, K = s["weight"], s["bias"], s["case"]["taps"]
    if mode == "step":
        e = torch.cat([s["state"], s["x"][:, None]], 1)
        y = F.silu((e.float() * w.t()).sum(1) + b).to(s["x"].dtype)
        s["state"].copy_(e[:, 1:])
        return {"y": y, "state": s["state"]}
    x = s["x"]
    B, T, C = x.shape
    xf = x.float()
    if s["lengths"] is not None:
        valid = _valid(s["lengths"], T)
        xf = torch.where(valid, xf, 0.0)
    head = s["state"].float() if s["state"] is not None else xf.new_zeros(B, K - 1, C)
    e = torch.cat([head, xf], 1)
    pre = sum(e[:, k:k + T] * w[:, k] for k in range(K)) + b
    y = F.silu(pre)
    if s["lengths"] is not None:
        y = torch.where(valid, y, 0.0)
    if mode == "prompt":
        at = (s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device="cuda"))[:, None] + torch.arange(K - 1, device="cuda")
        return {"y": y.to(x.dtype), "state": e[torch.arange(B, device="cuda")[:, None], at].to(x.dtype)}
    sig = torch.sigmoid(pre)
    g = s["dy"].float() * (sig * (1 + pre * (1 - sig)))
    if s["lengths"] is not None:
        g = torch.where(valid, g, 0.0)
    gp = F.pad(g, (0, 0, 0, K - 1))
    dx = sum(gp[:, K - 1 - k:K - 1 - k + T] * w[:, k] for k in range(K))
    dw = torch.stack([(g * e[:, k:k + T]).sum((0, 1)) for k in range(K)], -1)
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dweight": dw, "dbias": g.sum((0, 1))}


# ---------------------------------------------------------------------------------------------- selective state space scan
def _scan(s):
    mode = s["case"]["mode"]
    if own:
        from audio8_amd import ops
        if mode == "step":
            return {"y": ops.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"]), "state": s["state"]}
        if mode == "prompt":
            y, state = ops.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"],
                                          lengths=s["lengths"], return_state=True)
            return {"y": y, "state": state}
        y = ops.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], lengths=s["lengths"])
        return {"y": y, **_grads([y], {k: s[k] for k in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")}, [s["dy"]])}
    with torch.no_grad():
        return _scan_step_plain(s) if mode == "step" else _scan_plain(s, mode)


def _per_channel(m, C):
    """[..., G, N] shared by a group's channels -> f32 [..., C, N]."""
    return m.float().repeat_interleave(C // m.shape[-2], -2)


def _scan_step_plain(s):
    u, C = s["u"].float(), s["u"].shape[-1]
    delta = F.softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * u)[..., None] * _per_channel(s["B"], C)
    y = (h * _per_channel(s["C"], C)).sum(-1) + s["D"] * u
    if s["z"] is not None:
        y = y * F.silu(s["z"].float())
    s["state"].copy_(h)
    return {"y": y.to(s["u"].dtype), "state": s["state"]}


def _recur(a, b, h0):
    """h[:, t] = a[:, t] h[:, t-1] + b[:, t], h[:, -1] = h0.  The frames are cut into blocks of about the square root of their number: all
    blocks recur side by side, then one block's end goes into the next one's beginning."""
    B, T = a.shape[:2]
    L = max(1, math.isqrt(T))
    n = -(-T // L)
    a = F.pad(a, (0, 0, 0, 0, 0, n * L - T), value=1.0).unflatten(1, (n, L))
    h = F.pad(b, (0, 0, 0, 0, 0, n * L - T)).unflatten(1, (n, L))
    p = a.clone()
    for i in range(1, L):
        h[:, :, i] += a[:, :, i] * h[:, :, i - 1]
        p[:, :, i] *= p[:, :, i - 1]
    first = torch.empty_like(h[:, :, 0])
    first[:, 0] = h0
    for i in range(1, n):
        first[:, i] = h[:, i - 1, -1] + p[:, i - 1, -1] * first[:, i - 1]
    return h.addcmul_(p, first[:, :, None]).flatten(1, 2)[:, :T]


def _scan_plain(s, mode):
    u, z, dy = s["u"], s["z"], s.get("dy")
    B, T, C = u.shape
    uf = u.float()
    raw = s["dt"].float() + s["dt_bias"]
    delta = F.softplus(raw)
    Bc, Cc = _per_channel(s["B"], C), _per_channel(s["C"], C)
    gate = F.silu(z.float()) if z is not None else torch.ones_like(uf)
    if s["lengths"] is not None:                       # frames behind an utterance's end: a step of length zero, no output
        valid = _valid(s["lengths"], T)
        delta, uf, gate = torch.where(valid, delta, 0.0), torch.where(valid, uf, 0.0), torch.where(valid, gate, 0.0)
    a = torch.exp(delta[..., None] * s["A"])
    h0 = s["state"] if s["state"] is not None else a.new_zeros(B, C, a.shape[-1])
    h = _recur(a, (delta * uf)[..., None] * Bc, h0)
    y = (h * Cc).sum(-1) + s["D"] * uf
    out = {"y": (y * gate).to(u.dtype)}
    if mode == "prompt":
        return {**out, "state": h[:, -1].clone()}
    N, G = a.shape[-1], s["B"].shape[-2]
    dyf = dy.float()
    g = dyf * gate
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    adj = _recur(nxt.flip(1), (Cc * g[..., None]).flip(1), torch.zeros_like(h0)).flip(1)
    dC = (g[..., None] * h).unflatten(2, (G, C // G)).sum(3)
    dB = (adj * (delta * uf)[..., None]).unflatten(2, (G, C // G)).sum(3)
    sB = (adj * Bc).sum(-1)
    back = adj * a * torch.cat([h0[:, None], h[:, :-1]], 1)
    ddelta = uf * sB + (back * s["A"]).sum(-1)
    draw_ = ddelta * torch.sigmoid(raw)
    if s["lengths"] is not None:
        draw_ = torch.where(valid, draw_, 0.0)
    out["du"] = (delta * sB + s["D"] * g).to(u.dtype)
    out["ddt"] = draw_.to(u.dtype)
    out["dA"] = (back * delta[..., None]).sum((0, 1))
    out["dB"], out["dC"] = dB.to(u.dtype), dC.to(u.dtype)
    out["dD"] = (g * uf).sum((0, 1))
    if z is not None:
        sig = torch.sigmoid(z.float())
        dz = dyf * y * (sig * (1 + z.float() * (1 - sig)))
        out["dz"] = (torch.where(valid, dz, 0.0) if s["lengths"] is not None else dz).to(u.dtype)
    out["ddt_bias"] = draw_.sum((0, 1))
    return out


# ------------------------------------------------------------------------------------------------------ gated residual norms
NORM_LEAVES = ("x", "o", "weight", "bias", "post_weight", "post_bias", "gate", "scale")


def _norm(s):
    if own:
        from audio8_amd import ops
        r, n = ops.gated_residual_norm(s["x"], s["o"], s["weight"], s["bias"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                                       scale=s["scale"], eps=EPS, kind=s["case"]["kind"])
        if s["case"]["mode"] == "prompt":
            return {"r": r, "n": n}
        return {"r": r, "n": n, **_grads([r, n], {k: s[k] for k in NORM_LEAVES}, [s["dr"], s["dn"]])}
    with torch.no_grad():
        return _norm_plain(s)


def _hat(v, layer):
    if layer:
        v = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * rstd, rstd


def _hat_back(dh, h, rstd, layer):
    d = dh - h * (dh * h).mean(-1, keepdim=True)
    return rstd * (d - dh.mean(-1, keepdim=True) if layer else d)


def _norm_plain(s):
    layer, dt = s["case"]["kind"] == "layer", s["x"].dtype
    x, o = s["x"].float(), s["o"].float()
    p = o
    if s["post_weight"] is not None:
        ohat, orstd = _hat(o, layer)
        p = ohat * s["post_weight"]
        if s["post_bias"] is not None:
            p = p + s["post_bias"]
    gate = s["gate"].float() if s["gate"] is not None else 1.0
    scale = s["scale"] if s["scale"] is not None else 1.0
    r = x + scale * gate * p
    rhat, rrstd = _hat(r, layer)
    n = rhat * s["weight"]
    if s["bias"] is not None:
        n = n + s["bias"]
    out = {"r": r.to(dt), "n": n.to(dt)}
    if s["case"]["mode"] == "prompt":
        return out
    dr, dn = s["dr"].float(), s["dn"].float()
    dx = dr + _hat_back(dn * s["weight"], rhat, rrstd, layer)
    dp = dx * gate * scale
    out["dx"] = dx.to(dt)
    out["dweight"] = (dn * rhat).sum((0, 1))
    if s["bias"] is not None:
        out["dbias"] = dn.sum((0, 1))
    if s["post_weight"] is not None:
        out["dpost_weight"] = (dp * ohat).sum((0, 1))
        if s["post_bias"] is not None:
            out["dpost_bias"] = dp.sum((0, 1))
        out["do"] = _hat_back(dp * s["post_weight"], ohat, orstd, layer).to(dt)
    else:
        out["do"] = dp.to(dt)
    if s["gate"] is not None:
        dgate = dx * scale * p
        out["dgate"] = (dgate.sum(1, keepdim=True) if s["gate"].shape[1] != x.shape[1] else dgate).to(dt)
    if s["scale"] is not None:
        out["dscale"] = (dx * gate * p).sum((0, 1))
    return out


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    B, T, C = case["batch"], case["frames"], case["channels"]
    m = B * T * C
    train = case["mode"] == "train"
    if case["op"] == "conv":
        K = case["taps"]
        if train:                                      # x, dy -> y, dx
            return {"bytes": 4 * m * e + 8 * C * (K + 1), "flops": m * (6 * K + 20)}
        return {"bytes": 2 * m * e + 2 * B * (K - 1) * C * e + 4 * C * (K + 1), "flops": m * (2 * K + 5)}
    if case["op"] == "scan":
        N, bc = case["states"], 2 * B * T * case["groups"] * case["states"] * e
        own_, z = 4 * C * (N + 2), 1 if case["gated"] else 0
        if train:                                      # u, dt, z, dy, B, C -> y, du, ddt, dz, dB, dC
            return {"bytes": (6 + 2 * z) * m * e + 2 * bc + 2 * own_, "flops": m * (25 * N + 40)}
        return {"bytes": (3 + z) * m * e + bc + own_ + 8 * B * C * N, "flops": m * (7 * N + 20)}
    g = {"row": m, "utterance": B * C, "none": 0}[case["gate"]] * e
    if train:                                          # x, o, gate, dr, dn -> r, n, dx, do, dgate
        return {"bytes": 8 * m * e + 2 * g + 40 * C, "flops": 50 * m}
    return {"bytes": 4 * m * e + g + 20 * C, "flops": 18 * m}


# --------------------------------------------------------------------------- the definitions in 64 bits, gradients by the tape
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (v.detach().double().requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in s.items()}
    return {"conv": _conv_exact, "scan": _scan_exact, "norm": _norm_exact}[case["op"]](d)


def _conv_exact(s):
    K, mode = s["case"]["taps"], s["case"]["mode"]
    x = s["x"][:, None] if mode == "step" else s["x"]
    B, T, C = x.shape
    head = s["state"] if s["state"] is not None else x.new_zeros(B, K - 1, C)
    e = torch.cat([head, x], 1)
    pre = (e.unfold(1, K, 1) * s["weight"]).sum(-1) + s["bias"]
    y = pre / (1 + torch.exp(-pre))
    if s["lengths"] is not None:
        y = y * _valid(s["lengths"], T).double()
    if mode == "step":
        return {"y": y[:, 0], "state": e[:, 1:]}
    if mode == "prompt":
        ends = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
        return {"y": y, "state": torch.stack([e[i, t:t + K - 1] for i, t in enumerate(ends)])}
    return {"y": y.detach(), **_grads([y], {k: s[k] for k in ("x", "weight", "bias")}, [s["dy"]])}


def _scan_exact(s):
    mode = s["case"]["mode"]
    names = [k for k in ("u", "dt", "B", "C", "z") if s[k] is not None]
    frames = {k: (s[k][:, None] if mode == "step" else s[k]) for k in names}
    B, T, C = frames["u"].shape
    h = s["state"] if s["state"] is not None else frames["u"].new_zeros(B, C, s["A"].shape[1])
    ends = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    share = torch.arange(C, device="cuda") // (C // frames["B"].shape[2])
    ys = []
    cut = {k: frames[k].unbind(1) for k in names}
    for t in range(T):
        live = (t < ends)[:, None].double()
        raw = cut["dt"][t] + s["dt_bias"]
        delta = torch.logaddexp(raw, torch.zeros_like(raw)) * live
        h = torch.exp(delta[..., None] * s["A"]) * h + (delta * cut["u"][t])[..., None] * cut["B"][t][:, share]
        y = (h * cut["C"][t][:, share]).sum(-1) + s["D"] * cut["u"][t]
        if s["z"] is not None:
            y = y * cut["z"][t] / (1 + torch.exp(-cut["z"][t]))
        ys.append(y * live)
    y = torch.stack(ys, 1)
    if mode == "step":
        return {"y": y[:, 0], "state": h}
    if mode == "prompt":
        return {"y": y, "state": h}
    return {"y": y.detach(), **_grads([y], {k: s[k] for k in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")}, [s["dy"]])}


def _norm_exact(s):
    def norm(v, w, b):
        mean = v.mean(-1, keepdim=True) if s["case"]["kind"] == "layer" else 0.0
        v = (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + EPS) * w
        return v if b is None else v + b

    p = s["o"] if s["post_weight"] is None else norm(s["o"], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        p = p * s["gate"]
    if s["scale"] is not None:
        p = p * s["scale"]
    r = s["x"] + p
    n = norm(r, s["weight"], s["bias"])
    if s["case"]["mode"] == "prompt":
        return {"r": r, "n": n}
    return {"r": r.detach(), "n": n.detach(), **_grads([r, n], {k: s[k] for k in NORM_LEAVES}, [s["dr"], s["dn"]])}
