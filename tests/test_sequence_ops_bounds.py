"""The selective scan's frame chunks and the norms' sums over many rows, with bounds per element.

Scan in chunks against the same frames in short calls chained through state and dstate (up to 7 tiles of 16 frames a call is never split).  Calls begin
at tile borders, so both evaluate a tile in the same way from the state in front of it, and differ in that state (or adjoint): a chunk hands it
on as exp(A sum of steps), a chain as a product of one exp per frame.  Each frame adds at most two roundings (exp2's argument and value, the
product), relative to what is handed on, which itself decays by the exponent whose rounding it carries: 2 T roundings for T frames, and T more in
the sums over frames, which the two add up in other orders.  The yardstick per element is the magnitude of its own terms (oracle, `mag`).
Against the definition: 16 T + 40 roundings reach a state or an adjoint (8 a frame each way), at most one ulp each and independent of one another, so
eight standard deviations are 8 sqrt(16 T + 40) ulps; sums over channels or frames add their length under the root.

Norm backward over many rows: a parameter gradient is a sum over frames in registers (rows per block / rows side by side, at most 40 at these sizes),
over a block's waves (4) and over blocks (at most 1536 / 32 by lane, then 64): 110 roundings behind the terms' own 4 (C / 32 + 40).
"""
import pytest
import torch

from oracle import seq_ref as R

ULP = 2.0 ** -24


def rnd(*shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def over(got, ref, mag, F):
    """How far the worst element is beyond its bound (f32): half a step of the value and F roundings of its terms' magnitude."""
    g = got.detach().double().cpu()
    assert tuple(g.shape) == tuple(ref.shape), (g.shape, ref.shape)
    e = (g - ref).abs() - ULP * ref.abs() - F * ULP * mag
    return float(e.nan_to_num(nan=float("inf")).max()) if g.numel() else 0.0


# ------------------------------------------------------------------------------------------------ frame chunks of the scan
CHUNKED = [  # B, T, D, N, G, lengths, frames per chained call
    (1, 781, 64, 16, 1, None, 112),
    (2, 600, 96, 11, 2, [600, 333], 96),
    (3, 400, 40, 17, 1, [129, 400, 250], 64),
    (1, 2500, 32, 4, 1, None, 112),
]


def scan_case(case):
    B, T, D, N, G, lengths, _ = case
    a = dict(u=rnd(B, T, D, seed=1), dt=rnd(B, T, D, seed=2, scale=0.5), A=-torch.exp(rnd(D, N, seed=3) - 1), B=rnd(B, T, G, N, seed=4), C=rnd(B, T, G, N, seed=5),
             D=rnd(D, seed=6), z=rnd(B, T, D, seed=7), dt_bias=rnd(D, seed=8) - 3, state=rnd(B, D, N, seed=9))
    n = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    return a, n, rnd(B, T, D, seed=10), rnd(B, D, N, seed=11)


SEQ = ("u", "dt", "B", "C", "z")
SUMS = ("dA", "dD", "ddt_bias")


def run_scan(f, a, n, dy, dst):
    """-> outputs and gradients of one call of f (ops.selective_scan or a stand-in)."""
    g = {k: v.detach().requires_grad_() for k, v in a.items()}
    y, out = f(*(g[k] for k in ("u", "dt", "A", "B", "C")), D=g["D"], z=g["z"], dt_bias=g["dt_bias"], state=g["state"], lengths=n, return_state=True)
    return y, out, lambda dout: {"d" + k: t for k, t in zip(g, torch.autograd.grad([y, out], list(g.values()), [dy, dout]))}


def chained(f, a, n, dy, dst, L):
    T, parts, state = dy.shape[1], [], a["state"]
    for t in range(0, T, L):
        part = {k: (v[:, t:t + L] if k in SEQ else v) for k, v in a.items()}
        y, state, back = run_scan(f, {**part, "state": state}, (n - t).int() if n is not None else None, dy[:, t:t + L], None)
        parts.append((y, back))
    got, c = [], dst
    for _, back in reversed(parts):
        got.insert(0, back(c))
        c = got[0]["dstate"]
    res = {"y": torch.cat([y for y, _ in parts], 1), "state": state, "dstate": c}
    for k in got[0]:
        if k != "dstate":
            res[k] = sum(g[k].double() for g in got) if k in SUMS else torch.cat([g[k] for g in got], 1)
    return res


@pytest.mark.gpu
@pytest.mark.parametrize("case", CHUNKED, ids=str)
def test_a_scan_in_chunks_is_the_chain_of_its_parts(case):
    from audio8_amd import ops
    a, n, dy, dst = scan_case(case)
    mag = R.scan(**a, lengths=n, dy=dy, dstate_out=dst, mag=True)
    dev = {k: v.cuda() for k, v in a.items()}
    m = n.cuda() if n is not None else None
    y, out, back = run_scan(ops.selective_scan, dev, m, dy.cuda(), None)
    got = {"y": y, "state": out, **back(dst.cuda())}
    want = chained(ops.selective_scan, dev, m, dy.cuda(), dst.cuda(), case[-1])
    for k, v in want.items():
        assert over(got[k], v.detach().double().cpu(), mag[k], 3 * case[1] + 100) <= 0, k
    B, T, D, N, G = case[:5]
    more = {"dB": D // G, "dC": D // G, **{k: B * T for k in SUMS}}
    for k, v in R.scan(**a, lengths=n, dy=dy, dstate_out=dst).items():
        assert over(got[k], v, mag[k], 8 * (16 * T + 40 + N + more.get(k, 0)) ** 0.5) <= 0, "definition: " + k


def oracle_scan_in_two(a, n, dy, dst, at, wrong):
    """The oracle's scan of frames 0 .. at, then of the rest, with the state and the adjoint between them off by the factor `wrong`."""
    def part(lo, hi):
        return {k: (v[:, lo:hi] if k in SEQ else v) for k, v in a.items()}
    T = dy.shape[1]
    n0, n1 = (None, None) if n is None else ((n.clamp(max=at)), (n - at))
    first = R.scan(**part(0, at), lengths=n0)
    second = R.scan(**{**part(at, T), "state": first["state"] * wrong}, lengths=n1, dy=dy[:, at:], dstate_out=dst)
    first = R.scan(**part(0, at), lengths=n0, dy=dy[:, :at], dstate_out=second["dstate"] * wrong)
    res = {"y": torch.cat([first["y"], second["y"]], 1), "state": second["state"], "dstate": first["dstate"]}
    for k in ("du", "ddt", "dB", "dC", "dz"):
        res[k] = torch.cat([first[k], second[k]], 1)
    return {**res, **{k: first[k] + second[k] for k in SUMS}}


@pytest.mark.parametrize("case", CHUNKED, ids=str)
def test_the_bound_of_the_chunks_sees_a_carry_that_is_off_by_a_hundredth(case):
    """In everything that has a frame axis (what sums over frames or lies hundreds of frames from the border has room for it)."""
    a, n, dy, dst = scan_case(case)
    at = min(320, case[1] // 2 // 16 * 16)
    ref, mag = (R.scan(**a, lengths=n, dy=dy, dstate_out=dst, mag=m) for m in (False, True))
    for wrong in (1.0, 1.01):
        off = oracle_scan_in_two(a, n, dy, dst, at, wrong)
        for k in ("y", "du", "ddt", "dB", "dC", "dz"):
            assert (over(off[k], ref[k], mag[k], 3 * case[1] + 100) > 0) == (wrong != 1.0), k


def growing(T, tail):
    """States that grow by exp(1.2 .. 2.4) a frame: silent but for the last frames, upstream gradients for the first ones alone."""
    D, N = 64, 16
    a = dict(u=torch.zeros(1, T, D), dt=1.2 + rnd(1, T, D, seed=2).abs().clamp(max=1.0) * 0.6, A=1 + rnd(D, N, seed=3).abs().clamp(max=1.0) * 0.3, B=rnd(1, T, 1, N, seed=4),
             C=rnd(1, T, 1, N, seed=5))
    a["u"][:, -tail:] = rnd(1, tail, D, seed=1)
    dy = torch.zeros(1, T, D)
    dy[:, :tail] = rnd(1, tail, D, seed=6)
    return a, dy


@pytest.mark.gpu
@pytest.mark.parametrize("T", [128, 781, 2500])
def test_a_growing_system_with_a_silent_beginning(T):
    """A chunk's decay factor may overflow where the state it multiplies is zero (forward: before the first sound; backward: behind the last upstream
    gradient).  Rounding: exp2's argument is at most 3.5 a frame over 16 frames, so 8 + 4 roundings per frame and state, 16 states."""
    from audio8_amd import ops
    a, dy = growing(T, 16)
    g = {k: v.cuda().requires_grad_() for k, v in a.items()}
    y, out = ops.selective_scan(*g.values(), softplus=False, return_state=True)
    got = {"y": y, "state": out, **{"d" + k: t for k, t in zip(g, torch.autograd.grad(y, list(g.values()), dy.cuda()))}}
    ref, mag = (R.scan(**a, softplus=False, dy=dy, mag=m) for m in (False, True))
    for k, v in got.items():
        assert torch.isfinite(v).all(), k
        assert over(v, ref[k], mag[k], 12 * 16 + 40 + {"dB": 64, "dC": 64}.get(k, 16)) <= 0, k


@pytest.mark.gpu
def test_a_chunk_that_grows_behind_one_that_decays():
    """What one chunk hands on is tiny, the next one's factor is beyond f32's range, their product is not.  128 frames, two chunks: exponents -57 and +102
    of a state of size one forward, of an adjoint of 1e-12 backward.  Rounding: exponents up to 147 binary steps in one factor, 2 T for the frames."""
    from audio8_amd import ops
    D, N, T = 64, 16, 128
    a = dict(u=rnd(1, T, D, seed=1, scale=1e-30), dt=torch.cat([torch.full((1, 64, D), 0.9), torch.full((1, 64, D), -1.6)], 1), A=-torch.ones(D, N), B=rnd(1, T, 1, N, seed=4),
             C=rnd(1, T, 1, N, seed=5), state=rnd(1, D, N, seed=6))
    dy, dst = rnd(1, T, D, seed=7, scale=1e-30), rnd(1, D, N, seed=8, scale=1e-12)
    g = {k: v.cuda().requires_grad_() for k, v in a.items()}
    y, out = ops.selective_scan(*(g[k] for k in ("u", "dt", "A", "B", "C")), state=g["state"], softplus=False, return_state=True)
    got = {"y": y, "state": out, **{"d" + k: t for k, t in zip(g, torch.autograd.grad([y, out], list(g.values()), [dy.cuda(), dst.cuda()]))}}
    ref, mag = (R.scan(**a, softplus=False, dy=dy, dstate_out=dst, mag=m) for m in (False, True))
    for k, v in got.items():
        assert torch.isfinite(v).all(), k
        # (below 1e-36 a product of two f32 factors is no longer an f32 with all its bits)
        assert over(v, ref[k], mag[k] + 1e-30, 2 * T + 2 * 147 + 40 + {"dB": D, "dC": D}.get(k, T)) <= 0, k


# ------------------------------------------------------------------------------------------------ column sums of the norms
ROWS = [  # B, T, C, kind, gate
    (7, 1600, 136, "layer", "utterance"),
    (3, 1700, 640, "rms", "rows"),
    (2, 1201, 1100, "layer", "utterance"),
    (2, 600, 4104, "layer", "utterance"),
    (5, 333, 768, "layer", "none"),
    (1, 4099, 24, "rms", "rows"),
]
PARAMS = ("dw", "db", "dpw", "dpb", "dgate", "dscale")


def norm_case(case):
    B, T, C, kind, gate = case
    v = lambda s: 1 + rnd(C, seed=s, scale=0.2)  # noqa: E731
    a = dict(x=rnd(B, T, C, seed=1) + 1, o=rnd(B, T, C, seed=2, scale=3.0) - 2, w=v(3), b=v(4), pw=v(5), pb=v(6),
             gate={"none": None, "rows": rnd(B, T, C, seed=7), "utterance": rnd(B, 1, C, seed=7)}[gate], scale=v(8))
    return a, rnd(B, T, C, seed=9), rnd(B, T, C, seed=10)


def norm_roundings(case):
    return 4 * (case[2] / 32 + 40) + 110


@pytest.mark.gpu
@pytest.mark.parametrize("case", ROWS, ids=str)
def test_norm_gradients_over_many_rows(case):
    from audio8_amd import ops
    a, dr, dn = norm_case(case)
    g = {k: v.cuda().requires_grad_() for k, v in a.items() if v is not None}
    r, n = ops.gated_residual_norm(g["x"], g["o"], g["w"], g["b"], post_weight=g["pw"], post_bias=g["pb"], gate=g.get("gate"), scale=g["scale"], kind=case[3])
    got = {"r": r, "n": n, **{"d" + k: t for k, t in zip(g, torch.autograd.grad([r, n], list(g.values()), [dr.cuda(), dn.cuda()]))}}
    ref, mag = (R.residual_norm(**a, kind=case[3], dr=dr, dn=dn, mag=m) for m in (False, True))
    for k, v in got.items():
        assert over(v, ref[k], mag[k], norm_roundings(case)) <= 0, k


@pytest.mark.parametrize("case", ROWS, ids=str)
def test_the_bound_of_the_norm_gradients_sees_lost_sums_and_lost_rows(case):
    """A gradient that is zero is beyond the bound in most columns; one that lacks the four rows which a block's waves take at once, in some."""
    a, dr, dn = norm_case(case)
    T = case[1]
    ref, mag = (R.residual_norm(**a, kind=case[3], dr=dr, dn=dn, mag=m) for m in (False, True))
    few = {k: (v[:, T // 2:T // 2 + 4] if v is not None and v.dim() == 3 and v.shape[1] == T else v) for k, v in a.items()}
    lost = R.residual_norm(**few, kind=case[3], dr=dr[:, T // 2:T // 2 + 4], dn=dn[:, T // 2:T // 2 + 4])
    for k in PARAMS:
        if k not in ref or (k == "dgate" and case[4] == "rows"):
            continue
        bound = ULP * ref[k].abs() + norm_roundings(case) * ULP * mag[k]
        assert (ref[k].abs() > bound).double().mean() > 0.95, k
        assert (lost[k].abs() > bound).any(), k
