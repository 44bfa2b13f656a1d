"""The selective scan in growing systems, with bounds per element (yardstick: the magnitude of an element's own terms, the oracle's `mag`)."""
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
