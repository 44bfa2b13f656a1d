"""Causal sequence operators without a GPU: the float64 oracle's gradients against differences, and the refusals of the C entry points
and of the Python surface (all of them raised before anything is launched)."""
import ctypes as C

import pytest
import torch

from oracle import seq_ref as R


def rnd(*shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def differences(f, inputs, grads, up, seed):
    """Directional central differences of sum_k <f_k, up_k> against <grads, direction>.  Step 1e-5 in float64: truncation ~ 1e-10 x third
    derivative, cancellation ~ 1e-16 / 1e-5 x |f|: 1e-6 of the terms' size covers both."""
    for i, (name, v) in enumerate(inputs.items()):
        d = rnd(*v.shape, seed=seed + i)

        def at(e):
            o = f(**{**inputs, name: v + e * d})
            return sum((o[k] * u).sum() for k, u in up.items())
        num, ana = (at(1e-5) - at(-1e-5)) / 2e-5, (grads[name] * d).sum()
        size = (grads[name] * d).abs().sum() + 1
        assert abs(num - ana) < 1e-6 * size, (name, float(num), float(ana))


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("K", [2, 4])
def test_conv_oracle_gradient(act, K):
    B, T, Cn = 2, 5, 3
    ins = dict(x=rnd(B, T, Cn, seed=1), w=rnd(Cn, K, seed=2), b=rnd(Cn, seed=3), state=rnd(B, K - 1, Cn, seed=4))
    lengths = torch.tensor([5, 2])
    up = dict(y=rnd(B, T, Cn, seed=5), state=rnd(B, K - 1, Cn, seed=6))
    o = R.conv(**ins, act=act, lengths=lengths, dy=up["y"], dstate_out=up["state"])
    differences(lambda **k: R.conv(**k, act=act, lengths=lengths), ins, dict(x=o["dx"], w=o["dw"], b=o["dbias"], state=o["dstate"]), up, 10)


@pytest.mark.parametrize("softplus", [True, False])
def test_scan_oracle_gradient(softplus):
    B, T, D, N, G = 2, 6, 4, 3, 2
    ins = dict(u=rnd(B, T, D, seed=1), dt=0.3 * rnd(B, T, D, seed=2), A=-rnd(D, N, seed=3).abs(), B=rnd(B, T, G, N, seed=4), C=rnd(B, T, G, N, seed=5),
               D=rnd(D, seed=6), z=rnd(B, T, D, seed=7), dt_bias=rnd(D, seed=8), state=rnd(B, D, N, seed=9))
    lengths = torch.tensor([6, 3])
    up = dict(y=rnd(B, T, D, seed=10), state=rnd(B, D, N, seed=11))
    o = R.scan(**ins, softplus=softplus, lengths=lengths, dy=up["y"], dstate_out=up["state"])
    grads = {k: o["dstate" if k == "state" else "d" + k] for k in ins}
    differences(lambda **k: R.scan(**k, softplus=softplus, lengths=lengths), ins, grads, up, 20)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows", [True, False])
def test_residual_norm_oracle_gradient(kind, rows):
    B, T, Cn = 2, 3, 5
    v = lambda s: rnd(Cn, seed=s)  # noqa: E731
    ins = dict(x=rnd(B, T, Cn, seed=1), o=rnd(B, T, Cn, seed=2), w=v(3), b=v(4), pw=v(5), pb=v(6), gate=rnd(B, T if rows else 1, Cn, seed=7), scale=v(8))
    up = dict(r=rnd(B, T, Cn, seed=9), n=rnd(B, T, Cn, seed=10))
    o = R.residual_norm(**ins, kind=kind, dr=up["r"], dn=up["n"])
    differences(lambda **k: {q: t for q, t in R.residual_norm(**k, kind=kind).items() if q in up}, ins, {k: o["d" + k] for k in ins}, up, 30)


# ------------------------------------------------------------------------------------------------ refusals
def _err(lib):
    return lib.a8_last_error()


def test_entry_points_refuse_bad_descriptors_before_launching():
    from audio8_amd import _lib as L
    lib = L.lib()
    n, m = C.c_int64(), C.c_int64()
    d = L.CausalConvDesc()
    d.size = L.CONV_DESC_SIZE - 4
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"descriptor size" in _err(lib)
    assert lib.a8_causal_conv_fwd(None, None) == 1
    d.size, d.dtype = L.CONV_DESC_SIZE, 5
    assert lib.a8_causal_conv_bwd(C.byref(d), None) == 1 and b"bad dtype" in _err(lib)
    d.dtype, d.B, d.T, d.C, d.K = 0, 1, 4, 8, 5
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"2 to 4 taps" in _err(lib)
    d.K, d.act = 4, 9
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"activation" in _err(lib)
    d.act = 1
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"null weight" in _err(lib)
    d.w = 4096
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"null x" in _err(lib)
    assert lib.a8_causal_conv_step(C.byref(d), None) == 1 and b"one frame" in _err(lib)
    d.x = d.y = d.state = d.state_out = 4096
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"state_out" in _err(lib)
    assert lib.a8_causal_conv_bwd_partial_floats(C.byref(d), None) == 1
    s = L.SelectiveScanDesc()
    s.size = 8
    assert lib.a8_selective_scan_fwd(C.byref(s), None) == 1 and b"descriptor size" in _err(lib)
    s.size, s.B, s.T, s.D, s.N, s.G = L.SCAN_DESC_SIZE, 1, 4, 8, 33, 1
    assert lib.a8_selective_scan_fwd(C.byref(s), None) == 1 and b"1 to 32 states" in _err(lib)
    s.N, s.G = 16, 3
    assert lib.a8_selective_scan_bwd(C.byref(s), None) == 1 and b"groups" in _err(lib)
    s.G = 2
    assert lib.a8_selective_scan_fwd(C.byref(s), None) == 1 and b"null A" in _err(lib)
    s.A = 4096
    assert lib.a8_selective_scan_fwd(C.byref(s), None) == 1 and b"null u" in _err(lib)
    assert lib.a8_selective_scan_bwd(C.byref(s), None) == 1 and b"null" in _err(lib)
    assert lib.a8_selective_scan_step(C.byref(s), None) == 1 and b"one frame" in _err(lib)
    assert lib.a8_selective_scan_workspace(C.byref(s), 1, None, C.addressof(n)) == 1
    assert lib.a8_selective_scan_workspace(C.byref(s), 1, C.addressof(m), C.addressof(n)) == 0 and m.value > 0 and n.value > 0
    r = L.ResidualNormDesc()
    r.size = 0
    assert lib.a8_residual_norm_fwd(C.byref(r), None) == 1 and b"descriptor size" in _err(lib)
    r.size, r.B, r.T, r.C = L.RNORM_DESC_SIZE, 1, 1, 8193
    assert lib.a8_residual_norm_fwd(C.byref(r), None) == 1 and b"8192" in _err(lib)
    r.C, r.kind = 8, 2
    assert lib.a8_residual_norm_fwd(C.byref(r), None) == 1 and b"kind" in _err(lib)
    r.kind, r.post = 1, 1
    assert lib.a8_residual_norm_bwd(C.byref(r), None) == 1 and b"post weight" in _err(lib)
    r.post = 0
    assert lib.a8_residual_norm_fwd(C.byref(r), None) == 1 and b"null x" in _err(lib)
    assert lib.a8_residual_norm_bwd(C.byref(r), None) == 1 and b"null operand" in _err(lib)
    assert lib.a8_residual_norm_bwd_workspace(C.byref(r), None) == 1


def test_entry_points_refuse_more_frames_than_their_indices_hold():
    from audio8_amd import _lib as L
    lib = L.lib()
    n, m = C.c_int64(), C.c_int64()
    d, s = L.CausalConvDesc(), L.SelectiveScanDesc()
    d.size, d.B, d.T, d.C, d.K, d.w = L.CONV_DESC_SIZE, 1, 2 ** 31 - 1, 1, 4, 4096
    s.size, s.B, s.T, s.D, s.N, s.G, s.A = L.SCAN_DESC_SIZE, 1, 2 ** 31 - 1, 1, 1, 1, 4096
    for call in (lambda: lib.a8_causal_conv_fwd(C.byref(d), None), lambda: lib.a8_causal_conv_bwd(C.byref(d), None),
                 lambda: lib.a8_causal_conv_bwd_partial_floats(C.byref(d), C.byref(n)), lambda: lib.a8_selective_scan_fwd(C.byref(s), None),
                 lambda: lib.a8_selective_scan_bwd(C.byref(s), None), lambda: lib.a8_selective_scan_workspace(C.byref(s), 0, C.byref(m), C.byref(n))):
        assert call() == 1 and b"too large" in _err(lib)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_the_python_surface_refuses_sizes_that_a_descriptor_does_not_hold(n):
    """C ints hold 31 bits: 2^32 + 5 frames would become 5 (views of one element: nothing is allocated)."""
    from audio8_amd import ops
    one = torch.ones(1)
    for B, T in ((1, n), (n, 1)):
        x, bc = one.expand(B, T, 1), one.expand(B, T, 1, 1)
        for call in (lambda: ops.causal_conv(x, torch.ones(1, 4)), lambda: ops.selective_scan(x, x, torch.ones(1, 1), bc, bc), lambda: ops.gated_residual_norm(x, x, one)):
            with pytest.raises(ValueError, match="too large"):
                call()
    x = one.expand(n, 1)
    with pytest.raises(ValueError, match="too large"):
        ops.causal_conv_step(x, one.expand(n, 3, 1), torch.ones(1, 4))
    with pytest.raises(ValueError, match="too large"):
        ops.selective_scan_step(x, x, torch.ones(1, 1), one.expand(n, 1, 1), one.expand(n, 1, 1), one.expand(n, 1, 1))


@pytest.mark.parametrize("B, T, width", [(2 ** 24 + 1, 2, 8), (2 ** 22, 1, 1024), (2 ** 25 + 1, 1, 1024)])
def test_norm_backward_refuses_grids_beyond_the_launch_limit_before_it_launches(B, T, width):
    """A gate per utterance: a block per utterance in the backward, a thread per element of the gate's gradient behind it."""
    from audio8_amd import _lib as L
    lib = L.lib()
    r = L.ResidualNormDesc()
    r.size, r.B, r.T, r.C = L.RNORM_DESC_SIZE, B, T, width
    r.x = r.o = r.gate = r.w = r.dr = r.dn = r.dx = r.d_o = r.dgate = r.stats = r.ws = 4096
    r.x_ld = r.o_ld = r.g_bs = width
    assert lib.a8_residual_norm_bwd(C.byref(r), None) == 1 and b"too large" in _err(lib)


@pytest.mark.parametrize("B, T", [(4096, 1), (2 ** 20, 1), (2 ** 26, 2 ** 13), (1, 1), (8, 781), (1, 2 ** 30 - 1)])
def test_conv_backward_partial_sums_follow_the_frames(B, T):
    """At most the size of x or 8192 blocks' partial sums (64 channels each), and never fewer than one block's."""
    from audio8_amd import _lib as L
    n, d = C.c_int64(), L.CausalConvDesc()
    d.size, d.B, d.T, d.C, d.K, d.w = L.CONV_DESC_SIZE, B, T, 1536, 4, 4096
    assert L.lib().a8_causal_conv_bwd_partial_floats(C.byref(d), C.byref(n)) == 0
    assert 5 * 1536 <= n.value <= 2 * max(4096 * 64 * 5 + 5 * 1536, B * T * 1536 // 2)


def test_backwards_refuse_more_channels_than_their_column_sums_take_before_they_launch():
    from audio8_amd import _lib as L
    lib = L.lib()
    d, s = L.CausalConvDesc(), L.SelectiveScanDesc()
    d.size, d.B, d.T, d.C, d.K, d.w, d.x, d.dy, d.dx, d.partials = L.CONV_DESC_SIZE, 1, 1, 2 ** 26, 4, 4096, 4096, 8192, 16384, 4096
    assert lib.a8_causal_conv_bwd(C.byref(d), None) == 1 and b"too large" in _err(lib)
    s.size, s.B, s.T, s.D, s.N, s.G, s.A = L.SCAN_DESC_SIZE, 1, 1, 2 ** 26, 1, 1, 4096
    s.u = s.dt = s.Bm = s.Cm = s.dy = s.ckpt = s.du = s.ddt = s.dBm = s.dCm = s.ws = 4096
    assert lib.a8_selective_scan_bwd(C.byref(s), None) == 1 and b"too large" in _err(lib)


def test_entry_points_refuse_outputs_that_other_blocks_still_read():
    from audio8_amd import _lib as L
    lib = L.lib()
    d, s = L.CausalConvDesc(), L.SelectiveScanDesc()
    d.size, d.B, d.T, d.C, d.K, d.w = L.CONV_DESC_SIZE, 1, 4, 8, 4, 4096
    d.x, d.y = 4096, 4096
    assert lib.a8_causal_conv_fwd(C.byref(d), None) == 1 and b"y may not be x" in _err(lib)
    d.dy, d.dx, d.partials = 8192, 8192, 4096
    assert lib.a8_causal_conv_bwd(C.byref(d), None) == 1 and b"may not be an input" in _err(lib)
    d.dx, d.dstate, d.dstate_out = 16384, 4096, 4096
    assert lib.a8_causal_conv_bwd(C.byref(d), None) == 1 and b"may not be an input" in _err(lib)
    s.size, s.B, s.T, s.D, s.N, s.G, s.A = L.SCAN_DESC_SIZE, 1, 4, 8, 4, 1, 4096
    s.u = s.dt = s.Bm = s.Cm = s.h0 = s.h_out = 4096
    s.y = 8192
    assert lib.a8_selective_scan_fwd(C.byref(s), None) == 1 and b"h_out" in _err(lib)
    s.dh0 = s.dh_out = 4096
    assert lib.a8_selective_scan_bwd(C.byref(s), None) == 1 and b"dh0" in _err(lib)


def test_the_python_surface_refuses_wrong_arguments():
    from audio8_amd import ops
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    x, w = f(2, 5, 8), f(8, 4)
    for bad, msg in ((dict(x=f(5, 8)), "axes"), (dict(weight=f(8, 5)), "2 to 4 taps"), (dict(weight=f(7, 4)), "weight"), (dict(bias=f(7)), "bias"),
                     (dict(activation="gelu"), "activation"), (dict(state=f(2, 4, 8)), "state"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths")):
        with pytest.raises(ValueError, match=msg):
            ops.causal_conv(**{"x": x, "weight": w, **bad})
    for bad in (dict(weight=w.bfloat16()), dict(state=f(2, 3, 8).bfloat16()), dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(x=x.half())):
        with pytest.raises(TypeError):
            ops.causal_conv(**{"x": x, "weight": w, **bad})
    with pytest.raises(RuntimeError, match="GPU"):
        ops.causal_conv(x, w)
    with pytest.raises(ValueError, match="axes"):
        ops.causal_conv_step(x, f(2, 3, 8), w)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.causal_conv_step(f(2, 8), f(2, 8, 3).transpose(1, 2), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.causal_conv_step(f(2, 8).requires_grad_(), f(2, 3, 8), w)
    s = dict(u=x, dt=x, A=f(8, 16), B=f(2, 5, 2, 16), C=f(2, 5, 2, 16))
    for bad, msg in ((dict(u=f(2, 8)), "axes"), (dict(A=f(8, 33)), "1 to 32"), (dict(A=f(7, 16)), "A has"), (dict(B=f(2, 5, 3, 16)), "groups"), (dict(C=f(2, 4, 2, 16)), "C has"),
                     (dict(dt=f(2, 5, 7)), "dt has"), (dict(z=f(2, 4, 8)), "z has"), (dict(D=f(9)), "D has"), (dict(dt_bias=f(1)), "dt_bias"), (dict(state=f(2, 8, 15)), "state")):
        with pytest.raises(ValueError, match=msg):
            ops.selective_scan(**{**s, **bad})
    for bad in (dict(z=x.bfloat16()), dict(A=f(8, 16).double()), dict(B=f(2, 5, 2, 16).bfloat16()), dict(state=f(2, 8, 16).bfloat16())):
        with pytest.raises(TypeError):
            ops.selective_scan(**{**s, **bad})
    with pytest.raises(RuntimeError, match="GPU"):
        ops.selective_scan(**s)
    with pytest.raises(ValueError, match="step"):
        ops.selective_scan_step(x, x, f(8, 16), f(2, 5, 2, 16), f(2, 5, 2, 16), f(2, 8, 16))
    for bad, msg in ((dict(kind="batch"), "kind"), (dict(weight=f(7)), "weight"), (dict(weight=None, bias=f(8)), "without its weight"), (dict(post_bias=f(8)), "without its weight"),
                     (dict(gate=f(2, 4, 8)), "gate"), (dict(gate=f(1, 5, 8)), "gate"), (dict(scale=f(1)), "scale"), (dict(o=f(2, 4, 8)), "o has"), (dict(x=f(8)), "axes")):
        with pytest.raises(ValueError, match=msg):
            ops.gated_residual_norm(**{"x": x, "o": x, "weight": f(8), **bad})
    with pytest.raises(TypeError):
        ops.gated_residual_norm(x, x, f(8), gate=x.bfloat16())
    with pytest.raises(ValueError, match="8192"):
        ops.gated_residual_norm(f(1, 1, 8200), f(1, 1, 8200), f(8200))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.gated_residual_norm(x, x, f(8))


# ------------------------------------------------------------------------------------------------ what torch does with a call by its function
def _stand_ins(monkeypatch):
    """The launches replaced by plain copies: y (r, n) = 2 x, whatever the operator."""
    from audio8_amd import kernels as K

    def twice(x):
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        y.detach().numpy()[...] = 2 * x.detach().numpy()
        return y
    monkeypatch.setattr(K, "causal_conv_fwd", lambda x, *a: (twice(x), None, None))
    monkeypatch.setattr(K, "selective_scan_fwd", lambda u, *a: (twice(u), None, None, None))
    monkeypatch.setattr(K, "residual_norm_fwd", lambda x, *a: (twice(x), twice(x), None, None))
    monkeypatch.setattr(K, "causal_conv_step", lambda x, *a: twice(x))
    monkeypatch.setattr(K, "selective_scan_step", lambda u, *a: twice(u))


def _calls():
    from audio8_amd import ops
    w, A, v = rnd(8, 4, seed=1).float(), rnd(8, 4, seed=2).float(), rnd(8, seed=3).float()
    return [lambda x: ops.causal_conv(x, w), lambda x: ops.selective_scan(x, x, A, x[..., :4], x[..., :4]), lambda x: ops.gated_residual_norm(x, x, v)[1]]


def _steps():
    from audio8_amd import ops
    w, A = rnd(8, 4, seed=1).float(), rnd(8, 4, seed=2).float()
    return [lambda x: ops.causal_conv_step(x, torch.zeros(2, 3, 8), w), lambda x: ops.selective_scan_step(x, x, A, x[:, :4], x[:, :4], torch.zeros(2, 8, 4))]


@pytest.mark.parametrize("recording", [False, True])
def test_a_forward_mode_gradient_is_refused_and_not_dropped(monkeypatch, recording):
    import torch.autograd.forward_ad as fw
    _stand_ins(monkeypatch)
    with torch.set_grad_enabled(recording), fw.dual_level():
        for call, x in [(c, rnd(2, 5, 8, seed=4).float()) for c in _calls()] + [(c, rnd(2, 8, seed=4).float()) for c in _steps()]:
            with pytest.raises(NotImplementedError):
                call(fw.make_dual(x, torch.ones_like(x)))
            assert torch.equal(call(x), 2 * x)             # without a tangent it is a call like any other


@pytest.mark.parametrize("recording", [False, True])
def test_a_trace_holds_the_operator_and_no_step(monkeypatch, recording):
    _stand_ins(monkeypatch)
    with torch.set_grad_enabled(recording):
        for call in _calls():
            traced = torch.jit.trace(call, (rnd(2, 5, 8, seed=4).float(),), check_trace=False)
            x = rnd(2, 5, 8, seed=5).float()
            assert torch.equal(traced(x), 2 * x)
        for step in _steps():
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(step, (rnd(2, 8, seed=4).float(),), check_trace=False)


def test_a_step_refuses_to_drop_a_parameters_gradient(monkeypatch):
    from audio8_amd import ops
    _stand_ins(monkeypatch)
    x, bc = rnd(2, 8, seed=1).float(), rnd(2, 4, seed=2).float()
    conv = dict(weight=rnd(8, 4, seed=3).float(), bias=rnd(8, seed=4).float())
    scan = dict(A=rnd(8, 4, seed=5).float(), D=rnd(8, seed=6).float(), dt_bias=rnd(8, seed=7).float())
    for par, step in ((conv, lambda p: ops.causal_conv_step(x, torch.zeros(2, 3, 8), **p)),
                      (scan, lambda p: ops.selective_scan_step(x, x, B=bc, C=bc, state=torch.zeros(2, 8, 4), **p))):
        assert torch.equal(step(par), 2 * x)
        for k, v in par.items():
            learnt = {**par, k: v.clone().requires_grad_()}
            with pytest.raises(RuntimeError, match="no gradient"):
                step(learnt)
            with torch.no_grad():
                assert torch.equal(step(learnt), 2 * x)
