"""ops.linear on a slice of a wider projection: evenly spaced rows that are no dense matrix."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [8, 64])
def test_linear_of_a_slice(K, dtype):
    from audio8_amd import ops
    gen = torch.Generator().manual_seed(K)
    wide = torch.randn(3, 40, K + 32, generator=gen).to(dtype).cuda()
    w = torch.randn(192, K, generator=gen).cuda().requires_grad_()
    dy = torch.randn(3, 40, 192, generator=gen).to(dtype).cuda()
    res = []
    for x in (wide[..., 8:8 + K], wide[..., 8:8 + K].contiguous()):
        x = x.detach().requires_grad_()
        y = ops.linear(x, w, None)
        res.append([y, *torch.autograd.grad(y, [x, w], dy)])
    for p, q in zip(*res):
        assert torch.equal(p, q)
    ref = wide[..., 8:8 + K].double() @ w.detach().to(dtype).double().t()
    assert (res[0][0].double() - ref).abs().max() < 2.0 ** -7 * ref.abs().max()
