"""Rows at the end of their type's range (masked by its lowest value, in whole or
in part): their sum is past fp32, their mean is not.  A constant row is its bias."""
import pytest
import torch

from distributed_kfac_pytorch_amd.ops import ln

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize('D', [2, 7, 64, 100, 513, 650, 1030, 2500, 4104, 9000, 16384, 16387, 40000])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('sum_', [False, True])
def test_rows_of_the_lowest_value(D, dtype, sum_):
    low = torch.finfo(dtype).min
    g = torch.Generator(device='cuda').manual_seed(D)
    x = torch.randn(6, D, device='cuda', generator=g).to(dtype)
    x[0], x[1] = low, -low
    x[2, ::2] = low                                     # a variance past fp32 makes the row its bias
    x[3, D // 2] = low
    x[4] = 2.0 ** 15 if dtype == F16 else 2.0 ** 100
    z = torch.zeros_like(x) if sum_ else None
    w = torch.randn(D, device='cuda', generator=g).to(dtype).requires_grad_(True)
    b = torch.randn(D, device='cuda', generator=g).to(dtype).requires_grad_(True)
    dy = torch.randn(6, D, device='cuda', generator=g).to(dtype)
    x.requires_grad_(True)
    y = ln.layer_norm(x, D, w, b, z=z)
    y = y[0] if sum_ else y
    assert torch.equal(y[[0, 1, 4]], b.expand(3, D))     # constant rows
    plain = [5] if dtype != F16 else [2, 3, 5]
    if dtype != F16:
        assert torch.equal(y[2:4], b.expand(2, D))       # a variance past fp32: h is 0, as torch has it
    s = x.detach()[plain].double()
    d = s - s.mean(1, keepdim=True)
    h = d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
    # the mean's D / 64 + 16 roundings meet 1 / deviation, the rest is relative
    n = (D / 64 + 16) * 2.0 ** -24
    top = s.abs().amax(1, keepdim=True) * h.abs().amax(1, keepdim=True) / \
        d.abs().amax(1, keepdim=True)
    want = h * w.detach().double() + b.detach().double()
    allow = w.detach().double().abs() * (n * top + 2 * n * h.abs()) + \
        (torch.finfo(dtype).eps / 2 + 2.0 ** -22) * (want.abs() + b.detach().double().abs()) + 1e-7
    off = (y.detach()[plain].double() - want).abs()
    assert (off <= allow).all(), float((off / allow).max())
    for a in torch.autograd.grad(y, [x, w, b], dy):
        assert torch.isfinite(a).all()
