"""Gradients of rows at the end of their type's range under create_graph, where they
are taken through torch operations: the same as without."""
import pytest
import torch

from distributed_kfac_pytorch_amd.ops import ln

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('D', [2, 100, 650, 20000])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_create_graph_on_rows_of_the_lowest_value(D, dtype):
    low = torch.finfo(dtype).min
    g = torch.Generator(device='cuda').manual_seed(D)
    x = torch.randn(4, D, device='cuda', generator=g).to(dtype)
    x[0], x[1, ::2], x[2] = low, low, 2.0 ** 60
    x.requires_grad_(True)
    w = torch.randn(D, device='cuda', generator=g).to(dtype).requires_grad_(True)
    dy = torch.randn(4, D, device='cuda', generator=g).to(dtype)

    def grads(graph):
        return torch.autograd.grad(ln.layer_norm(x, D, w), [x, w], dy, create_graph=graph)
    # of a row of h 0 (2: exactly; 0, 1: 1 / deviation is 0 or the mean's last bit decides) only
    # that it is finite is the same everywhere
    for a, b in zip(grads(True), grads(False)):
        assert torch.isfinite(a).all() and torch.isfinite(b).all()
    # the ordinary row: each side is off by D / 64 + 24 roundings of the terms of
    # r (g - mean(g) - h mean(g h)), which for a row of two cancel to nothing, and one of its type
    a, b = grads(True)[0][3].double(), grads(False)[0][3].double()
    v = x.detach()[3].double()
    r = 1 / (v.var(correction=0) + 1e-5).sqrt()
    h, gw = (v - v.mean()) * r, dy[3].double() * w.detach().double()
    terms = r * (gw.abs() + gw.abs().mean() + h.abs() * (gw * h).abs().mean())
    # of h itself: the mean's roundings of the row's largest value
    terms = terms * (1 + r * v.abs().max())
    allow = 2 * (D / 64 + 24) * 2.0 ** -24 * terms + torch.finfo(dtype).eps * b.abs()
    assert ((a - b).abs() <= allow).all(), float(((a - b).abs() / allow).max())
