"""Gradients of constant rows of a large offset (csrc/ln.hip): what lies behind a
row's end in its threads' registers must not meet (0 - mean) / deviation, which is
past fp32's range there.  With s - mean = 0 the formulas are
dx = (g - mean(g)) / sqrt(eps), dw = 0, db = sum dy."""
import math

import pytest
import torch

from distributed_kfac_pytorch_amd.ops import ln

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


@pytest.mark.parametrize('D', [3, 8, 9, 20, 100, 104, 257, 650, 1030, 1032, 3001, 5000, 9000, 12300,
                               16385, 20000])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('weights', [False, True])
def test_constant_rows_of_large_offset(D, dtype, weights):
    # 2^109 / sqrt(1e-12) is 2^129, past fp32; D 2^109 is not, and its sums are exact
    rows, eps = 37, 1e-12
    x = torch.ones(rows, D, device='cuda')
    x[0::3] *= 2.0 ** 109
    x[1::3] *= -2.0 ** 109
    x = x.to(dtype).requires_grad_(True)
    gen = torch.Generator(device='cuda').manual_seed(D)
    dy = torch.randn(rows, D, device='cuda', generator=gen).to(dtype)
    w = b = None
    if weights:
        w = torch.randn(D, device='cuda', generator=gen).to(dtype).requires_grad_(True)
        b = torch.zeros(D, device='cuda', dtype=dtype, requires_grad=True)
    y = ln.layer_norm(x, D, w, b, eps)
    assert not y.any()
    got = torch.autograd.grad(y, [x] + ([w, b] if weights else []), dy)
    g = dy.double() * (w.detach().double() if weights else 1)
    want = (g - g.mean(1, keepdim=True)) / math.sqrt(float(torch.tensor(eps)))
    # a sum along a row is a chain of at most D / 64 + 16 roundings; five more behind it
    most = (g.abs() + g.abs().mean(1, keepdim=True)) / math.sqrt(eps)
    off = (got[0].double() - want).abs()
    allow = (D / 64 + 24) * U * most + torch.finfo(dtype).eps / 2 * (1 + 1e-3) * want.abs()
    assert torch.isfinite(got[0]).all() and (off <= allow).all(), float((off / allow).max())
    if weights:
        assert not got[1].any()
        off = (got[2].double() - dy.double().sum(0)).abs()
        assert (off <= (rows + 8) * U * dy.double().abs().sum(0)
                + torch.finfo(dtype).eps / 2 * (1 + 1e-3) * dy.double().sum(0).abs()).all()
