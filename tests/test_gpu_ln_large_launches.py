"""Longer rows, and more of them, than one launch of layer norm takes (fewer than
2^32 threads): its workgroups stride over them, and every row has the bits that it
has in a smaller call."""
import math

import pytest
import torch

from distributed_kfac_pytorch_amd.ops import ln

pytestmark = pytest.mark.gpu

DEV = 'cuda'
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def randn(shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


@pytest.mark.parametrize('sum_', [False, True])
def test_many_long_rows_of_a_norm(sum_):
    N, D = (1 << 16) + 9, 16385
    x = randn((N, D), BF16)
    z = x.flip(1) if sum_ else None
    w, b = randn(D, BF16, 2), randn(D, BF16, 3)
    dy = x[:1].expand(N, D)

    def run(s):
        y = x[s].detach().requires_grad_(True)
        o = ln.layer_norm(y, D, w, b, z=None if z is None else z[s])
        o = o if sum_ else (o,)
        return [v.detach() for v in o] + [torch.autograd.grad(o[0], y, dy[s])[0]]
    whole = run(slice(0, N))
    for s in (slice(0, 11), slice(1 << 15, (1 << 15) + 5), slice((1 << 16) - 3, N)):
        for a, c in zip(whole, run(s)):
            assert torch.equal(a[s], c)


@pytest.mark.parametrize('D', [2 ** 21 + 34, 2 ** 27 + 6])
def test_weight_gradients_of_a_very_long_row(D):
    """Ones of both signs: every sum is exact, the mean is 0 and the variance 1."""
    x = torch.ones(D, device=DEV)
    x[1::2] = -1
    x.requires_grad_(True)
    w = torch.ones(D, device=DEV, requires_grad=True)
    b = torch.zeros(D, device=DEV, requires_grad=True)
    y = ln.layer_norm(x, D, w, b)
    dy = randn(D, F32)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    r = 1 / math.sqrt(1 + 1e-5)
    assert torch.equal(db, dy)
    for got, one in ((y.detach(), x.detach()), (dw, dy * x.detach())):
        # 1 + eps, its root, its reciprocal and two products: five roundings
        assert float((got - one * r).abs().div(one.abs().clamp(min=1e-30)).max()) < 8 * U
