"""modules.LayerNorm on nested tensors: torch's own norm, as nn.LayerNorm would have it."""
import pytest
import torch
import torch.nn as nn

from distributed_kfac_pytorch_amd.modules import LayerNorm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('layout', [torch.strided, torch.jagged])
def test_nested_tensors(layout):
    """Sequences of different lengths in one tensor, values and gradients."""
    ours = LayerNorm(32, device='cuda')
    ref = nn.LayerNorm(32, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(0)
    rows = [torch.randn(n, 32, device='cuda', generator=g) for n in (2, 5, 1)]
    probe = torch.randn(32, device='cuda', generator=g)
    out = []
    for m in (ours, ref):
        x = torch.nested.nested_tensor(rows, layout=layout, requires_grad=True)
        y = m(x)
        flat = y.values() if layout == torch.jagged else torch.nested.to_padded_tensor(y, 0.0)
        (flat * probe).sum().backward()
        out.append((list(y.detach().unbind()), m.weight.grad.clone(), list(x.grad.unbind())))
    for a, b in zip(out[0][0] + [out[0][1]] + out[0][2], out[1][0] + [out[1][1]] + out[1][2]):
        assert torch.equal(a, b)
