"""modules.LayerNorm in a trace: torch's own norm, and no complaints."""
import warnings

import pytest
import torch

from distributed_kfac_pytorch_amd.modules import LayerNorm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('sum_', [False, True])
def test_a_trace_does_not_warn_of_python_values(sum_):
    m = LayerNorm(32, device='cuda')
    x = torch.randn(4, 32, device='cuda')
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        warnings.simplefilter('error', torch.jit.TracerWarning)
        t = torch.jit.trace(m, (x, x) if sum_ else (x,))
    y = torch.randn(9, 32, device='cuda')               # another length than the trace's
    got, want = (t(y, y), m(y, y)) if sum_ else ((t(y),), (m(y),))
    for a, b in zip(got, want):
        assert torch.allclose(a, b, atol=1e-5)
