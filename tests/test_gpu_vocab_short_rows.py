"""Many alternatives of short rows (csrc/vocab.hip): nearly every element is a
candidate, so that the ones below the k-th are dropped before they are ordered."""
import pytest
import torch

from distributed_kfac_pytorch_amd.ops import vocab
from tests import _vocab_oracle as oracle

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize('N,V,k', [(5000, 512, 128), (3000, 1000, 100), (2000, 401, 128),
                                   (600, 1023, 33), (2, 512, 128), (5000, 1024, 128)])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('values', ['spread', 'steps', 'equal'])
def test_many_alternatives_of_short_rows(N, V, k, dtype, values):
    g = torch.Generator(device='cuda').manual_seed(V + k)
    x = torch.randn(N, V, device='cuda', generator=g) * 3
    x = {'spread': x, 'steps': (x * 2).round(), 'equal': torch.zeros_like(x)}[values].to(dtype)
    r = vocab.token_logprobs(x, top_k=k)
    want = oracle.order(x)[:, :k]
    assert torch.equal(r.top_ids, want)
    lp = torch.log_softmax(x.double(), -1).gather(1, want)
    # |lp| < 32, a rounding of which is 2^-20: three of them, and the sum's own 30 of 2^-24
    assert float((r.top_logprobs - lp).abs().max()) < 6 * 2.0 ** -20
    again = vocab.token_logprobs(x, top_k=k)
    assert torch.equal(r.top_ids, again.top_ids)
    assert torch.equal(r.top_logprobs, again.top_logprobs)
