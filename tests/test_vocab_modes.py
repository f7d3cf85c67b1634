"""ops.vocab under dispatch modes and torch.compile: the formulas in torch operations
that these can see, with the values and gradients of the ordinary call."""
import math

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint, create_selective_checkpoint_contexts
from torch.utils.flop_counter import FlopCounterMode

from distributed_kfac_pytorch_amd.ops import vocab
from tests import _vocab_oracle as oracle

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
F32, BF16 = torch.float32, torch.bfloat16


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def inputs(device, dtype=F32, V=130):
    """Ordinary, masked, NaN and tied rows, signed zeros and signed NaN."""
    _, x = oracle.edge_rows(V, dtype, device)
    more = torch.randn(3, V, generator=torch.Generator().manual_seed(1)).to(device, dtype)
    more[0] = math.nan
    more[1, 3] = -torch.tensor(math.nan)
    x = torch.cat([x, more]).requires_grad_(True)
    N = len(x)
    t = (torch.arange(N) * 7 % V).to(device)
    t[2] = -100
    ids = torch.stack([t.clamp(min=0), (t + 3) % V], 1)
    ids[4] = -1
    q = torch.linspace(-1, 1, 2 * N).view(N, 2).to(device)
    return x, t, ids, q, torch.linspace(0.5, 1.5, N).to(device)


def all_of(x, t, ids, q, g):
    r = vocab.token_logprobs(x, t, top_k=7, entropy=True, temperature=0.8)
    loss = vocab.topk_distill_loss(x, ids, q, 1.3)
    d = torch.autograd.grad([r.logprobs, r.entropy, loss], x, [g, g, g])[0]
    return r.top_ids, r.logprobs, r.entropy, r.top_logprobs, loss, d


def same(a, b, dtype):
    assert torch.equal(a[0], b[0])
    for u, v in zip(a[1:], b[1:]):
        # fp32 formulas of some ten roundings on both sides, one rounding to bf16 in the gradient
        tol = 2 * torch.finfo(u.dtype).eps if u.dtype == BF16 else 1e-5
        assert torch.allclose(u.double(), v.double(), rtol=tol, atol=tol, equal_nan=True)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_a_dispatch_mode_sees_operations(device, dtype):
    args = inputs(device, dtype)
    want = all_of(*args)
    with Seen() as mode:
        got = all_of(*args)
    same(got, want, dtype)
    assert any('exp' in n for n in mode.names) and any('sort' in n for n in mode.names)


@pytest.mark.parametrize('device', DEVICES)
def test_flop_counter_and_selective_checkpoint(device):
    x, t, ids, q, g = inputs(device)
    head = torch.nn.Linear(8, 50).to(device)
    h = torch.randn(6, 8, generator=torch.Generator().manual_seed(0)).to(device)
    t, ids, q = torch.arange(6, device=device), ids[:6] % 50, q[:6]

    def loss(h):
        out = head(h)
        r = vocab.token_logprobs(out, t, entropy=True)
        return (vocab.topk_distill_loss(out, ids, q) - r.logprobs - 0.1 * r.entropy).sum()
    want = torch.autograd.grad(loss(h), head.weight)[0]
    with FlopCounterMode(display=False) as count:
        got = torch.autograd.grad(loss(h), head.weight)[0]
    assert count.get_total_flops() >= 2 * 6 * 8 * 50 and torch.allclose(got, want, atol=1e-5)

    def contexts():
        return create_selective_checkpoint_contexts([torch.ops.aten.addmm.default])
    out = checkpoint(loss, h, use_reentrant=False, context_fn=contexts)
    assert torch.allclose(torch.autograd.grad(out, head.weight)[0], want, atol=1e-5)


@pytest.mark.parametrize('device', DEVICES)
def test_compiled(device):
    x, t, ids, q, g = inputs(device)
    want = all_of(x, t, ids, q, g)

    def values(x):
        r = vocab.token_logprobs(x * 1, t, top_k=7, entropy=True, temperature=0.8)
        return r.top_ids, r.logprobs, r.entropy, r.top_logprobs, \
            vocab.topk_distill_loss(x * 1, ids, q, 1.3)
    torch._dynamo.reset()
    got = torch.compile(values, backend='eager')(x)
    d = torch.autograd.grad([got[1], got[2], got[4]], x, [g, g, g])[0]
    same(got + (d,), want, F32)
    torch._dynamo.reset()


def test_transforms_are_still_refused():
    x, t = torch.randn(2, 5), torch.tensor([1, 2])
    with pytest.raises(TypeError):
        torch.func.vmap(lambda v: vocab.token_logprobs(v, t[0]).logprobs)(x)
    with pytest.raises(TypeError):
        torch.func.jvp(lambda v: vocab.token_logprobs(v, t).logprobs, (x,), (x,))
    with pytest.raises(TypeError):
        torch.jit.trace(lambda v: vocab.token_logprobs(v, t).logprobs, (x,))
