"""Logits of a diverged model: rows that are NaN throughout, or NaN beside nothing
but masked columns.  Values, loss and gradients are NaN, on both devices and
however a row is cut over workgroups; they are not the 0 of a masked row."""
import math

import pytest
import torch

from distributed_kfac_pytorch_amd.ops import vocab
from tests import _vocab_oracle as oracle

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def nan_rows(V, dtype, device):
    """NaN rows between ordinary and masked ones, and which are NaN."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=g) * 3
    x[1] = math.nan                                     # all of it
    x[2:7] = -math.inf
    x[2, V // 3] = math.nan                             # one beside masked columns
    x[3, 0] = math.nan
    x[4, V - 1] = math.nan
    x[5, :max(V - 2, 1)] = math.nan                     # a padded head: the last ones masked
    bad = torch.tensor([False] + [True] * 5 + [False] * 2)      # row 6 is masked, 0 and 7 ordinary
    return x.to(dtype).to(device), bad


def check(V, dtype, device, k, reps=1):
    x, bad = nan_rows(V, dtype, device)
    x, bad = x.repeat(reps, 1).requires_grad_(True), bad.repeat(reps)
    N, some = len(x), slice(0, 8)                       # the oracle goes row by row
    t = (torch.arange(N) % V).to(device)
    g = torch.linspace(0.5, 1.5, N).to(device)
    gh = torch.linspace(-0.5, 0.25, N).to(device)
    r = vocab.token_logprobs(x, t, top_k=k, entropy=True, temperature=0.8)
    o = oracle.token_logprobs(x.detach()[some], t[some], k, 0.8, g=g[some], gh=gh[some])
    d, = torch.autograd.grad([r.logprobs, r.entropy], [x], [g, gh])
    ids = torch.stack([t, (t + V // 2) % V], 1)
    q = torch.stack([g, gh], 1)
    loss = vocab.topk_distill_loss(x, ids, q, 1.5)
    od = oracle.distill(x.detach()[some], ids[some], q[some], 1.5, g[some])
    dk, = torch.autograd.grad(loss, x, g)
    for name, got, want in (('logprobs', r.logprobs, o['logprobs']),
                            ('entropy', r.entropy, o['entropy']),
                            ('top_logprobs', r.top_logprobs, o['top_logprobs']),
                            ('dlogits', d, o['dlogits']), ('loss', loss, od['loss']),
                            ('distill dlogits', dk, od['dlogits'])):
        oracle.check(name, got[some], want)
        rows = torch.isnan(got.detach()).reshape(N, -1).all(1).cpu()
        assert torch.equal(rows, bad), (name, rows[some].tolist())
        assert not torch.isnan(got.detach()[~bad]).any(), name
    oracle.check_ids(r.top_ids[some], o['top_ids'])
    for only in (r.logprobs, r.entropy):                # each gradient by itself
        if only is r.logprobs:
            out = vocab.token_logprobs(x, t).logprobs
        else:
            out = vocab.token_logprobs(x, entropy=True).entropy
        e, = torch.autograd.grad(out.sum(), x)
        assert torch.equal(torch.isnan(e).all(1).cpu(), bad)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('V', [1, 5, 130, 4100, 70001])
def test_rows_of_nan_are_nan(V, dtype, device):
    check(V, dtype, device, min(V, 3))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('V,k,reps', [(200, 128, 1), (4100, 128, 1), (70001, 128, 1),
                                      (1000, 5, 600), (9000, 40, 80)])
def test_rows_of_nan_with_other_launches(V, k, reps, dtype):
    """Workgroups of 256 threads for many alternatives, one wave a row for many rows,
    rows that are not cut."""
    check(V, dtype, 'cuda', k, reps)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_one_row_cut_over_workgroups(dtype):
    for at in (None, 0, 35000, 70000):
        x = torch.full((1, 70001), math.nan if at is None else -math.inf, device='cuda').to(dtype)
        if at is not None:
            x[0, at] = math.nan
        x.requires_grad_(True)
        r = vocab.token_logprobs(x, torch.tensor([7], device='cuda'), top_k=2, entropy=True)
        assert r.logprobs.isnan().all() and r.entropy.isnan().all()
        assert r.top_logprobs.isnan().all()
        assert r.top_ids.tolist() == [[0, 1] if at in (None,) else [at, 1 if at == 0 else 0]]
        assert torch.autograd.grad(r.logprobs.sum(), x)[0].isnan().all()
        loss = vocab.topk_distill_loss(x, torch.tensor([[7, 9]], device='cuda'),
                                       torch.zeros(1, 2, device='cuda'))
        assert loss.isnan().all() and torch.autograd.grad(loss.sum(), x)[0].isnan().all()


@pytest.mark.parametrize('device', DEVICES)
def test_a_gradient_scaler_sees_a_diverged_head(device):
    """One diverged row makes the head's gradient NaN, so that a scaler skips the step."""
    head = torch.nn.Linear(8, 50).to(device)
    h = torch.randn(4, 8, generator=torch.Generator().manual_seed(0)).to(device)
    h[2] = math.nan
    t = torch.arange(4, device=device)
    r = vocab.token_logprobs(head(h), t, entropy=True)
    for loss in (-r.logprobs.sum(), r.entropy.sum()):
        g, = torch.autograd.grad(loss, head.weight, retain_graph=True)
        assert g.isnan().all() and loss.isnan()
