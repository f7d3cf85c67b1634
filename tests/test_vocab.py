"""ops.vocab on the CPU: values and gradients from the definitions, the defined
edges, and what is refused."""
import math

import pytest
import torch
import torch.nn.functional as F

from distributed_kfac_pytorch_amd.ops import vocab
from tests import _vocab_oracle as oracle

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


@pytest.mark.parametrize('dtype', [F32, F64, BF16])
def test_is_log_softmax(dtype):
    torch.manual_seed(0)
    x = torch.randn(2, 5, 11, dtype=dtype, requires_grad=True)
    t = torch.randint(0, 11, (2, 5))
    r = vocab.token_logprobs(x, t, top_k=3, entropy=True)
    wide = x.detach().to(F64).requires_grad_(True)
    lp = F.log_softmax(wide, -1)
    tol = 1e-12 if dtype == F64 else 1e-6
    assert torch.allclose(r.logprobs.double(), lp.gather(-1, t[..., None])[..., 0], atol=tol)
    assert torch.allclose(r.entropy.double(), -(lp.exp() * lp).sum(-1), atol=tol)
    top = lp.topk(3, -1)
    assert torch.equal(r.top_ids, top[1])
    assert torch.allclose(r.top_logprobs.double(), top[0], atol=tol)
    assert r.logprobs.dtype == (F64 if dtype == F64 else F32)
    (r.logprobs.sum() + 0.5 * r.entropy.sum()).backward()
    (lp.gather(-1, t[..., None]).sum() - 0.5 * (lp.exp() * lp).sum()).backward()
    assert x.grad.dtype == dtype
    assert torch.allclose(x.grad.double(), wide.grad, atol=max(tol, 2 * torch.finfo(dtype).eps))
    ce = F.cross_entropy(x.detach().float().reshape(-1, 11), t.reshape(-1))
    assert torch.allclose(-r.logprobs.detach().float().mean(), ce, atol=1e-6)


@pytest.mark.parametrize('T', [0.7, 1.0, 3.0])
def test_differences(T):
    torch.manual_seed(0)
    x = torch.randn(4, 9, dtype=F64, requires_grad=True)
    t = torch.tensor([1, 8, -100, 0])
    assert torch.autograd.gradcheck(
        lambda v: vocab.token_logprobs(v, t, entropy=True, temperature=T)[:2], x)
    ids = torch.tensor([[1, 5, 1], [0, -1, -1], [-1, -1, -1], [2, 3, 8]])
    q = torch.randn(4, 3, dtype=F64)
    assert torch.autograd.gradcheck(lambda v: vocab.topk_distill_loss(v, ids, q, T), x)


@pytest.mark.parametrize('V', [5, 130])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_edges(V, dtype):
    names, x = oracle.edge_rows(V, dtype)
    N = len(names)
    x = x.requires_grad_(True)
    t = torch.arange(N) % V
    g, gh = torch.linspace(-1, 1, N), torch.linspace(0.5, -0.5, N)
    r = vocab.token_logprobs(x, t, top_k=5, entropy=True)
    o = oracle.token_logprobs(x.detach(), t, 5, g=g, gh=gh)
    oracle.check('logprobs', r.logprobs, o['logprobs'])
    oracle.check('entropy', r.entropy, o['entropy'])
    oracle.check('top', r.top_logprobs, o['top_logprobs'])
    oracle.check_ids(r.top_ids, o['top_ids'])
    d, = torch.autograd.grad([r.logprobs, r.entropy], [x], [g, gh])
    oracle.check('dlogits', d, o['dlogits'])
    ids = torch.stack([torch.arange(N) % V, (torch.arange(N) + 2) % V], 1)
    q = torch.randn(N, 2, generator=torch.Generator().manual_seed(1)).to(dtype)
    loss = vocab.topk_distill_loss(x, ids, q)
    o = oracle.distill(x.detach(), ids, q, g=g)
    oracle.check('loss', loss, o['loss'])
    oracle.check('dlogits', torch.autograd.grad(loss, x, g)[0], o['dlogits'])


def test_teacher_rows():
    x = torch.randn(9, 6, requires_grad=True)
    n, i = math.nan, math.inf
    ids = torch.tensor([[0, 1], [-1, -1], [2, 2], [6, 1], [-2, 1], [3, -1], [0, 1], [0, 1], [0, 1]])
    t = torch.tensor([[0., 1], [0, n], [1, 2], [0, 0], [0, 0], [1, n], [-i, -i], [n, 0], [i, 0]])
    g = torch.ones(9)
    loss = vocab.topk_distill_loss(x, ids, t)
    o = oracle.distill(x.detach(), ids, t, g=g)
    assert [math.isnan(v) for v in loss.tolist()] == [False] * 3 + [True, True, False, False,
                                                                   True, True]
    assert loss[1] == 0 and loss[6] == 0
    oracle.check('loss', loss, o['loss'])
    oracle.check('dlogits', torch.autograd.grad(loss, x, g)[0], o['dlogits'])


def masked_by_lowest(dtype, device='cpu'):
    """Rows of which the teacher's tokens are partly masked by the type's lowest
    value, its mass on them from nearly all to nearly nothing."""
    x = torch.randn(4, 40, generator=torch.Generator().manual_seed(0))
    x[:, 1::3] = torch.finfo(dtype).min
    ids = torch.tensor([[0, 1, 4], [3, 4, 7], [2, 5, 1], [0, 10, 2]])
    q = torch.tensor([[20.0, -3, 0], [30.0, -1, -2], [1.0, 2, -24], [1.0, 0, -1]])
    return x.to(dtype).to(device), ids.to(device), q.to(device)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('T', [0.3, 1.0])
def test_teacher_mass_on_masked_tokens(dtype, T):
    x, ids, q = masked_by_lowest(dtype)
    oracle.check('loss', vocab.topk_distill_loss(x, ids, q, T), oracle.distill(x, ids, q, T)['loss'])


def test_targets_out_of_range_are_nan():
    x = torch.randn(4, 6, requires_grad=True)
    t = torch.tensor([6, -1, 3, -100])
    r = vocab.token_logprobs(x, t)
    assert torch.isnan(r.logprobs).tolist() == [True, True, False, False]
    r.logprobs.sum().backward()
    assert torch.isnan(x.grad).all(1).tolist() == [True, True, False, False]
    assert not x.grad[3].any()
    r = vocab.token_logprobs(x, t, ignore_index=-1)
    assert torch.isnan(r.logprobs).tolist() == [True, False, False, True]


def test_a_teachers_alternatives_train_a_student():
    """The alternatives of one call are the other's teacher; over the whole
    vocabulary the loss is the full divergence."""
    torch.manual_seed(0)
    teacher, student = torch.randn(7, 20, dtype=F64), torch.randn(7, 20, dtype=F64)
    tgt = torch.tensor([0, 1, 2, -100, 4, 5, 6])
    r = vocab.token_logprobs(teacher, tgt, top_k=20)
    loss = vocab.topk_distill_loss(student, r.top_ids, r.top_logprobs)
    kl = F.kl_div(F.log_softmax(student, 1), F.log_softmax(teacher, 1), log_target=True,
                  reduction='none').sum(1)
    kl[3] = 0                                    # its alternatives are the unused ids
    assert torch.allclose(loss, kl)


def test_empty_and_shapes():
    x = torch.empty(0, 3, 5, requires_grad=True)
    r = vocab.token_logprobs(x, torch.empty(0, 3, dtype=torch.long), top_k=2, entropy=True)
    assert r.logprobs.shape == r.entropy.shape == (0, 3) and r.top_ids.shape == (0, 3, 2)
    r.logprobs.sum().backward()
    assert x.grad.shape == x.shape
    loss = vocab.topk_distill_loss(x, torch.empty(0, 3, 2, dtype=torch.long),
                                   torch.empty(0, 3, 2))
    assert loss.shape == (0, 3)
    r = vocab.token_logprobs(torch.randn(5), torch.tensor(3), top_k=5, entropy=True)
    assert r.logprobs.shape == () and r.top_ids.shape == (5,)
    r = vocab.token_logprobs(torch.randn(2, 5), top_k=1)
    assert r.logprobs is None and r.entropy is None and r.top_ids.shape == (2, 1)
    assert vocab.token_logprobs(torch.randn(2, 5), torch.tensor([1, 2]).int()).logprobs.shape == (2,)
    assert vocab.token_logprobs(torch.randn(2, 1), torch.tensor([0, 0])).logprobs.tolist() == [0, 0]


def test_alternatives_have_no_gradient():
    x = torch.randn(2, 5, requires_grad=True)
    r = vocab.token_logprobs(x, torch.tensor([1, 2]), top_k=2)
    assert r.logprobs.requires_grad and not r.top_logprobs.requires_grad
    g, = torch.autograd.grad(r.logprobs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                       # no second derivative, and no silent one


@pytest.mark.parametrize('call,error', [
    (lambda x, t: vocab.token_logprobs(x.long(), t), TypeError),
    (lambda x, t: vocab.token_logprobs(x[..., :0], t), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t.float()), TypeError),
    (lambda x, t: vocab.token_logprobs(x, t[:1]), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t.to('meta')), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, top_k=6), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, top_k=-1), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, top_k=1.5), ValueError),
    (lambda x, t: vocab.token_logprobs(torch.randn(2, 200), t, top_k=129), ValueError),
    (lambda x, t: vocab.token_logprobs(x), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, temperature=0.0), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, temperature=-1.0), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, temperature=9e-5), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, temperature=2e4), ValueError),
    (lambda x, t: vocab.token_logprobs(x[:1, :1].expand(2, 2 ** 30 + 1), t), ValueError),
    (lambda x, t: vocab.token_logprobs(x[:1].expand(2 ** 25, 5), t[:1].expand(2 ** 25)),
     ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, temperature=math.nan), ValueError),
    (lambda x, t: vocab.token_logprobs(x, t, temperature=math.inf), ValueError),
    (lambda x, t: vocab.topk_distill_loss(x, t, x), ValueError),
    (lambda x, t: vocab.topk_distill_loss(x, t[:, None], x), ValueError),
    (lambda x, t: vocab.topk_distill_loss(x, t[:, None], t[:, None]), TypeError),
    (lambda x, t: vocab.topk_distill_loss(x, t[:, None][:, :0], x[:, :0]), ValueError),
    (lambda x, t: vocab.topk_distill_loss(x, t[:, None].float(), x[:, :1]), TypeError),
    (lambda x, t: vocab.topk_distill_loss(x, t[:, None].expand(2, 129), x[:, :1].expand(2, 129)),
     ValueError),
    (lambda x, t: vocab.topk_distill_loss(
        x, t[:, None], x[:, :1].clone().requires_grad_(True)), ValueError),
    (lambda x, t: torch.func.vmap(lambda v: vocab.token_logprobs(v, t[0]).logprobs)(x), TypeError),
    (lambda x, t: torch.func.jvp(lambda v: vocab.token_logprobs(v, t).logprobs, (x,), (x,)),
     TypeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call(torch.randn(2, 5), torch.tensor([1, 2]))
