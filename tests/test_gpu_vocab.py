"""Vocabulary-head kernels (csrc/vocab.hip through ops/vocab.py) against the
definitions in 64 bits (tests/_vocab_oracle.py)."""
import math

import pytest
import torch

from distributed_kfac_pytorch_amd.ops import _lib, vocab
from tests import _vocab_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def logits(N, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed + V)
    return (torch.randn(N, V, device=DEV, generator=g) * scale).to(dtype)


def grads(N, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(N, device=DEV, generator=g), torch.randn(N, device=DEV, generator=g) * 0.1


def teacher(N, V, K, dtype, seed=0):
    """K different ids a row, some slots unused."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cell = max(V // K, 1)
    ids = (torch.randint(0, cell, (N, K), device=DEV, generator=g) +
           cell * torch.arange(K, device=DEV)) % V
    ids[torch.rand(N, K, device=DEV, generator=g) < 0.2] = -1
    return ids, (torch.randn(N, K, device=DEV, generator=g) * 2).to(dtype)


def check_logprobs(x, t, k, T=1.0, ignore=-100, entropy=True):
    x = x.detach().requires_grad_(True)
    N = x.shape[0]
    g, gh = grads(N)
    r = vocab.token_logprobs(x, t, top_k=k, entropy=entropy, temperature=T, ignore_index=ignore)
    o = oracle.token_logprobs(x.detach(), t, k, T, ignore, g if t is not None else None,
                              gh if entropy else None)
    outs, gs = [], []
    if t is not None:
        oracle.check('logprobs', r.logprobs, o['logprobs'])
        outs, gs = [r.logprobs], [g]
    if entropy:
        oracle.check('entropy', r.entropy, o['entropy'])
        outs, gs = outs + [r.entropy], gs + [gh]
    if k:
        oracle.check_ids(r.top_ids, o['top_ids'])
        oracle.check('top_logprobs', r.top_logprobs, o['top_logprobs'])
    if outs:
        oracle.check('dlogits', torch.autograd.grad(outs, [x], gs)[0], o['dlogits'])


def check_distill(x, ids, q, T=1.0):
    x = x.detach().requires_grad_(True)
    g, _ = grads(x.shape[0])
    loss = vocab.topk_distill_loss(x, ids, q, T)
    o = oracle.distill(x.detach(), ids, q, T, g)
    oracle.check('loss', loss, o['loss'])
    oracle.check('dlogits', torch.autograd.grad(loss, x, g)[0], o['dlogits'])


VOCABS = [1, 2, 7, 8, 9, 127, 1000, 2049, 10007, 50001, 131072, 262147]


@pytest.mark.parametrize('V', VOCABS)
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_logprobs(V, dtype):
    for N, k in ((1, min(V, 20)), (5, min(V, 128)), (3, 1)):
        t = torch.randint(0, V, (N,), device=DEV)
        t[N // 2:N // 2 + (N > 1)] = -100
        check_logprobs(logits(N, V, dtype, N), t, k, T=0.8)


@pytest.mark.parametrize('V', VOCABS)
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_distill(V, dtype):
    for N, K in ((1, 1), (6, 16), (3, 128)):
        ids, q = teacher(N, V, K, dtype, V)
        check_distill(logits(N, V, dtype, N), ids, q, T=1.7)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_many_rows(dtype):
    x = logits(700, 130, dtype)
    t = torch.randint(0, 130, (700,), device=DEV)
    t[::7] = -100
    check_logprobs(x, t, 9)
    ids, q = teacher(700, 130, 33, dtype)
    check_distill(x, ids, q)


@pytest.mark.parametrize('V', [5, 130, 4100, 70001])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_edges(V, dtype):
    names, x = oracle.edge_rows(V, dtype, DEV)
    N = len(names)
    t = (torch.arange(N, device=DEV) * 7) % V
    check_logprobs(x, t, min(V, 128))
    check_logprobs(x, None, 3)
    check_logprobs(x, t, 0, entropy=False)
    ids = torch.stack([t, (t + 2) % V, (t + V // 2) % V], 1)
    check_distill(x, ids, torch.randn(N, 3, device=DEV).to(dtype))


@pytest.mark.parametrize('V,k', [(300, 128), (4100, 128), (50001, 64), (131072, 128), (131073, 20)])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('where', ['ties', 'strided', 'run', 'end', 'nans'])
def test_alternatives_wherever_they_lie(V, k, dtype, where):
    """Top values that fall on one thread's share, in one run, at the end, or that
    are equal by the thousand."""
    for N in (1, 3):
        x = logits(N, V, dtype, scale=0.5)
        n = min(V, 3 * k)
        top = torch.linspace(20, 40, n, device=DEV).to(dtype)
        if where == 'ties':
            x = (x * 2).round()
        elif where == 'strided':
            for step in (8, 2048, 256):
                if n * step <= V:
                    x[:, 3:3 + n * step:step] = top
        elif where == 'run':
            x[:, V // 3:V // 3 + n] = top[:V - V // 3]
        elif where == 'end':
            x[:, V - n:] = top.flip(0)
        else:
            x[0, V // 2::5] = math.nan
        r = vocab.token_logprobs(x, top_k=k)
        assert torch.equal(r.top_ids, oracle.order(x)[:, :k])


def test_lengths_of_every_rest():
    """Every length around a vector, a wave and a workgroup's stride."""
    for V in list(range(1, 20)) + [63, 64, 65, 255, 256, 257, 511, 513, 1023, 1025, 2047, 2048]:
        x = logits(2, V, BF16)
        check_logprobs(x, torch.tensor([0, V - 1], device=DEV), min(V, 5))
        check_distill(x, *teacher(2, V, 3, BF16))


@pytest.mark.parametrize('layout', ['offset', 'sliced', 'every_other', 'transposed', 'expanded',
                                    'three_dims'])
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_layouts(layout, dtype):
    V = 1003
    base = logits(12, 2100, dtype)
    v = {'offset': lambda: base.flatten()[3:3 + 12 * V].view(12, V),
         'sliced': lambda: base[:, 5:5 + V],
         'every_other': lambda: base[:, ::2][:, :V],
         'transposed': lambda: logits(V, 12, dtype).t(),
         'expanded': lambda: base[:1, :V].expand(12, V),
         'three_dims': lambda: base[:, :V].view(4, 3, V).transpose(0, 1)}[layout]()
    x = v.detach().requires_grad_(True)
    t = torch.randint(0, V, v.shape[:-1] + (2,), device=DEV)[..., 0]        # strided, too
    ids = torch.randint(0, V, v.shape[:-1] + (4,), device=DEV)[..., ::2]
    q = torch.randn(v.shape[:-1] + (4,), device=DEV)[..., ::2]
    g, gh = torch.randn(2, *v.shape[:-1], device=DEV)
    r = vocab.token_logprobs(x, t, top_k=4, entropy=True)
    loss = vocab.topk_distill_loss(x, ids, q)
    d1, = torch.autograd.grad([r.logprobs, r.entropy], x, [g, gh])
    d2, = torch.autograd.grad(loss, x, g)
    flat = v.reshape(-1, V)
    o = oracle.token_logprobs(flat, t.reshape(-1), 4, g=g.reshape(-1), gh=gh.reshape(-1))
    oracle.check('logprobs', r.logprobs.reshape(-1), o['logprobs'])
    oracle.check_ids(r.top_ids.reshape(-1, 4), o['top_ids'])
    oracle.check('dlogits', d1.reshape(-1, V), o['dlogits'])
    o = oracle.distill(flat, ids.reshape(-1, 2), q.reshape(-1, 2), g=g.reshape(-1))
    oracle.check('loss', loss.reshape(-1), o['loss'])
    oracle.check('dlogits', d2.reshape(-1, V), o['dlogits'])


def test_gradients_of_means_and_parts():
    """One number expanded over the rows, a partly expanded one, and one output only."""
    x = logits(6, 301, F32).view(2, 3, 301).requires_grad_(True)
    t = torch.randint(0, 301, (2, 3), device=DEV)

    def d(f, T=1.0):
        r = vocab.token_logprobs(x, t, entropy=True, temperature=T)
        return torch.autograd.grad(f(r), x)[0].reshape(6, 301)

    def want(g, gh):
        v = [None if a is None else torch.as_tensor(a, device=DEV).float().expand(2, 3).reshape(-1)
             for a in (g, gh)]
        return oracle.token_logprobs(x.detach().reshape(6, 301), t.reshape(-1), g=v[0],
                                     gh=v[1])['dlogits']
    sixth = torch.tensor(1.0, device=DEV) / 6
    oracle.check('mean', d(lambda r: r.logprobs.mean()), want(sixth, None))
    oracle.check('sum', d(lambda r: r.entropy.sum()), want(None, 1.0))
    w = torch.tensor([[1.0], [2.0]], device=DEV)
    oracle.check('part', d(lambda r: (r.logprobs.sum(1, keepdim=True) * w).sum()), want(w, None))
    ids, q = teacher(6, 301, 5, F32)
    loss = vocab.topk_distill_loss(x, ids.view(2, 3, 5), q.view(2, 3, 5))
    got, = torch.autograd.grad(loss.mean(), x)
    oracle.check('distill', got.reshape(6, 301),
                 oracle.distill(x.detach().reshape(6, 301), ids, q, g=sixth.expand(6))['dlogits'])


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('T', [0.3, 1.0])
def test_teacher_mass_on_masked_tokens(dtype, T):
    from tests.test_vocab import masked_by_lowest
    check_distill(*masked_by_lowest(dtype, DEV), T)


def test_bad_ids_are_nan_and_stay_in_their_row():
    x = logits(5, 260, BF16).requires_grad_(True)
    t = torch.tensor([260, 3, -1, 2 ** 40, -100], device=DEV)
    r = vocab.token_logprobs(x, t, top_k=2, entropy=True)
    assert torch.isnan(r.logprobs).tolist() == [True, False, True, True, False]
    assert torch.isfinite(r.entropy).all()
    g, = torch.autograd.grad(r.logprobs.sum(), x)
    assert torch.isnan(g).all(1).tolist() == [True, False, True, True, False]
    assert torch.isfinite(g[[1, 4]]).all() and not g[4].any()
    n, i = math.nan, math.inf
    ids = torch.tensor([[0, 260], [-2, 1], [5, 5], [-1, -1], [7, 8]], device=DEV)
    q = torch.tensor([[0., 0], [0, 0], [1, 2], [n, n], [i, 0]], device=DEV)
    loss = vocab.topk_distill_loss(x, ids, q)
    assert torch.isnan(loss).tolist() == [True, True, False, False, True]
    g, = torch.autograd.grad(loss.sum(), x)
    o = oracle.distill(x.detach(), ids, q, g=torch.ones(5))
    oracle.check('loss', loss, o['loss'])
    oracle.check('dlogits', g, o['dlogits'])


def test_same_id_in_every_slot():
    for K in (2, 64, 128):
        x = logits(3, 500, F32)
        ids = torch.full((3, K), 77, device=DEV)
        ids[1, K // 2:] = 499
        check_distill(x, ids, torch.randn(3, K, device=DEV))


def test_rows_that_are_skipped_are_not_read():
    x = logits(4, 333, F32)
    x[1] = math.nan
    t = torch.tensor([1, -100, 2, 3], device=DEV)
    x.requires_grad_(True)
    r = vocab.token_logprobs(x, t, top_k=3, entropy=True)
    assert r.logprobs[1] == 0 and r.entropy[1] == 0 and r.top_ids[1].tolist() == [-1] * 3
    assert (r.top_logprobs[1] == -math.inf).all()
    assert not torch.autograd.grad((r.logprobs + r.entropy).sum(), x)[0][1].any()
    ids = torch.tensor([[1, 2], [-1, -1], [3, 4], [5, -1]], device=DEV)
    loss = vocab.topk_distill_loss(x, ids, torch.randn(4, 2, device=DEV))
    assert loss[1] == 0 and torch.isfinite(loss).all()
    assert not torch.autograd.grad(loss.sum(), x)[0][1].any()


@pytest.mark.parametrize('T', [1e-4, 1e-2, 50.0, 1e4])
def test_temperatures(T):
    x = logits(4, 777, F32)
    t = x.argmax(1)
    r = vocab.token_logprobs(x, t, top_k=2, entropy=True, temperature=T)
    o = oracle.token_logprobs(x, t, 2, T)
    oracle.check('logprobs', r.logprobs, o['logprobs'])
    oracle.check('entropy', r.entropy, o['entropy'])
    oracle.check('top_logprobs', r.top_logprobs, o['top_logprobs'])
    ids, q = teacher(4, 777, 5, F32)
    check_distill(x, ids, q, T)


def test_cpu_and_gpu_agree():
    """The same calls on both devices, defined edges among them."""
    names, x = oracle.edge_rows(130, F32)
    t = torch.arange(len(names)) % 130
    t[3] = -100
    a = vocab.token_logprobs(x, t, top_k=7, entropy=True)
    b = vocab.token_logprobs(x.to(DEV), t.to(DEV), top_k=7, entropy=True)
    assert torch.equal(a.top_ids, b.top_ids.cpu())
    for u, v in zip(a[:3], b[:3]):
        assert torch.allclose(u, v.cpu(), rtol=1e-5, atol=1e-5, equal_nan=True)


@pytest.mark.parametrize('N,V,dtype', [(3, 131072, BF16), (64, 10000, F32), (700, 1003, F16)])
def test_bitwise_repeatable_and_captured(N, V, dtype):
    """Twice the same bits, on another stream too; a captured step replays them
    for new inputs, with eager work between the replays."""
    t = torch.randint(0, V, (N,), device=DEV)
    t[0] = -100
    ids, q = teacher(N, V, 40, dtype)
    g, gh = grads(N)

    def step(x):
        x = x.detach().requires_grad_(True)
        r = vocab.token_logprobs(x, t, top_k=40, entropy=True)
        loss = vocab.topk_distill_loss(x, ids, q, 1.5)
        return tuple(v.detach() for v in r) + (loss.detach(),) + \
            torch.autograd.grad([r.logprobs, r.entropy], x, [g, gh]) + \
            torch.autograd.grad(loss, x, g)
    x = logits(N, V, dtype)
    first = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs)
    for k in range(3):
        xs.copy_(logits(N, V, dtype, 10 + k))
        ref = step(xs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), k


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_rows_past_32_bits(dtype):
    """Offsets of the last rows pass 2^32 bytes and 2^31 elements."""
    V, N = 131072, 16400
    x = torch.zeros(N, V, dtype=dtype, device=DEV)
    x[-1] = logits(1, V, dtype)[0]
    x[-2, 5] = 3.0
    t = torch.full((N,), -100, device=DEV)
    t[-2:] = torch.tensor([5, 77])
    x.requires_grad_(True)
    r = vocab.token_logprobs(x, t, top_k=4, entropy=True)
    o = oracle.token_logprobs(x.detach()[-2:], t[-2:], 4, g=torch.ones(2))
    oracle.check('logprobs', r.logprobs[-2:], o['logprobs'])
    oracle.check('entropy', r.entropy[-2:], o['entropy'])
    oracle.check_ids(r.top_ids[-2:], o['top_ids'])
    d, = torch.autograd.grad(r.logprobs.sum(), x)
    oracle.check('dlogits', d[-2:], o['dlogits'])
    assert not d[:3].any()
    del d, r
    ids = torch.full((N, 2), -1, device=DEV)
    ids[-2:] = torch.tensor([[5, 7], [V - 1, 0]])
    q = torch.tensor([[1.0, 0.5]], device=DEV).expand(N, 2)
    loss = vocab.topk_distill_loss(x, ids, q)
    o = oracle.distill(x.detach()[-2:], ids[-2:], q[-2:], g=torch.ones(2))
    oracle.check('loss', loss[-2:], o['loss'])
    d, = torch.autograd.grad(loss.sum(), x)
    oracle.check('dlogits', d[-2:], o['dlogits'])
    assert not d[:3].any()


def test_difference_quotient():
    """Along a direction, against the functions' own values: fp32 values of 50 rows
    are off by about 1e-6 each, over a step of 2^-5; the third derivative's h^2 is
    of the same size."""
    x, v = logits(50, 400, F32), logits(50, 400, F32, 9, 1.0)
    t = torch.randint(0, 400, (50,), device=DEV)
    ids, q = teacher(50, 400, 8, F32)
    h = 2.0 ** -5

    def f(x):
        r = vocab.token_logprobs(x, t, entropy=True)
        return r.logprobs.double().sum() + 0.3 * r.entropy.double().sum() + \
            vocab.topk_distill_loss(x, ids, q).double().sum()
    xg = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(f(xg), xg)
    slope = (g.double() * v.double()).sum()
    diff = (f(x + h * v) - f(x - h * v)) / (2 * h)
    assert abs(float(diff - slope)) < 2e-3 * float(g.double().norm() * v.double().norm())


def test_refusals_on_the_gpu():
    x, t = logits(2, 9, F32), torch.tensor([1, 2], device=DEV)
    with pytest.raises(TypeError):
        vocab.token_logprobs(x.double(), t)
    with pytest.raises(ValueError):
        vocab.token_logprobs(x, t.cpu())
    with pytest.raises(ValueError):
        vocab.topk_distill_loss(x, t[:, None].cpu(), x[:, :1])
    with pytest.raises(ValueError):
        vocab.topk_distill_loss(x, t[:, None], x[:, :1].cpu())
    assert _lib.lib().kfac_vocab_top_max() == vocab.TOP_MAX


def test_no_rows_on_the_gpu():
    x = torch.empty(0, 5, device=DEV, requires_grad=True)
    r = vocab.token_logprobs(x, torch.empty(0, dtype=torch.long, device=DEV), top_k=2,
                             entropy=True)
    loss = vocab.topk_distill_loss(x, torch.empty(0, 3, dtype=torch.long, device=DEV),
                                   torch.empty(0, 3, device=DEV))
    g, = torch.autograd.grad((r.logprobs + r.entropy + loss).sum(), x)
    assert g.shape == (0, 5) and r.top_ids.shape == (0, 2)


def test_without_a_graph_the_same_values():
    x = logits(9, 2003, BF16)
    t = torch.randint(0, 2003, (9,), device=DEV)
    ids, q = teacher(9, 2003, 7, F32)
    a = vocab.token_logprobs(x, t, top_k=3, entropy=True)
    la = vocab.topk_distill_loss(x, ids, q)
    x.requires_grad_(True)
    b = vocab.token_logprobs(x, t, top_k=3, entropy=True)
    lb = vocab.topk_distill_loss(x, ids, q)
    assert b.logprobs.requires_grad and lb.requires_grad and not la.requires_grad
    assert all(torch.equal(u, v) for u, v in zip(a, b)) and torch.equal(la, lb)


def test_checkpointed_and_repeated_backward():
    """Recomputed in a checkpoint, and twice from one graph: the same gradient."""
    from torch.utils.checkpoint import checkpoint
    head = torch.nn.Linear(16, 700, device=DEV)
    h = torch.randn(6, 16, device=DEV)
    t = torch.randint(0, 700, (6,), device=DEV)
    ids, q = teacher(6, 700, 5, F32)

    def f(h):
        x = head(h)
        r = vocab.token_logprobs(x, t, entropy=True)
        return (vocab.topk_distill_loss(x, ids, q) - r.logprobs - 0.1 * r.entropy).sum()
    loss = f(h)
    a = torch.autograd.grad(loss, head.weight, retain_graph=True)[0]
    b = torch.autograd.grad(loss, head.weight)[0]
    c = torch.autograd.grad(checkpoint(f, h, use_reentrant=False), head.weight)[0]
    assert torch.equal(a, b) and torch.equal(a, c)


def test_second_derivatives_are_errors():
    x = logits(2, 50, F32).requires_grad_(True)
    r = vocab.token_logprobs(x, torch.tensor([1, 2], device=DEV), entropy=True)
    loss = vocab.topk_distill_loss(x, torch.tensor([[1], [2]], device=DEV), x.detach()[:, :1])
    for out in (r.logprobs, r.entropy, loss):
        g, = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_saved_inputs_are_guarded():
    """Logits or targets written over before the backward pass are an error; a
    teacher written over changes nothing (its masses were kept)."""
    t = torch.tensor([1, 2], device=DEV)
    base = logits(2, 50, F32).requires_grad_(True)
    x = base * 1
    lp = vocab.token_logprobs(x, t).logprobs
    t.add_(1)
    with pytest.raises(RuntimeError):
        lp.sum().backward()
    lp = vocab.token_logprobs(x, t).logprobs
    x.detach().mul_(2)
    with pytest.raises(RuntimeError):
        lp.sum().backward()
    x = base * 1
    ids, q = teacher(2, 50, 4, F32)
    o = oracle.distill(x.detach(), ids, q, g=torch.ones(2))
    loss = vocab.topk_distill_loss(x, ids, q)
    ids.fill_(-1)
    q.zero_()
    oracle.check('dlogits', torch.autograd.grad(loss.sum(), x)[0], o['dlogits'])


def test_runs_in_fp16_training():
    """Autocast and a scaled loss: fp16 logits, gradients in fp16."""
    head = torch.nn.Linear(32, 500).to(DEV)
    h = torch.randn(20, 32, device=DEV)
    t = torch.randint(0, 500, (20,), device=DEV)
    with torch.autocast('cuda', dtype=F16):
        x = head(h)
        r = vocab.token_logprobs(x, t, entropy=True)
    assert x.dtype == F16 and r.logprobs.dtype == F32
    (-1024 * r.logprobs.mean()).backward()
    assert head.weight.grad.dtype == F32 and torch.isfinite(head.weight.grad).all()
    assert head.weight.grad.any()
