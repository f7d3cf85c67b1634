"""More vocabulary rows than one launch takes (fewer than 2^32 threads): the ranges
are seen to be seamless, since every row has the bits that it has in a smaller call."""
import pytest
import torch

from distributed_kfac_pytorch_amd.ops import vocab

pytestmark = pytest.mark.gpu

DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
GROUPS = 1 << 22                      # csrc/vocab.hip MAX_GROUPS


def randn(shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


def pieces(N):
    """Two smaller calls, neither of which is cut where the whole is."""
    return [slice(0, N // 2), slice(N // 2, N)]


# 2^24 rows of 256 threads are 2^32 of them
@pytest.mark.parametrize('N,V,k,dtype', [(GROUPS + 5, 8, 0, F16), (GROUPS + 5, 9, 2, F32),
                                         (GROUPS + 77, 40, 33, BF16), (2 ** 24 + 3, 64, 0, F16)])
def test_many_vocabulary_rows(N, V, k, dtype):
    x = randn((N, V), dtype)
    t = torch.arange(N, device=DEV) % V
    t[::3] = -100
    g = randn(N, F32, 2)

    def run(s):
        y = x[s].detach().requires_grad_(True)
        r = vocab.token_logprobs(y, t[s], top_k=k, entropy=True)
        d, = torch.autograd.grad([r.logprobs, r.entropy], [y], [g[s], g[s]])
        return [v.detach() for v in (r.logprobs, r.entropy, d, r.top_logprobs, r.top_ids)
                if v is not None]
    whole = run(slice(0, N))
    for s in pieces(N):
        for a, b in zip(whole, run(s)):
            assert torch.equal(a[s], b)
    # a few rows against log_softmax; |lp| < 16 in roundings of 2^-21, one more a term
    at = torch.tensor([1, GROUPS - 1, GROUPS, GROUPS + 1, N - 1], device=DEV)
    lp = torch.log_softmax(x[at].double(), -1)
    want = torch.where(t[at] == -100, 0.0, lp.gather(1, t[at].clamp(min=0)[:, None])[:, 0])
    assert float((whole[0][at] - want).abs().max()) < 8 * 2.0 ** -20


@pytest.mark.parametrize('N,V,K,dtype', [(GROUPS + 5, 8, 3, BF16), (GROUPS + 5, 11, 1, F32)])
def test_many_rows_of_a_teacher(N, V, K, dtype):
    x = randn((N, V), dtype)
    ids = (torch.arange(N, device=DEV)[:, None] * 5 + torch.arange(K, device=DEV) * 3) % V
    ids[::7] = -1
    q, g = randn((N, K), dtype, 3), randn(N, F32, 2)

    def run(s):
        y = x[s].detach().requires_grad_(True)
        loss = vocab.topk_distill_loss(y, ids[s], q[s], 2.0)
        return loss.detach(), torch.autograd.grad(loss, y, g[s])[0]
    whole = run(slice(0, N))
    assert bool(whole[0][-1] != 0) and not whole[0][::7].any()
    for s in pieces(N):
        for a, b in zip(whole, run(s)):
            assert torch.equal(a[s], b)


def test_many_rows_of_a_long_vocabulary_cut_the_gradient():
    """More workgroups than rows: every row's gradient is cut into 25."""
    N, V = GROUPS // 25 + 11, 100001
    x = randn((7, V), BF16).expand(N // 7 + 1, 7, V).reshape(-1, V)[:N].requires_grad_(True)
    t = torch.arange(N, device=DEV) % 7                  # a row and its copies have one target
    lp = vocab.token_logprobs(x, t).logprobs
    d, = torch.autograd.grad(lp.sum(), x)
    d, lp = d[:N // 7 * 7].view(-1, 7, V), lp[:N // 7 * 7].view(-1, 7)
    assert torch.equal(lp, lp[:1].expand_as(lp))
    for k in range(0, len(d), 1000):
        assert torch.equal(d[k:k + 1000], d[:1].expand_as(d[k:k + 1000]))
    assert torch.equal(d[-1], d[0])
