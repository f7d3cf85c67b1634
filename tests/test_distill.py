"""A teacher's alternatives, a student's loss on them, its layer norms and a K-FAC
step, run together: the language-model example and the bare training step."""
import pytest
import torch
import torch.nn.functional as F

import distributed_kfac_pytorch_amd as kfac
from distributed_kfac_pytorch_amd.models import TransformerLM
from distributed_kfac_pytorch_amd.ops import vocab

V, T = 64, 2.0


def _models(device):
    torch.manual_seed(0)
    teacher = TransformerLM(V, d_model=48, n_layers=2, n_heads=4, d_ff=96, max_len=16)
    student = TransformerLM(V, d_model=32, n_layers=2, n_heads=4, d_ff=64, max_len=16)
    return teacher.to(device).eval().requires_grad_(False), student.to(device)


def _loss(teacher, student, tokens, targets):
    with torch.no_grad():
        top = vocab.token_logprobs(teacher(tokens), targets, top_k=8)
    out = student(tokens)
    r = vocab.token_logprobs(out, targets, entropy=True)
    kd = vocab.topk_distill_loss(out, top.top_ids, top.top_logprobs, T)
    live = (targets != -100).sum()
    return (T * T * kd.sum() - 0.5 * r.logprobs.sum() - 0.01 * r.entropy.sum()) / live


def _plain_loss(teacher, student, tokens, targets):
    """The same from torch's operations."""
    lt, out = F.log_softmax(teacher(tokens), -1), student(tokens)
    tv, ti = lt.topk(8, -1)
    q = F.log_softmax(tv / T, -1)
    live = (targets != -100).float()
    kd = (q.exp() * (q - F.log_softmax(out / T, -1).gather(-1, ti))).sum(-1)
    lp = F.log_softmax(out, -1)
    ce = -lp.gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    ent = -(lp.exp() * lp).sum(-1)
    return ((T * T * kd + 0.5 * ce - 0.01 * ent) * live).sum() / live.sum()


def _batch(step, device):
    g = torch.Generator().manual_seed(step)
    tokens = torch.randint(0, V, (4, 12), generator=g)
    targets = torch.randint(0, V, (4, 12), generator=g)
    targets[1, 7:] = -100                        # a padded sequence
    targets[3] = -100                            # an empty one
    return tokens.to(device), targets.to(device)


def _step_grads(device, steps=2):
    teacher, student = _models(device)
    pre = kfac.KFAC(student, factor_update_freq=1, inv_update_freq=1, lr=0.1, damping=0.003,
                    skip_layers=['embedding'], batch_first=False, use_hip_graphs=False)
    opt = torch.optim.SGD(student.parameters(), lr=0.1)
    raw, done = [], []
    for k in range(steps):
        opt.zero_grad()
        _loss(teacher, student, *_batch(k, device)).backward()
        raw.append([p.grad.cpu().clone() for p in student.parameters()])
        pre.step()
        done.append([p.grad.cpu().clone() for p in student.parameters()])
        opt.step()
    return raw, done


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_gradient_is_torchs(device):
    teacher, student = _models(device)
    batch = _batch(0, device)
    loss, ref = _loss(teacher, student, *batch), _plain_loss(teacher, student, *batch)
    assert abs(float(loss - ref)) < 1e-5 * abs(float(ref))
    g = torch.autograd.grad(loss, list(student.parameters()))
    r = torch.autograd.grad(ref, list(student.parameters()))
    # fp32 through two blocks: some hundred roundings of 6e-8 each
    for a, b in zip(g, r):
        assert float((a - b).norm()) < 1e-4 * max(float(b.norm()), 1e-3)


@pytest.mark.gpu
def test_distilled_kfac_step_gpu_matches_cpu():
    """Raw gradients to fp32 accuracy; the preconditioned ones within the band that
    tests/test_gpu_models.py has for an eigendecomposition in fp32."""
    cpu, gpu = _step_grads('cpu'), _step_grads('cuda')
    for a, b in zip(gpu[0][0], cpu[0][0]):
        assert float((a - b).norm()) < 1e-4 * max(float(b.norm()), 1e-3)
    for k, (gs, cs) in enumerate(zip(gpu[1], cpu[1])):
        for a, b in zip(gs, cs):
            assert float((a - b).norm() / b.norm().clamp_min(1e-12)) < 5e-3 * 10 ** k


@pytest.mark.gpu
def test_captured_training_step():
    """The whole step in a hipGraph, replayed between eager steps on other data."""
    teacher, student = _models('cuda')
    tokens, targets = _batch(0, 'cuda')
    params = list(student.parameters())

    def grads(tokens, targets):
        loss = _loss(teacher, student, tokens, targets)
        return [loss.detach()] + list(torch.autograd.grad(loss, params))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(tokens, targets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads(tokens, targets)
    for k in range(1, 4):
        new = _batch(k, 'cuda')
        ref = grads(*new)
        tokens.copy_(new[0])
        targets.copy_(new[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, ref):
            assert float((a - b).norm()) <= 1e-5 * max(float(b.norm()), 1e-3)


@pytest.mark.parametrize('model', ['lstm', 'transformer'])
@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_language_model_example_distils(model, device, tmp_path):
    from examples import torch_language_model as ex
    path = str(tmp_path / 'teacher.pt')
    argv = ['--model', model, '--epochs', '1', '--synthetic-tokens', '1200', '--vocab', '100',
            '--emsize', '32', '--nhid', '32', '--nlayers', '2', '--nheads', '4',
            '--batch-size', '4', '--bptt', '12'] + (['--no-cuda'] if device == 'cpu' else [])
    ex.main(argv + ['--save', path])
    argv[argv.index('--nlayers') + 1] = '1'
    hist = ex.main(argv + ['--teacher', path, '--teacher-nlayers', '2', '--distill-topk', '5'])
    assert hist[0]['train_loss'] > 0 and 0 <= hist[0]['val_top1'] <= 1
    assert 0 < hist[0]['val_entropy'] < 4.7                      # log 100 is 4.6
