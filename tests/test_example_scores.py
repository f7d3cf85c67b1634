"""The language-model example's validation loss and, with a teacher, its training
loss come from ops.vocab; they are torch's cross entropy."""
import pytest
import torch
import torch.nn.functional as F

from examples import torch_language_model as ex
from examples.rnn_utils.utils import Corpus, batchify, bptt_batches

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.mark.parametrize('device', DEVICES)
def test_score_is_cross_entropy(device):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4, 7, 50, generator=g).to(device).requires_grad_(True)
    out = x.transpose(0, 1)                              # as the Transformer LM's run_model has it
    t = torch.randint(0, 50, (28,), generator=g).to(device)
    nll = -ex.score(out, t).logprobs.mean()
    ce = F.cross_entropy(out.reshape(-1, 50), t)
    assert abs(float(nll - ce)) < 1e-5
    a, = torch.autograd.grad(nll, x)
    b, = torch.autograd.grad(ce, x)
    assert float((a - b).abs().max()) < 1e-7


@pytest.mark.parametrize('model', ['lstm', 'transformer'])
@pytest.mark.parametrize('device', DEVICES)
def test_validation_loss_of_the_saved_model(model, device, tmp_path):
    path = str(tmp_path / 'lm.pt')
    argv = ['--model', model, '--epochs', '1', '--synthetic-tokens', '1200', '--vocab', '100',
            '--emsize', '32', '--nhid', '32', '--nlayers', '1', '--nheads', '4',
            '--batch-size', '4', '--bptt', '12', '--save', path] + \
        (['--no-cuda'] if device == 'cpu' else [])
    val_loss = ex.main(argv)[0]['val_loss']
    args = ex.parse(argv)
    corpus = Corpus(args.data_dir, args.dataset, args.synthetic_tokens, args.vocab, seed=args.seed)
    val = batchify(corpus.valid, args.eval_batch_size).to(device)
    lm = ex.build_model(args, corpus.ntokens, args.emsize, args.nhid, args.nlayers).to(device)
    lm.load_state_dict(torch.load(path, weights_only=True))
    lm.eval()
    losses, hidden = [], lm.init_hidden(val.size(1)) if model == 'lstm' else None
    with torch.no_grad():
        for i in bptt_batches(val, args.bptt):
            data, targets = ex.get_batch(val, i, args.bptt)
            out, hidden = ex.run_model(lm, data, hidden, args)
            losses.append(float(F.cross_entropy(out.reshape(-1, out.size(-1)), targets)))
    assert abs(val_loss - sum(losses) / len(losses)) < 1e-4
