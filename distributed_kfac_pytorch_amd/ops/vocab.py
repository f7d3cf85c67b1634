"""Operators behind a vocabulary head (csrc/vocab.hip): what the language models
(models/transformer_lm.py, models/lstm_lm.py) are evaluated with and distilled by.

token_logprobs     log probabilities of given tokens, with the distribution's
                   entropy and its top alternatives; gradients for the log
                   probability and the entropy
topk_distill_loss  Kullback-Leibler divergence of a student from a teacher of
                   which only the top logits are known -- the ids and values
                   that token_logprobs(top_k=...) gives for the teacher

Logits are (..., V) of fp32, bf16 or fp16 (fp64 too on the CPU), any strides;
everything is computed and returned in fp32 (fp64 for fp64), the gradient in
the logits' type.  GPU tensors run on the HIP kernels (hipGraph-capturable,
bitwise reproducible, no host synchronisation; the autograd nodes are C++,
csrc/torch_ops.cpp), CPU tensors on the same formulas in torch; so does a call under
a dispatch mode (a FLOP counter, selective checkpointing) or a compiler, which have
to see operations.  Neither op has a second derivative.

What a kernel meets on the device cannot raise without a synchronisation: a
target out of range makes its row's log probability and that one's gradient NaN,
a teacher's id out of range its row's loss and gradient.
"""
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ['token_logprobs', 'topk_distill_loss', 'TokenLogprobs', 'TOP_MAX']

# most alternatives a row, and most slots of a teacher's row (csrc/vocab.hip)
TOP_MAX = 128

_GPU_TYPES = (torch.float32, torch.bfloat16, torch.float16)


class TokenLogprobs(NamedTuple):
    """Results of token_logprobs; None for what was not asked for."""
    logprobs: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _check(name, logits, temperature):
    if not isinstance(logits, torch.Tensor) or not logits.dtype.is_floating_point:
        raise TypeError('{}: logits must be a floating point tensor'.format(name))
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError('{}: logits must be (..., V) with V >= 1, got shape {}'.format(
            name, tuple(logits.shape)))
    if logits.is_cuda and logits.dtype not in _GPU_TYPES:
        raise TypeError('{}: GPU logits must be fp32, bf16 or fp16, got {}'.format(
            name, logits.dtype))
    V = logits.shape[-1]
    rows = logits.numel() // V
    if V > 2 ** 30 or rows >= 2 ** 25 or rows * -(-V // 4096) >= 2 ** 31:
        raise ValueError('{}: logits of shape {} are too many rows or columns'.format(
            name, tuple(logits.shape)))
    temperature = float(temperature)
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError('{}: temperature must be in [1e-4, 1e4], got {}'.format(
            name, temperature))
    return 1.0 / temperature


def _check_ids(name, what, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise TypeError('{}: {} must be an int64 or int32 tensor'.format(name, what))
    if t.shape != shape:
        raise ValueError('{}: {} must have shape {}, got {}'.format(
            name, what, tuple(shape), tuple(t.shape)))
    if t.device != device:
        raise ValueError('{}: {} is on {}, the logits are on {}'.format(
            name, what, t.device, device))


def _native(name, *tensors):
    """Whether the kernels run: the formulas below do elsewhere."""
    if _lib.plain_tensors(*tensors):
        return _lib.use_native(tensors[0])
    if not _lib.watched_tensors(*tensors):
        raise TypeError('{}: takes ordinary tensors, outside functorch transforms, forward-mode '
                        'levels and traces'.format(name))
    return False


# ------------------------------------------------ CPU tensors, modes: the formulas
def _cpu_stats(x, inv_t):
    """(x as computed in, M, L, lp): csrc/vocab.hip's names."""
    x = x if x.dtype == torch.float64 else x.float()
    M = x.amax(-1)
    dead = M == -math.inf
    d = (x - M.masked_fill(dead, 0.0)[:, None]) * inv_t
    L = d.exp().sum(-1).log()
    L = torch.where(torch.isnan(x).any(-1), math.nan, L)
    return x, M, L, (d - L[:, None]).masked_fill(dead[:, None], -math.inf)


def _gather(lp, ids):
    """lp at ids; NaN where an id is out of range."""
    bad = (ids < 0) | (ids >= lp.shape[1])
    return lp.gather(1, ids.masked_fill(bad, 0)).masked_fill(bad, math.nan)


def _cpu_entropy(lp, dead):
    p = lp.exp()
    h = -torch.where(p == 0, 0.0, p * lp).sum(-1)
    return torch.where(dead, torch.zeros_like(h), h)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, k, entropy, inv_t, ignore):
        shape = logits.shape[:-1]
        rows = logits.reshape(-1, logits.shape[-1])
        x, M, _, lp = _cpu_stats(rows, inv_t)
        skip = torch.zeros(len(x), dtype=torch.bool, device=x.device) if targets is None else \
            targets.reshape(-1) == ignore
        ctx.inv_t, ctx.skip = inv_t, skip
        ctx.set_materialize_grads(False)
        score = h = tl = ti = None
        if targets is not None:
            targets = targets.reshape(-1, 1).to(torch.int64).masked_fill(skip[:, None], 0)
            score = torch.where(skip, 0.0, _gather(lp, targets)[:, 0]).view(shape)
        if entropy:
            h = torch.where(skip, 0.0, _cpu_entropy(lp, M == -math.inf)).view(shape)
        if k:
            # stable, so that equal values keep the order of their indices; a device's sort
            # may tell zeros and NaN apart by their signs
            key = torch.where(torch.isnan(x), math.nan, x + 0.0)
            ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k]
            ti = ids.masked_fill(skip[:, None], -1).view(shape + (k,))
            tl = lp.gather(1, ids).masked_fill(skip[:, None], -math.inf).view(shape + (k,))
            ctx.mark_non_differentiable(tl, ti)
        ctx.save_for_backward(logits, targets, h)
        return score, h, tl, ti

    @staticmethod
    @once_differentiable
    def backward(ctx, g, gh, _tl, _ti):
        logits, targets, h = ctx.saved_tensors
        if g is None and gh is None:
            return (None,) * 6
        V = logits.shape[-1]
        _, M, _, lp = _cpu_stats(logits.reshape(-1, V), ctx.inv_t)
        p = lp.exp()
        d = torch.zeros_like(p)
        if g is not None:
            bad = (targets < 0) | (targets >= V)
            g = g.reshape(-1, 1).to(p.dtype)
            d = (-p * g).scatter_add_(1, targets.masked_fill(bad, 0), g)
            d = torch.where(bad, math.nan, d)
        if gh is not None:
            d = d - gh.reshape(-1, 1) * torch.where(p == 0, 0.0, p * (lp + h.reshape(-1, 1)))
        zero = ctx.skip | (M == -math.inf)
        d = torch.where(zero[:, None], 0.0, d * ctx.inv_t)
        return d.to(logits.dtype).view(logits.shape), None, None, None, None, None


def token_logprobs(logits, targets=None, top_k=0, entropy=False, temperature=1.0,
                   ignore_index=-100):
    """Log probabilities of `targets` under softmax(logits / temperature).

    Args:
      logits: (..., V).
      targets: integer ids of shape (...), or None (alternatives / entropy only).
      top_k: alternatives a row, at most min(V, TOP_MAX): ids by falling logit,
        ties to the lower id, NaN above every number.
      entropy: also return the entropy of softmax(logits / temperature), in nats.
      ignore_index: rows with this target are skipped (their logits are not
        read): logprob and entropy 0, top_ids -1, top_logprobs -inf, gradient 0.

    Returns TokenLogprobs(logprobs (...), entropy (...), top_logprobs (..., k),
    top_ids (..., k) int64).  logprobs and entropy have gradients (to the
    logits); the alternatives do not.

    A row of only -inf (everything masked) has log probabilities -inf, entropy
    0 and no gradient.  NaN or +inf in a row, also beside nothing but -inf or
    NaN, makes its results and its gradient NaN.
    """
    inv_t = _check('token_logprobs', logits, temperature)
    if targets is not None:
        _check_ids('token_logprobs', 'targets', targets, logits.shape[:-1], logits.device)
    k = int(top_k)
    if k != top_k or not 0 <= k <= min(TOP_MAX, logits.shape[-1]):
        raise ValueError('token_logprobs: top_k must be 0 .. {}, got {}'.format(
            min(TOP_MAX, logits.shape[-1]), top_k))
    if targets is None and not k and not entropy:
        raise ValueError('token_logprobs: nothing asked for (no targets, top_k 0, no entropy)')
    call = _lib.torch_ops().token_logprobs.default if _native('token_logprobs', logits, targets) \
        else _TokenLogprobs.apply
    return TokenLogprobs(*call(logits, targets, k, bool(entropy), inv_t, int(ignore_index)))


def _cpu_teacher(ids, teacher, V, inv_t, dtype):
    """(some used slot, id or 0, q, log q) of rows of slots; bad ids make q NaN."""
    t = teacher.to(dtype).masked_fill(ids == -1, -math.inf)
    t = t.masked_fill((ids < -1) | (ids >= V), math.nan)
    some = ~(t == -math.inf).all(1)
    top = torch.where(some, t.amax(1), torch.zeros((), dtype=dtype))[:, None]
    d = (t - top) * inv_t
    Z = d.exp().sum(1, keepdim=True)
    return some, ids.clamp(0, V - 1), d.exp() / Z, d - Z.log()


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, inv_t):
        V, K = logits.shape[-1], ids.shape[-1]
        x, M, L, _ = _cpu_stats(logits.reshape(-1, V), inv_t)
        ctx.inv_t = inv_t
        ctx.save_for_backward(logits, ids, teacher)
        some, at, q, logq = _cpu_teacher(ids.reshape(-1, K), teacher.reshape(-1, K), V, inv_t,
                                         x.dtype)
        # q (log q - lp), q taken into lp's product first: csrc/vocab.hip's distill_row
        dead = (M == -math.inf)[:, None]
        c = torch.where(dead, -math.inf, x.gather(1, at) - M[:, None])
        each = q * (logq + torch.where(dead, 0.0, L[:, None])) - q * c * inv_t
        each = torch.where(q == 0, 0.0, each)
        return torch.where(some, each.sum(1), 0.0).view(logits.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, ids, teacher = ctx.saved_tensors
        V, K = logits.shape[-1], ids.shape[-1]
        _, M, _, lp = _cpu_stats(logits.reshape(-1, V), ctx.inv_t)
        some, at, q, _ = _cpu_teacher(ids.reshape(-1, K), teacher.reshape(-1, K), V, ctx.inv_t,
                                      lp.dtype)
        bad = torch.where(torch.isnan(q).any(1, keepdim=True), math.nan, 1.0).to(lp.dtype)
        d = (lp.exp() * bad).scatter_add_(1, at, -q) * (g.reshape(-1, 1) * ctx.inv_t)
        d = torch.where((some & (M != -math.inf))[:, None], d, 0.0)
        return d.to(logits.dtype).view(logits.shape), None, None, None


def topk_distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0):
    """Distillation from a teacher's top logits: for each row

        sum_j q_j (log q_j - log softmax(logits / T)[id_j]),
        q = softmax(teacher_logits / T) over the row's K alternatives

    -- the divergence of the student's whole distribution from the teacher's,
    renormalised over the alternatives that are known.

    Args:
      logits: (..., V), the student's.
      teacher_ids: (..., K) integer ids, K <= TOP_MAX; -1 marks an unused slot
        (rows of different length, rows to be skipped).  An id that occurs
        twice has both masses.
      teacher_logits: (..., K) logits or log probabilities of these ids (a
        constant added to a row changes nothing); a -inf has no mass.  They
        are constants: a teacher that requires a gradient is refused.
      temperature: T, of both sides.  The loss is not multiplied by T^2.

    Returns the losses, of shape (...).  A row without mass (every slot unused
    or -inf) has loss 0 and no gradient; a student that gives one of the
    teacher's ids no probability has loss +inf.
    """
    name = 'topk_distill_loss'
    inv_t = _check(name, logits, temperature)
    if not isinstance(teacher_ids, torch.Tensor) or teacher_ids.dim() < 1 or \
            not 1 <= teacher_ids.shape[-1] <= TOP_MAX:
        raise ValueError('{}: teacher_ids must be (..., K) with K in 1 .. {}'.format(
            name, TOP_MAX))
    shape = logits.shape[:-1] + teacher_ids.shape[-1:]
    _check_ids(name, 'teacher_ids', teacher_ids, shape, logits.device)
    if not isinstance(teacher_logits, torch.Tensor) or \
            teacher_logits.dtype not in _GPU_TYPES + (torch.float64,):
        raise TypeError('{}: teacher_logits must be a floating point tensor'.format(name))
    if teacher_logits.shape != shape or teacher_logits.device != logits.device:
        raise ValueError('{}: teacher_logits must have shape {} on {}, got {} on {}'.format(
            name, tuple(shape), logits.device, tuple(teacher_logits.shape),
            teacher_logits.device))
    if teacher_logits.requires_grad:
        raise ValueError('{}: the teacher is a constant; detach teacher_logits'.format(name))
    if logits.is_cuda and teacher_logits.dtype == torch.float64:
        teacher_logits = teacher_logits.float()
    if _native(name, logits, teacher_ids, teacher_logits):
        return _lib.torch_ops().topk_distill.default(logits, teacher_ids, teacher_logits, inv_t)
    return _TopkDistill.apply(logits, teacher_ids.to(torch.int64), teacher_logits, inv_t)
