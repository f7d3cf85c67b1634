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
bitwise reproducible, no host synchronisation), CPU tensors on the same
formulas in torch.  Neither op has a second derivative.

What a kernel meets on the device cannot raise without a synchronisation: a
target or id out of range makes its row's results and gradient NaN.
"""
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ['token_logprobs', 'topk_distill_loss', 'TokenLogprobs', 'TOP_MAX']

# most alternatives a row, and most slots of a teacher's row (csrc/vocab.hip)
TOP_MAX = 128

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # csrc/common.h
_GPU_TYPES = tuple(_CODE)

# csrc/vocab.hip KfacVocabFwd, KfacVocabBwd
_fwd = _lib.PackedCall('kfac_vocab_forward', '13P4q5if0P')
_bwd = _lib.PackedCall('kfac_vocab_backward', '9P6q2if0P')


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


def _check_plain(name, *tensors):
    if not _lib.plain_tensors(*tensors):
        raise TypeError('{}: takes ordinary tensors, outside functorch transforms, forward-mode '
                        'levels, dispatch modes and traces'.format(name))


def _rows(t, rows, V):
    """(t as (rows, V) with contiguous rows, the distance between rows)."""
    if t.is_contiguous():
        return t, V
    t = t.reshape(rows, V)
    if V > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _row_grad(g):
    """(g or a copy of it, its address, the distance between its rows): the
    gradient of a mean or sum is one number expanded (distance 0)."""
    if g is None:
        return None, 0, 0
    if g.is_contiguous():
        return g, g.data_ptr(), 1
    if not any(g.stride()):
        return g, g.data_ptr(), 0
    g = g.contiguous()
    return g, g.data_ptr(), 1


def _workspace(code, rows, V, k, dev):
    """(workspace or None, its address) of one forward call."""
    n = _lib.lib().kfac_vocab_ws_bytes(code, rows, V, k)
    if not n:
        return None, 0
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr()


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# -------------------------------------------------------- CPU: the formulas
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


def _logprobs(logits, targets, k, entropy, inv_t, ignore, keep):
    """(logprobs, entropy, top_logprobs, top_ids, int64 targets, (M, L) where `keep`)."""
    shape = logits.shape[:-1]
    V = logits.shape[-1]
    rows = logits.numel() // V
    dt = torch.float64 if logits.dtype == torch.float64 else torch.float32
    lp = None if targets is None else logits.new_empty(shape, dtype=dt)
    h = logits.new_empty(shape, dtype=dt) if entropy else None
    tl = ti = stats = None
    if k:
        tl = logits.new_empty(shape + (k,), dtype=dt)
        ti = logits.new_empty(shape + (k,), dtype=torch.int64)
    tgt = None if targets is None else targets.to(torch.int64).contiguous()
    if rows == 0:
        pass
    elif _lib.use_native(logits):
        x, ld = _rows(logits, rows, V)
        code = _CODE[x.dtype]
        if keep:
            stats = logits.new_empty(2 * rows, dtype=torch.float32)
        ws, wp = _workspace(code, rows, V, k, logits.device)
        _fwd(logits.device, x.data_ptr(), _ptr(tgt), _ptr(lp), _ptr(h), _ptr(tl), _ptr(ti),
             _ptr(stats), 0, 0, 0, 0, 0, wp, ld, rows, V, ignore, code, k, 0, 0, 0, inv_t)
    else:
        x, M, _, all_lp = _cpu_stats(logits.reshape(rows, V), inv_t)
        skip = torch.zeros(rows, dtype=torch.bool) if tgt is None else tgt.reshape(-1) == ignore
        if lp is not None:
            v = _gather(all_lp, tgt.reshape(-1, 1).masked_fill(skip[:, None], 0))[:, 0]
            lp.copy_(torch.where(skip, 0.0, v).view(shape))
        if h is not None:
            v = _cpu_entropy(all_lp, M == -math.inf)
            h.copy_(torch.where(skip, 0.0, v).view(shape))
        if k:
            # stable, so that equal values keep the order of their indices
            ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
            ti.copy_(ids.masked_fill(skip[:, None], -1).view(shape + (k,)))
            tl.copy_(all_lp.gather(1, ids).masked_fill(skip[:, None], -math.inf)
                     .view(shape + (k,)))
    return lp, h, tl, ti, tgt, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, k, entropy, inv_t, ignore):
        lp, h, tl, ti, tgt, ctx.stats = _logprobs(logits, targets, k, entropy, inv_t, ignore, True)
        ctx.inv_t, ctx.ignore = inv_t, ignore
        ctx.set_materialize_grads(False)
        if k:
            ctx.mark_non_differentiable(tl, ti)
        ctx.save_for_backward(logits, tgt, h)
        return lp, h, tl, ti

    @staticmethod
    @once_differentiable
    def backward(ctx, g, gh, _tl, _ti):
        logits, tgt, h = ctx.saved_tensors
        if g is None and gh is None:
            return (None,) * 6
        V = logits.shape[-1]
        rows = logits.numel() // V
        dx = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if rows == 0:
            return dx, None, None, None, None, None
        if _lib.use_native(logits):
            x, ld = _rows(logits, rows, V)
            (g, gp, gs), (gh, ghp, ghs) = _row_grad(g), _row_grad(gh)
            _bwd(logits.device, x.data_ptr(), ctx.stats.data_ptr(), _ptr(h), _ptr(tgt), gp, ghp, 0,
                 0, dx.data_ptr(), ld, rows, V, ctx.ignore, gs, ghs, _CODE[x.dtype], 0, ctx.inv_t)
        else:
            _, M, _, lp = _cpu_stats(logits.reshape(rows, V), ctx.inv_t)
            p = lp.exp()
            d = torch.zeros_like(p)
            zero = M == -math.inf
            if g is not None:
                t, g = tgt.reshape(-1, 1), g.reshape(-1, 1)
                bad = (t < 0) | (t >= V)
                zero = zero | (t[:, 0] == ctx.ignore)
                d = (-p * g).scatter_add_(1, t.masked_fill(bad, 0), g.to(p.dtype))
                d = torch.where(bad, math.nan, d)
            elif tgt is not None:
                zero = zero | (tgt.reshape(-1) == ctx.ignore)
            if gh is not None:
                d = d - gh.reshape(-1, 1) * torch.where(
                    p == 0, 0.0, p * (lp + h.reshape(-1, 1)))
            dx.copy_(torch.where(zero[:, None], 0.0, d * ctx.inv_t).view(dx.shape))
        return dx, None, None, None, None, None


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
    0 and no gradient.  NaN or +inf in a row makes its results NaN.
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
    _check_plain('token_logprobs', logits, targets)
    args = logits, targets, k, bool(entropy), inv_t, int(ignore_index)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(*args))
    return TokenLogprobs(*_logprobs(*args, False)[:4])


def _cpu_teacher(ids, teacher, V, inv_t, dtype):
    """(some used slot, id or 0, q, log q) of rows of slots; bad ids make q NaN."""
    t = teacher.to(dtype).masked_fill(ids == -1, -math.inf)
    t = t.masked_fill((ids < -1) | (ids >= V), math.nan)
    some = ~(t == -math.inf).all(1)
    top = torch.where(some, t.amax(1), torch.zeros((), dtype=dtype))[:, None]
    d = (t - top) * inv_t
    Z = d.exp().sum(1, keepdim=True)
    return some, ids.clamp(0, V - 1), d.exp() / Z, d - Z.log()


def _distill(logits, ids, teacher, inv_t, keep):
    """(losses, ids and teacher as they are read, what the GPU's backward pass
    needs where `keep`: (M, L) of the rows, each id once and its mass)."""
    V, K = logits.shape[-1], ids.shape[-1]
    rows = logits.numel() // V
    dt = torch.float64 if logits.dtype == torch.float64 else torch.float32
    ids = ids.to(torch.int64).contiguous()
    teacher = teacher.contiguous()
    loss = logits.new_empty(logits.shape[:-1], dtype=dt)
    kept = None
    if rows and _lib.use_native(logits):
        x, ld = _rows(logits, rows, V)
        code = _CODE[x.dtype]
        stats = at = mass = None
        if keep:
            stats = logits.new_empty(2 * rows, dtype=torch.float32)
            at = ids.new_empty(rows * K, dtype=torch.int32)
            mass = logits.new_empty(rows * K, dtype=torch.float32)
            kept = stats, at, mass
        ws, wp = _workspace(code, rows, V, 0, logits.device)
        _fwd(logits.device, x.data_ptr(), 0, 0, 0, 0, 0, _ptr(stats), ids.data_ptr(),
             teacher.data_ptr(), loss.data_ptr(), _ptr(at), _ptr(mass), wp, ld, rows, V, 0, code,
             0, K, _CODE[teacher.dtype], 0, inv_t)
    elif rows:
        lp = _cpu_stats(logits.reshape(rows, V), inv_t)[3]
        some, at, q, logq = _cpu_teacher(ids.reshape(rows, K), teacher.reshape(rows, K), V, inv_t,
                                         dt)
        each = torch.where(q == 0, 0.0, q * (logq - lp.gather(1, at)))
        loss.copy_(torch.where(some, each.sum(1), 0.0).view(loss.shape))
    return loss, ids, teacher, kept


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, inv_t):
        loss, ids, teacher, ctx.kept = _distill(logits, ids, teacher, inv_t, True)
        ctx.save_for_backward(logits, ids, teacher)
        ctx.inv_t = inv_t
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, ids, teacher = ctx.saved_tensors
        V, K = logits.shape[-1], ids.shape[-1]
        rows = logits.numel() // V
        dx = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if rows and _lib.use_native(logits):
            x, ld = _rows(logits, rows, V)
            g, gp, gs = _row_grad(g)
            stats, at, mass = ctx.kept
            _bwd(logits.device, x.data_ptr(), stats.data_ptr(), 0, 0, gp, 0, at.data_ptr(),
                 mass.data_ptr(), dx.data_ptr(), ld, rows, V, 0, gs, 0, _CODE[x.dtype], K,
                 ctx.inv_t)
        elif rows:
            _, M, _, lp = _cpu_stats(logits.reshape(rows, V), ctx.inv_t)
            some, at, q, _ = _cpu_teacher(ids.reshape(rows, K), teacher.reshape(rows, K), V,
                                          ctx.inv_t, lp.dtype)
            bad = torch.where(torch.isnan(q).any(1, keepdim=True), math.nan, 1.0).to(lp.dtype)
            d = (lp.exp() * bad).scatter_add_(1, at, -q) * (g.reshape(-1, 1) * ctx.inv_t)
            live = some & (M != -math.inf)
            dx.copy_(torch.where(live[:, None], d, 0.0).view(dx.shape))
        return dx, None, None, None


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
    _check_plain(name, logits, teacher_ids, teacher_logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _TopkDistill.apply(logits, teacher_ids, teacher_logits, inv_t)
    return _distill(logits, teacher_ids, teacher_logits, inv_t, False)[0]
