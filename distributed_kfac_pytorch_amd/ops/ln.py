"""Layer norm with the residual add in front of it (csrc/ln.hip): the
normalisation layers of the Transformer LM (models/transformer_lm.py, through
`modules.LayerNorm`).

`layer_norm(x, normalized_shape, weight, bias, eps, z=None)` computes

    y = F.layer_norm(x, normalized_shape, weight, bias, eps)           without z
    s = x + z;  y = F.layer_norm(s, ...);  returns (y, s)               with z

with the semantics of torch's two operations: s has their promoted type, y the
type of s (fp32 under autocast, which runs layer norms in fp32).  On a GPU, for
fp32 / bf16 / fp16 tensors, it is one kernel forward and two or three backward
(hipGraph-capturable, bitwise reproducible; statistics and all sums in fp32);
anything else (CPU tensors, fp64, tensor subclasses, z of another shape,
functorch transforms, torch.compile traces) takes the two torch operations.
Unlike F.layer_norm, the weights may have another type than x.
`KFAC_FUSED_LN=0` disables the kernels.

A second derivative (create_graph=True) is taken through torch's operations.
K-FAC hooks Conv2d / Linear only; a layer norm is not preconditioned
(reference: kfac/layers/__init__.py registers Linear and Conv2d).
"""
import math
import os

import torch
import torch.nn.functional as F

from . import _lib

__all__ = ['layer_norm', 'eligible', 'ENABLED']

ENABLED = os.environ.get('KFAC_FUSED_LN', '1') != '0'

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _code(t):
    return 0 if t is None else _lib.DTYPE_CODE[t.dtype]


def eligible(x, normalized_shape, weight=None, bias=None, z=None):
    """True where the kernels run (see the module's text)."""
    if not (ENABLED and x.is_cuda and x.dtype in _TYPES and x.numel() > 0):
        return False
    n = len(normalized_shape)
    if n == 0 or tuple(x.shape[-n:]) != normalized_shape:
        return False
    if z is not None and (z.shape != x.shape or z.dtype not in _TYPES or z.device != x.device):
        return False
    for p in (weight, bias):
        if p is not None and (p.dtype not in _TYPES or p.device != x.device or
                              tuple(p.shape) != normalized_shape):
            return False
    return _lib.plain_tensors(x, z, weight, bias)


def _rows(t, rows, D):
    """t as (rows, D) with contiguous rows (a copy where no view has them) and
    the distance between rows."""
    if t.is_contiguous():
        return t, D
    t = t.reshape(rows, D)
    if D > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _forward(x, z, weight, bias, D, eps, ydtype):
    """(y, s, mean, rstd); s is x without z."""
    L = _lib.lib()
    rows = x.numel() // D
    if z is not None and x.dtype != z.dtype and x.dtype != torch.float32:
        x, z = z, x                              # the sum's type is the wider one's: fp32 ...
        if x.dtype != torch.float32:
            x = x.float()                        # ... also for bf16 + fp16
    y = torch.empty(x.shape, dtype=x.dtype if ydtype is None else ydtype, device=x.device)
    s = None if z is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    xr, ldx = _rows(x, rows, D)
    zr, ldz = (None, 0) if z is None else _rows(z, rows, D)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    with _lib.device_guard(x.device):
        _lib.check(L.kfac_ln_forward(
            xr.data_ptr(), ldx, _code(x), _ptr(zr), ldz, _code(z), _ptr(w), _code(w), _ptr(b),
            _code(b), y.data_ptr(), _code(y), _ptr(s), stats.data_ptr(),
            stats.data_ptr() + 4 * rows, rows, D, float(eps), _lib.stream(x.device)),
            'kfac_ln_forward')
    return y, (x if z is None else s), stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, weight, bias, shape, eps, ydtype):
        y, s, stats = _forward(x, z, weight, bias, math.prod(shape), eps, ydtype)
        ctx.save_for_backward(s, weight, bias, stats)
        ctx.shape, ctx.eps = shape, eps
        ctx.xdtype, ctx.zdtype = x.dtype, None if z is None else z.dtype
        ctx.set_materialize_grads(False)
        return y if z is None else (y, s)

    @staticmethod
    def backward(ctx, dy, ds=None):
        s, weight, bias, stats = ctx.saved_tensors
        if dy is None and ds is None:
            return (None,) * 7
        if dy is None:
            d, dw, db = ds, None, None
        elif torch.is_grad_enabled():            # create_graph: differentiable operations
            d, dw, db = _differentiable(ctx, s, weight, bias, dy, ds)
        else:
            d, dw, db = _backward(ctx, s, weight, bias, stats, dy, ds)
        if type(d) is tuple:
            dx, dz = d
        else:
            dx = None if d is None else d.to(ctx.xdtype)
            dz = None if d is None or ctx.zdtype is None else d.to(ctx.zdtype)
        return dx, dz, dw, db, None, None, None


def _backward(ctx, s, weight, bias, stats, dy, ds):
    """((dx, dz), dw, db), each None where it is not asked for."""
    L = _lib.lib()
    D = math.prod(ctx.shape)
    rows = s.numel() // D
    need_x, need_z, need_w, need_b = ctx.needs_input_grad[:4]
    sr, lds = _rows(s, rows, D)
    gr, ldg = _rows(dy, rows, D)
    er, lde = (None, 0) if ds is None else _rows(ds, rows, D)
    dx = torch.empty(s.shape, dtype=s.dtype, device=s.device) if need_x or need_z else None
    # one of x and z may be narrower than their sum: its gradient is stored on its own
    low = next((t for t in (ctx.xdtype, ctx.zdtype) if t not in (None, s.dtype)), None)
    same = dx is None or low is None or ctx.xdtype == ctx.zdtype
    dl = None if same else torch.empty(s.shape, dtype=low, device=s.device)
    dw = torch.empty(weight.shape, dtype=weight.dtype, device=s.device) if need_w else None
    db = torch.empty(bias.shape, dtype=bias.dtype, device=s.device) if need_b else None
    part = torch.empty(L.kfac_ln_ws_floats(_code(s), rows, D), dtype=torch.float32, device=s.device) \
        if need_w or need_b else None
    w = None if weight is None else weight.contiguous()
    with _lib.device_guard(s.device):
        _lib.check(L.kfac_ln_backward(
            gr.data_ptr(), ldg, _code(gr), _ptr(er), lde, sr.data_ptr(), lds, _code(s), _ptr(w),
            _code(w), _code(bias), stats.data_ptr(), stats.data_ptr() + 4 * rows, _ptr(dx),
            _ptr(dl), _code(dl), _ptr(dw), _ptr(db), _ptr(part), rows, D,
            _lib.stream(s.device)), 'kfac_ln_backward')

    def of(dtype):
        if dx is None or dtype is None:
            return None
        return dx if dtype == s.dtype else dl if dl is not None and dtype == low else dx.to(dtype)
    return (of(ctx.xdtype) if need_x else None, of(ctx.zdtype) if need_z else None), dw, db


def _differentiable(ctx, s, weight, bias, dy, ds):
    """(gradient of s, dw, db) by operations that autograd follows."""
    with torch.enable_grad():
        s_ = s if s.requires_grad else s.detach().requires_grad_(True)
        y = F.layer_norm(s_.to(dy.dtype), ctx.shape,
                         None if weight is None else weight.to(dy.dtype),
                         None if bias is None else bias.to(dy.dtype), ctx.eps)
        inputs = [s_] + [t for t in (weight, bias) if t is not None and t.requires_grad]
        g = list(torch.autograd.grad(y, inputs, dy, create_graph=True))
    d = g.pop(0)
    dw = g.pop(0) if weight is not None and weight.requires_grad else None
    db = g.pop(0) if bias is not None and bias.requires_grad else None
    return d if ds is None else d + ds, dw, db


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5, z=None):
    """F.layer_norm(x), or (F.layer_norm(x + z), x + z) where z is given."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not eligible(x, shape, weight, bias, z):
        s = x if z is None else x + z
        y = F.layer_norm(s, shape, weight, bias, eps)
        return y if z is None else (y, s)
    ydtype = torch.float32 if torch.is_autocast_enabled('cuda') else None
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, z, weight, bias)):
        return _LayerNorm.apply(x, z, weight, bias, shape, eps, ydtype)
    y, s, _ = _forward(x, z, weight, bias, math.prod(shape), eps, ydtype)
    return y if z is None else (y, s)
