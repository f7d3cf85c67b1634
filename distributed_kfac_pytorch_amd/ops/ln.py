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
functorch transforms, dispatch modes, traces) takes the two torch operations.
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

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # csrc/common.h

# csrc/ln.hip KfacLnFwd, KfacLnBwd
_fwd = _lib.PackedCall('kfac_ln_forward', '8P4q5if0P')
_bwd = _lib.PackedCall('kfac_ln_backward', '11P5q6i0P')


def eligible(x, normalized_shape, weight=None, bias=None, z=None):
    """True where the kernels run (see the module's text)."""
    if not (ENABLED and x.is_cuda and x.dtype in _CODE and x.numel() > 0):
        return False
    n = len(normalized_shape)
    if n == 0 or x.shape[-n:] != normalized_shape or \
            x.numel() // math.prod(normalized_shape) >= 2 ** 31:
        return False
    if z is not None and (z.shape != x.shape or z.dtype not in _CODE or z.device != x.device):
        return False
    for p in (weight, bias):
        if p is not None and (p.dtype not in _CODE or p.device != x.device or
                              p.shape != normalized_shape):
            return False
    return _lib.plain_tensors(x, z, weight, bias)


def _rows(t, rows, D):
    """(t as (rows, D) with contiguous rows -- a copy where no view has them --,
    its address, the distance between rows, its type's code); zeros for None."""
    if t is None:
        return None, 0, 0, 0
    ld = D
    if not t.is_contiguous():
        t = t.reshape(rows, D)
        if D > 1 and t.stride(1) != 1:
            t = t.contiguous()
        ld = t.stride(0)
    return t, t.data_ptr(), ld, _CODE[t.dtype]


def _like(t, dtype=None):
    """An uninitialised contiguous tensor of t's shape."""
    if dtype is None or dtype == t.dtype:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _vector(p):
    """(weight or bias contiguous, its address, its type's code); zeros for None."""
    if p is None:
        return None, 0, 0
    p = p.contiguous()
    return p, p.data_ptr(), _CODE[p.dtype]


def _forward(x, z, weight, bias, D, eps, ydtype, keep):
    """(y, s, mean and rstd where `keep`); s is x without z."""
    rows = x.numel() // D
    if z is not None and x.dtype != z.dtype and x.dtype != torch.float32:
        x, z = z, x                              # the sum's type is the wider one's: fp32 ...
        if x.dtype != torch.float32:
            x = x.float()                        # ... also for bf16 + fp16
    y = _like(x, ydtype)
    s, sp = x, 0
    if z is not None:
        s = _like(x)
        sp = s.data_ptr()
    stats, mp = None, 0
    if keep:
        stats = x.new_empty(2 * rows, dtype=torch.float32)
        mp = stats.data_ptr()
    x, xp, ldx, code = _rows(x, rows, D)
    z, zp, ldz, zcode = _rows(z, rows, D)
    w, wp, wcode = _vector(weight)
    b, bp, bcode = _vector(bias)
    _fwd(x.device, xp, zp, wp, bp, y.data_ptr(), sp, mp, mp and mp + 4 * rows, ldx, ldz, rows, D,
         code, zcode, wcode, bcode, _CODE[y.dtype], eps)
    return y, s, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, weight, bias, shape, eps, ydtype):
        y, s, ctx.stats = _forward(x, z, weight, bias, math.prod(shape), eps, ydtype, True)
        ctx.save_for_backward(s, weight, bias)
        ctx.shape, ctx.eps = shape, eps
        ctx.xdtype, ctx.zdtype = x.dtype, None if z is None else z.dtype
        ctx.set_materialize_grads(False)
        return y if z is None else (y, s)

    @staticmethod
    def backward(ctx, dy, ds=None):
        if dy is None and ds is None:
            return (None,) * 7
        s, weight, bias = ctx.saved_tensors
        dw = db = dl = None
        if dy is None:
            d = ds
        elif torch.is_grad_enabled():            # create_graph: differentiable operations
            d, dw, db = _differentiable(ctx, s, weight, bias, dy, ds)
        else:
            d, dl, dw, db = _backward(ctx, s, weight, bias, dy, ds)

        def of(dtype):
            if d is None or dtype is None:
                return None
            return d if dtype == d.dtype else dl if dl is not None and dtype == dl.dtype \
                else d.to(dtype)
        need = ctx.needs_input_grad
        return (of(ctx.xdtype) if need[0] else None, of(ctx.zdtype) if need[1] else None, dw, db,
                None, None, None)


def _backward(ctx, s, weight, bias, dy, ds):
    """(gradient of s, the same in the type of whichever of x and z is narrower,
    dw, db), each None where it is not asked for."""
    D = math.prod(ctx.shape)
    rows = s.numel() // D
    dtype = s.dtype
    need_x, need_z, need_w, need_b = ctx.needs_input_grad[:4]
    d = dl = dw = db = part = None
    dp = lp = wgp = bgp = pp = lcode = 0
    if need_x or need_z:
        d = _like(s)
        dp = d.data_ptr()
        low = ctx.xdtype if ctx.xdtype != dtype else ctx.zdtype
        if low is not None and low != dtype:
            dl = _like(s, low)
            lp, lcode = dl.data_ptr(), _CODE[low]
    w, wp, wcode = _vector(weight)
    if need_w:
        dw = _like(weight)
        wgp = dw.data_ptr()
    if need_b:
        db = _like(bias)
        bgp = db.data_ptr()
    code = _CODE[dtype]
    if need_w or need_b:
        part = s.new_empty(_lib.lib().kfac_ln_ws_floats(rows, D), dtype=torch.float32)
        pp = part.data_ptr()
    s, sp, lds, _ = _rows(s, rows, D)
    g, gp, ldg, gcode = _rows(dy, rows, D)
    e, ep, lde, _ = _rows(ds, rows, D)
    mp = ctx.stats.data_ptr()
    _bwd(s.device, gp, ep, sp, wp, mp, mp + 4 * rows, dp, lp, wgp, bgp, pp, ldg, lde, lds, rows, D,
         code, lcode, wcode, 0 if bias is None else _CODE[bias.dtype], gcode, 0)
    return d, dl, dw, db


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
    y, s, _ = _forward(x, z, weight, bias, math.prod(shape), eps, ydtype, False)
    return y if z is None else (y, s)
