"""Layer norm with the residual add in front of it (csrc/ln.hip): the
normalisation layers of the Transformer LM (models/transformer_lm.py, through
`modules.LayerNorm`).

`layer_norm(x, normalized_shape, weight, bias, eps, z=None)` computes

    y = F.layer_norm(x, normalized_shape, weight, bias, eps)           without z
    s = x + z;  y = F.layer_norm(s, ...);  returns (y, s)               with z

with the semantics of torch's two operations: s has their promoted type, y the
type of s (fp32 under autocast, which runs layer norms in fp32).  On a GPU, for
fp32 / bf16 / fp16 tensors, it is one kernel forward and two backward
(hipGraph-capturable, bitwise reproducible; statistics and all sums in fp32;
the autograd node is C++, csrc/torch_ops.cpp); anything else (CPU tensors, fp64,
tensor subclasses, z of another shape, functorch transforms, dispatch modes,
traces) takes the two torch operations.
Unlike F.layer_norm, the weights may have another type than x.
`KFAC_FUSED_LN=0` disables the kernels.  An installation that was built without
torch, or with another one, has no such node: torch's operations run, with a warning.

A second derivative (create_graph=True) is taken through elementary operations.
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


def eligible(x, normalized_shape, weight=None, bias=None, z=None):
    """True where the kernels run (see the module's text)."""
    # asked first: a trace warns of Python values taken from shapes, and a nested
    # tensor has no shape
    if not (ENABLED and x.is_cuda and x.dtype in _TYPES and not x.is_nested and
            _lib.plain_tensors(x, z, weight, bias)):
        return False
    n = len(normalized_shape)
    if x.numel() == 0 or n == 0 or x.shape[-n:] != normalized_shape or \
            x.numel() // math.prod(normalized_shape) >= 2 ** 31:
        return False
    if z is not None and (z.shape != x.shape or z.dtype not in _TYPES or z.device != x.device):
        return False
    for p in (weight, bias):
        if p is not None and (p.dtype not in _TYPES or p.device != x.device or
                              p.shape != normalized_shape):
            return False
    return _lib.has_torch_ops()


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5, z=None):
    """F.layer_norm(x), or (F.layer_norm(x + z), x + z) where z is given."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not eligible(x, shape, weight, bias, z):
        s = x if z is None else x + z
        y = F.layer_norm(s, shape, weight, bias, eps)
        return y if z is None else (y, s)
    y, s = _lib.torch_ops().layer_norm.default(x, z, weight, bias, len(shape), eps,
                                               torch.is_autocast_enabled('cuda'))
    return y if z is None else (y, s)
