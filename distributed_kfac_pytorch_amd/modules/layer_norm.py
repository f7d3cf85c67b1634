"""nn.LayerNorm on the gfx950 kernels of ops/ln.py, with an optional residual."""
import torch.nn as nn

from ..ops.ln import layer_norm

__all__ = ['LayerNorm']


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm (same arguments, parameters and state_dict) whose call takes
    the residual add with it: ``norm(x)``, or ``y, s = norm(x, z)`` with
    s = x + z and y the norm of s -- one pass over the tensors where
    ``ops.ln.eligible`` holds, torch's two operations elsewhere."""

    def forward(self, x, z=None):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps, z)
