"""Layer norm in the two forms batch norm has: backward from the stored input, and from the stored
output (monet/lm_ops/ln.py:13-40 has the first).  The row statistics of the forward travel in
``op.params``; a recomputed forward finds the same ones again."""
from __future__ import annotations

import torch

from .. import functional as F
from .base import OP, InputStorage, OutputStorage, implements


class _LayerNorm(OP):
    params = None
    inplace = False

    def forward(self, input_, normalized_shape, weight=None, bias=None, eps=1e-5, *args, **kwargs):
        with torch.no_grad():
            out, mean, rstd = F.layer_norm(input_, normalized_shape, weight, bias, eps, inplace=self.inplace)
            self.params = list(normalized_shape), mean, rstd
            return out


def _present(dx, dw, db):
    """One gradient per tensor argument: an absent weight or bias has none."""
    return tuple(g for g in (dx, dw, db) if g is not None)


@implements(['aten::layer_norm'],
            ['normal', 'multiway', 'newnode', 'multiway_newnode', 'conv_multiway_newnode',
             'conv_normal'])
class InputActLayerNorm(_LayerNorm):
    """Backward from the stored input x."""
    backward_storage = InputStorage(0, 2, 3)

    def backward(self, grad_output, stored, nodel=False):
        with torch.no_grad():
            input_, weight, bias = stored
            shape, mean, rstd = self.params
            grads = F.layer_norm_bwd_from_input(grad_output, input_, shape, weight, mean, rstd,
                                                weight is not None, bias is not None)
            if not nodel:
                del stored[2], stored[1], stored[0]
            return _present(*grads)


@implements(['aten::layer_norm'], ['multiway', 'multiway_newnode', 'conv_multiway_newnode'])
class OutputActLayerNorm(_LayerNorm):
    """Backward from the stored OUTPUT y, xhat = (y - bias) / weight: the input is not kept and the
    forward can run in place.  Every weight must be non-zero."""
    backward_storage = [InputStorage(2, 3), OutputStorage()]
    divides_by = 2                      # position of the argument that must not hold a zero

    def backward(self, grad_output, stored, nodel=False):
        with torch.no_grad():
            weight, bias, output = stored
            shape, _, rstd = self.params
            grads = F.layer_norm_bwd_from_output(grad_output, output, shape, weight, bias, rstd,
                                                 weight is not None, bias is not None)
            if not nodel:
                del stored[2], stored[1], stored[0]
            return _present(*grads)
