"""Dropout that stores no mask and can be recomputed.

``aten::dropout`` (elementary.py, monet/lm_ops/elementary.py:5-95) defers to autograd, which keeps a
mask, and draws another one when its forward is repeated.  ``monet::dropout`` keeps a 64-bit seed in
``op.params``, which the executor hands to every later instance of the node: backward and recomputed
forward regenerate the mask.  It has a node name of its own, so the slots of ``aten::dropout`` are
untouched; to use it rename the node (``runner.Runner(..., counter_dropout=True)`` does)."""
from __future__ import annotations

import torch

from .. import functional as F
from .base import COMMON_MODES, OP, implements


def training_p(p, training) -> float:
    """The probability that applies: nothing is dropped outside training."""
    return float(p) if training else 0.0


@implements(['monet::dropout'], COMMON_MODES)
class CounterDropout(OP):
    backward_storage = None
    params = None
    inplace = False

    def forward(self, x, p, training=True, *args, **kwargs):
        with torch.no_grad():
            if self.params is None:
                p = training_p(p, training)
                self.params = p, (F.dropout_seed(x.device) if p > 0 else None), F.is_nhwc(x)
            p, seed, nhwc = self.params
            x = _in_order(x, nhwc)
            return F.dropout(x, p, seed, inplace=self.inplace)

    def backward(self, grad_output, stored, nodel=False):
        assert len(stored) == 0
        with torch.no_grad():
            p, seed, nhwc = self.params
            return F.dropout_bwd(_in_order(grad_output, nhwc), p, seed)


def _in_order(t, nhwc):
    """`t` in the physical order of the first forward's input, which the mask is indexed by."""
    if nhwc:
        return t.contiguous(memory_format=torch.channels_last)
    return t.contiguous()
