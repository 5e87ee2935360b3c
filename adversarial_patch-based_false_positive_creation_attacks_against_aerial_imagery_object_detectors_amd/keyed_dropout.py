"""Dropout from a counter-based generator, its mask never stored (``po_dropout``).

Beside the patch transformer's keyed draws (``load_data``'s ``po_draws``): an
element's fate is a function of (seed, step, global row, column), so the
backward pass draws the mask again instead of reading it, and a rank that
holds rows ``[row0, row0 + rows)`` of a batch drops what a single process
drops there.  The reference has no dropout; its randomness is the CUDA
generator's (load_data.py:548-574).
"""
import torch.nn as nn

from . import _native as nat


def keyed_dropout(x, p, seed, step=0, row0=0, residual=None):
    """``where(u >= p, x / (1 - p), 0) [+ residual]`` with u drawn from (seed, step, row0 + row, column).

    x: float32, float16 or bfloat16 on the GPU, of any shape; its last dimension
    are the columns, what is before it the rows.  p in [0, 1], taken to the nearest
    multiple of 2^-16; the scale is that probability's own.  seed: whole number
    of 64 bits, one for each place in a model that drops.  step: whole number of 64
    bits, or an int64 tensor of one element on x's device, read by the kernel
    (a captured graph that adds to it draws a new mask on every replay).
    residual: of x's shape and type.  Dropped elements are exactly 0, whatever x
    holds there; the sum is formed in 32 bits and rounded once.
    Differentiable any number of times backwards; forward-mode derivatives raise."""
    return nat.head().keyed_dropout(x, p, seed, step, row0, residual)


class KeyedDropout(nn.Module):
    """``keyed_dropout`` as a module: drops while training, and is the identity (plus
    the residual) in eval mode.  The caller advances ``step`` (a whole number, or an int64
    tensor on the device) between training steps."""

    def __init__(self, p=0.5, seed=0):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("KeyedDropout: p must be in [0, 1], got %r" % p)
        self.p, self.seed, self.step = p, seed, 0

    def forward(self, x, residual=None, row0=0):
        if not self.training:
            return x if residual is None else x + residual
        return keyed_dropout(x, self.p, self.seed, self.step, row0, residual)

    def extra_repr(self):
        return "p=%g, seed=%d" % (self.p, self.seed)
