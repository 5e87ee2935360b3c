"""Dropout from a counter-based generator, its mask never stored (``po_dropout``).

Beside the patch transformer's keyed draws (``load_data``'s ``po_draws``): an
element's fate is a function of (seed, step, global row, column), so the
backward pass draws the mask again instead of reading it, and a rank that
holds rows ``[row0, row0 + rows)`` of a batch drops what a single process
drops there.  The reference has no dropout; its randomness is the CUDA
generator's (load_data.py:548-574).
"""
import torch
import torch.nn as nn

from . import _native as nat


def _launch(x, residual, drop, seed, step, row0):
    """y, and the step taken as a device number where step is one (else None)."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    on_device = isinstance(step, torch.Tensor)
    used = torch.empty(1, dtype=torch.int64, device=x.device) if on_device else None
    if x.numel() == 0:
        if on_device:
            used.copy_(step.reshape(1))
        return y, used
    xm, ldx = nat.rows2d(x)
    rm, ldr = (None, 0) if residual is None else nat.rows2d(residual)
    rows, cols = xm.shape
    nat.call("po_dropout", xm.data_ptr(), ldx, None if rm is None else rm.data_ptr(), ldr, nat.DTYPES[x.dtype], rows, cols,
             seed, 0 if on_device else step, step.data_ptr() if on_device else None,
             used.data_ptr() if on_device else None, row0, drop, y.data_ptr(), cols, nat.raw_stream(x))
    return y, used


def _run(x, residual, drop, seed, step, row0):
    with nat.device_of(*(t for t in (x, residual, step) if isinstance(t, torch.Tensor))):
        return _launch(x, residual, drop, seed, step, row0)


class _KeyedDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, drop, seed, step, row0):
        y, used = _run(x, residual, drop, seed, step, row0)
        ctx.key = (drop, seed, step if used is None else None, row0)
        if used is not None:
            ctx.save_for_backward(used)      # the caller may move its step on before the backward pass
        return y

    @staticmethod
    def backward(ctx, dy):
        drop, seed, step, row0 = ctx.key
        if step is None:
            (step,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            # the same linear map; through apply where it has to be differentiable again
            if torch.is_grad_enabled():
                dx = _KeyedDropout.apply(dy, None, drop, seed, step, row0)
            else:
                dx = _run(dy, None, drop, seed, step, row0)[0]
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None, None


def keyed_dropout(x, p, seed, step=0, row0=0, residual=None):
    """``where(u >= p, x / (1 - p), 0) [+ residual]`` with u drawn from (seed, step, row0 + row, column).

    x: float32, float16 or bfloat16 on the GPU, of any shape; its last dimension
    are the columns, what is before it the rows.  p in [0, 1], taken to the nearest
    multiple of 2^-16; the scale is that probability's own.  seed: whole number
    of 64 bits, one for each place in a model that drops.  step: whole number of 64
    bits, or an int64 tensor of one element on x's device, read by the kernel
    (a captured graph that adds to it draws a new mask on every replay).
    residual: of x's shape and type.  Dropped elements are exactly 0, whatever x
    holds there; the sum is formed in 32 bits and rounded once."""
    if not isinstance(x, torch.Tensor) or x.dtype not in nat.DTYPES:
        raise TypeError("keyed_dropout: x must be a float32, float16 or bfloat16 tensor")
    if x.dim() < 1:
        raise ValueError("keyed_dropout: x needs at least one dimension")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("keyed_dropout: p must be in [0, 1], got %r" % p)
    if residual is not None and (not isinstance(residual, torch.Tensor) or residual.shape != x.shape or
                                 residual.dtype != x.dtype):
        raise ValueError("keyed_dropout: residual must have x's shape and type")
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1:
            raise TypeError("keyed_dropout: a step on the device is one int64")
    elif not 0 <= int(step) < 1 << 64:
        raise ValueError("keyed_dropout: step must be in [0, 2^64)")
    if not 0 <= int(seed) < 1 << 64:
        raise ValueError("keyed_dropout: seed must be in [0, 2^64)")
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    if int(row0) < 0 or int(row0) + rows > 1 << 32:
        raise ValueError("keyed_dropout: rows row0 .. row0 + rows must stay within 2^32")
    args = (x, residual, round(p * 65536), int(seed), step if isinstance(step, torch.Tensor) else int(step), int(row0))
    if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad):
        return _KeyedDropout.apply(*args)
    return _run(*args)[0]


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
