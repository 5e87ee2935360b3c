"""Softmax cross entropy of a linear head over a large vocabulary (``po_linear_ce_fwd``
/ ``_bwd``): the logits are never in memory, neither is their gradient beyond a
piece of the vocabulary.

Beside the cell loss over a detector's few classes (``train_patch.cell_loss``,
reference train_patch.py:468-503): the class objective of a head whose classes
are thousands of embeddings.  With a frozen vocabulary only the embeddings'
gradient is computed.
"""
import ctypes
import functools

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native as nat

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_MAX_STRIDE = 1 << 21


def _matrix(t):
    m, ld = nat.rows2d(t)
    return (m, ld) if ld <= _MAX_STRIDE else (m.contiguous(), m.shape[1])


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(h_at, ldh, w_at, ldw, dtype, N, V, D, dh, dw):
    """(forward, backward) bytes: a function of the sizes and of whether rows start on 16 bytes."""
    fwd, bwd = ctypes.c_int64(), ctypes.c_int64()
    nat.call("po_linear_ce_workspace", h_at, ldh, w_at, ldw, dtype, N, V, D, dh, dw, ctypes.byref(fwd), ctypes.byref(bwd))
    return fwd.value, bwd.value


def _workspace(h, ldh, w, ldw, dh, dw, backward):
    # 256 + the offset into 16 bytes stands for the address
    byts = _workspace_bytes(256 + h.data_ptr() % 16, ldh, 256 + w.data_ptr() % 16, ldw, nat.DTYPES[h.dtype], h.shape[0],
                            w.shape[0], h.shape[1], int(dh), int(dw))[backward]
    return torch.empty(byts, dtype=torch.uint8, device=h.device)


def _forward(hidden, weight, target, ignore_index, reduction, scale):
    """(loss, what the backward pass needs: target as a vector, statistics [N][2] and the count behind them)."""
    with nat.device_of(hidden, weight, target):
        h, ldh = _matrix(hidden)
        w, ldw = _matrix(weight)
        t = target.reshape(-1).contiguous()
        N, D = h.shape
        loss = torch.empty(target.shape if reduction == 0 else (), dtype=torch.float32, device=h.device)
        stat = torch.empty(2 * N + 1, dtype=torch.float32, device=h.device)
        if N:
            ws = _workspace(h, ldh, w, ldw, False, False, False)
            nat.call("po_linear_ce_fwd", h.data_ptr(), ldh, w.data_ptr(), ldw, nat.DTYPES[h.dtype], N, w.shape[0], D,
                     t.data_ptr(), ignore_index, scale, reduction, ws.data_ptr(), ws.numel(), stat.data_ptr(),
                     loss.data_ptr(), stat.data_ptr() + 8 * N, nat.raw_stream(h))
        elif reduction:
            loss.fill_(float("nan") if reduction == 2 else 0.0)
    return loss, t, stat


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction, scale):
        loss, t, stat = _forward(hidden, weight, target, ignore_index, reduction, scale)
        ctx.save_for_backward(hidden, weight, t, stat)
        ctx.meta = (ignore_index, reduction, scale)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, t, stat = ctx.saved_tensors
        ignore_index, reduction, scale = ctx.meta
        need_h, need_w = ctx.needs_input_grad[:2]
        with nat.device_of(hidden, weight, grad):
            h, ldh = _matrix(hidden)
            w, ldw = _matrix(weight)
            (N, D), V = h.shape, w.shape[0]
            if not N:
                return (torch.zeros_like(hidden) if need_h else None, torch.zeros_like(weight) if need_w else None,
                        None, None, None, None)
            g = grad.reshape(-1).contiguous()
            dh = torch.empty(N, D, dtype=h.dtype, device=h.device) if need_h else None
            dw = torch.empty(V, D, dtype=w.dtype, device=w.device) if need_w else None
            ws = _workspace(h, ldh, w, ldw, need_h, need_w, True)
            nat.call("po_linear_ce_bwd", h.data_ptr(), ldh, w.data_ptr(), ldw, nat.DTYPES[h.dtype], N, V, D,
                     t.data_ptr(), ignore_index, scale, reduction, stat.data_ptr(), stat.data_ptr() + 8 * N, g.data_ptr(),
                     ws.data_ptr(), ws.numel(), None if dh is None else dh.data_ptr(), D,
                     None if dw is None else dw.data_ptr(), D, nat.raw_stream(h))
        return (None if dh is None else dh.view(hidden.shape)), dw, None, None, None, None


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean", scale=1.0):
    """Cross entropy of ``scale * hidden @ weight.T`` against ``target``, in float32.

    hidden [..., D] and weight [V, D] of one type (float32, float16 or bfloat16),
    target [...] int64.  Rows with ``ignore_index`` have loss and gradient 0,
    whatever hidden holds there; "mean" divides by the others' number (NaN if there is none).  A
    target outside the vocabulary makes its row's loss (and the gradients) NaN:
    nothing is read back to raise for it.  scale > 0 (an inverse temperature).
    The gradients have the inputs' type; their sums are kept in 32 bits.  In
    float16 use a loss scale, as for any float16 training: gradients below 6e-8 are 0.
    Gradients of second order are not available."""
    for name, m in (("hidden", hidden), ("weight", weight)):
        if not isinstance(m, torch.Tensor) or m.dtype not in nat.DTYPES:
            raise TypeError("linear_cross_entropy: %s must be a float32, float16 or bfloat16 tensor" % name)
    if hidden.dtype != weight.dtype:
        raise TypeError("linear_cross_entropy: hidden is %s, weight %s" % (hidden.dtype, weight.dtype))
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("linear_cross_entropy: hidden [..., D] and weight [V, D] expected, got %s and %s" %
                         (tuple(hidden.shape), tuple(weight.shape)))
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("linear_cross_entropy: the vocabulary is empty")
    if not isinstance(target, torch.Tensor) or target.dtype != torch.int64 or target.shape != hidden.shape[:-1]:
        raise ValueError("linear_cross_entropy: target must be int64 of hidden's shape without its last dimension")
    if reduction not in REDUCTIONS:
        raise ValueError("linear_cross_entropy: reduction must be one of %s" % ", ".join(REDUCTIONS))
    if not 0.0 < float(scale) < float("inf"):
        raise ValueError("linear_cross_entropy: scale must be positive and finite, got %r" % (scale,))
    args = (hidden, weight, target, int(ignore_index), REDUCTIONS[reduction], float(scale))
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(*args)
    return _forward(*args)[0]


class LinearCrossEntropy(nn.Module):
    """``linear_cross_entropy`` with a weight of its own: ``forward(hidden, target)``."""

    def __init__(self, dim, vocab, ignore_index=-100, reduction="mean", scale=1.0, device=None, dtype=None):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(vocab, dim, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=dim ** -0.5)
        self.ignore_index, self.reduction, self.scale = ignore_index, reduction, scale

    def forward(self, hidden, target):
        return linear_cross_entropy(hidden, self.weight, target, self.ignore_index, self.reduction, self.scale)
