"""Matrix product in 8-bit integers with a scale for each token and each output channel
(``po_quantize_rows``, ``po_int8_matmul``), for serving.

Beside the convolutions' operand precisions (``po_conv``: exact float32 and split
float16): a linear layer of a deployed detector head, its weights kept in 8 bits and its
activations quantised token by token on the way.  Inference only.  Up to 2^21 tokens a call.
"""
import warnings

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _native as nat

MAX_INNER = (1 << 17) - 1        # 127 * 128 * MAX_INNER stays below 2^31


def _no_grad(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad() or on detached tensors" % name)
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("%s has no gradient, nor a forward-mode derivative: call it on detached tensors" % name)


def _check_inner(name, K):
    if not 1 <= K <= MAX_INNER:
        raise ValueError("%s: the inner dimension must be in [1, %d], got %d" % (name, MAX_INNER, K))


def _quantize(x):
    """(q [rows, K rounded up to 64], scale [rows]) of x as rows."""
    m, ld = nat.rows2d(x)
    rows, K = m.shape
    q = torch.empty(rows, (K + 63) // 64 * 64, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows:
        nat.call("po_quantize_rows", m.data_ptr(), ld, nat.DTYPES[x.dtype], rows, K, q.data_ptr(), q.stride(0),
                 scale.data_ptr(), nat.raw_stream(x))
    return q, scale


def _weights(w):
    """w as rows that start on 16 bytes and are laid out to a multiple of 16 (a copy if it is not)."""
    K = w.shape[1]
    ld = w.stride(0) if w.shape[0] > 1 else (K + 15) // 16 * 16
    if (K == 1 or w.stride(1) == 1) and ld % 16 == 0 and (K + 15) // 16 * 16 <= ld <= 1 << 22 and w.data_ptr() % 16 == 0 \
            and (w.shape[0] > 1 or K % 16 == 0):
        return w, ld
    w = lay_out(w)
    return w, w.stride(0)


def _matmul(q, sx, rows, K, wq, wscale, bias, dtype):
    y = torch.empty(rows, wq.shape[0], dtype=dtype, device=q.device)
    if rows:
        w, ldw = _weights(wq)
        nat.call("po_int8_matmul", q.data_ptr(), q.stride(0), sx.data_ptr(), w.data_ptr(), ldw, wscale.data_ptr(),
                 None if bias is None else bias.data_ptr(), rows, wq.shape[0], K, y.data_ptr(), wq.shape[0],
                 nat.DTYPES[dtype], nat.raw_stream(q))
    return y


def _check_weights(name, K, wq, wscale, bias):
    if not isinstance(wq, torch.Tensor) or wq.dtype != torch.int8 or wq.dim() != 2 or wq.shape[1] != K or wq.shape[0] < 1:
        raise ValueError("%s: the weights must be int8 [out, %d]" % (name, K))
    for t, what in ((wscale, "weight scales"), (bias, "bias")):
        if t is None and what == "bias":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (wq.shape[0],):
            raise ValueError("%s: the %s must be float32 [%d]" % (name, what, wq.shape[0]))


def lay_out(wq):
    """int8 [out, K] -> the same values as a view of padded rows, the layout the product reads
    without a copy: rows start on 128 bytes, and long ones not on 256."""
    return nat.head().lay_out(wq)


def quantize_rows(x):
    """(q, scale): int8 of x's shape and one float32 scale for each row of its last dimension,
    ``scale = max|row| / 127``, ``q = row / scale`` to the nearest (the exact quotient, ties to
    even; at most 127, which quotients pass where the scale itself is rounded at 2^-149).  A row
    of zeros gets scale 0, a row that holds NaN or an infinity scale NaN and q 0."""
    if not isinstance(x, torch.Tensor) or x.dtype not in nat.DTYPES or x.dim() < 1:
        raise TypeError("quantize_rows: x must be a float32, float16 or bfloat16 tensor of rows")
    _check_inner("quantize_rows", x.shape[-1])
    _no_grad("quantize_rows", x)
    with nat.device_of(x):
        q, scale = _quantize(x)
    return q[:, :x.shape[-1]].view(x.shape), scale.view(x.shape[:-1])


def int8_matmul(q, scale, wq, wscale, bias=None, dtype=torch.bfloat16):
    """``(q @ wq.T) * scale[..., None] * wscale + bias`` with whole-number sums in 32 bits, in dtype.

    q int8 [..., K], scale float32 [...]; wq int8 [out, K], wscale and bias float32 [out].
    Weights whose rows do not start on 16 bytes (K or the stride no multiple of 16) are copied
    first: ``lay_out`` them once instead."""
    if not isinstance(q, torch.Tensor) or q.dtype != torch.int8 or q.dim() < 1:
        raise TypeError("int8_matmul: q must be int8 rows")
    K = q.shape[-1]
    _check_inner("int8_matmul", K)
    if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or scale.shape != q.shape[:-1]:
        raise ValueError("int8_matmul: scale must be float32 of q's shape without its last dimension")
    if dtype not in nat.DTYPES:
        raise TypeError("int8_matmul: dtype must be float32, float16 or bfloat16")
    _check_weights("int8_matmul", K, wq, wscale, bias)
    _no_grad("int8_matmul", scale, wscale, bias)
    with nat.device_of(*(t for t in (q, scale, wq, wscale, bias) if t is not None)):
        m, ld = nat.rows2d(q)
        if K % 16 or ld % 16 or m.data_ptr() % 16 or ld > 1 << 22:
            store = torch.zeros(m.shape[0], (K + 63) // 64 * 64, dtype=torch.int8, device=q.device)
            store[:, :K] = m                                 # what lies behind a row's end must be 0
            m = store
        elif m.shape[0] == 1:
            m = m.as_strided((1, K), (K, 1))
        y = _matmul(m, scale.reshape(-1).contiguous(), m.shape[0], K, wq, wscale.contiguous(),
                    None if bias is None else bias.contiguous(), dtype)
    return y.view(q.shape[:-1] + (wq.shape[0],))


def int8_linear(x, wq, wscale, bias=None):
    """A linear layer in 8 bits: x [..., K] quantised row by row, times wq [out, K], in x's type."""
    return nat.head().int8_linear(x, wq, wscale, bias)


class Int8Linear(nn.Module):
    """A linear layer whose weights are kept in 8 bits, laid out once.

    weight [out, K] float (quantised row by row with ``quantize_rows``), bias [out] or None.
    A served layer: its output is cut off from the graph of an input that requires a gradient,
    with a warning where grad mode is on (``int8_linear`` raises)."""

    def __init__(self, weight, bias=None):
        super().__init__()
        with torch.no_grad():
            q, scale = quantize_rows(weight.detach())
            self.register_buffer("wq", lay_out(q))
            self.register_buffer("wscale", scale)
            self.register_buffer("bias", None if bias is None else bias.detach().float().clone())

    @classmethod
    def from_linear(cls, linear):
        """Of an ``nn.Linear`` on the GPU."""
        return cls(linear.weight, linear.bias)

    def _apply(self, fn, *args, **kw):
        # moves go through; the scales stay 32 bits under .half() and the like, and the
        # weights' layout is made anew (a copy of a view is packed)
        scale, bias = self.wscale, self.bias
        super()._apply(fn, *args, **kw)
        self.wscale = scale.to(self.wq.device)
        self.bias = None if bias is None else bias.to(self.wq.device)
        self.wq = lay_out(self.wq)
        return self

    def forward(self, x):
        if torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad:
            warnings.warn("Int8Linear has no gradient: its output is cut off from its input's graph; call it under "
                          "torch.no_grad() or on detached tensors", stacklevel=2)
        with torch.no_grad():
            return int8_linear(x, self.wq, self.wscale, self.bias)

    def extra_repr(self):
        return "in=%d, out=%d" % (self.wq.shape[1], self.wq.shape[0])
