"""Softmax cross entropy of a linear head over a large vocabulary (``po_linear_ce_fwd``
/ ``_bwd``, ``po_linear_ce_frozen_fwd`` / ``_bwd``): the logits are never in memory, neither is their gradient beyond a
piece of the vocabulary.

Beside the cell loss over a detector's few classes (``train_patch.cell_loss``,
reference train_patch.py:468-503): the class objective of a head whose classes
are thousands of embeddings.  Against a frozen vocabulary (a weight that requires no
gradient) the embeddings' gradient is made in the forward pass, a piece's
exponentials being at hand there: two products where three would be.  A loss that is
not differentiated belongs under ``torch.no_grad()``.
"""
import torch
import torch.nn as nn

from . import _native as nat


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean", scale=1.0):
    """Cross entropy of ``scale * hidden @ weight.T`` against ``target``, in float32.

    hidden [..., D] and weight [V, D] of one type (float32, float16 or bfloat16),
    target [...] int64.  Rows with ``ignore_index`` have loss and gradient 0,
    whatever hidden holds there; "mean" divides by the others' number (NaN if there is none).  A
    target outside the vocabulary makes its row's loss NaN, and its row of hidden's
    gradient and all of weight's, unless that loss's upstream gradient is 0:
    nothing is read back to raise for it.  scale > 0 (an inverse temperature).
    The gradients have the inputs' type; their sums are kept in 32 bits.  Of 16-bit
    inputs the gradient of the logits is rounded to their type before its products, but for the
    target's part against a frozen weight and for all of it of up to 8 rows (and 2048 columns).  In
    float16 use a loss scale, as for any float16 training: gradients below 6e-8 are 0.
    Gradients of second order and forward-mode derivatives are not available, and raise."""
    return nat.head().linear_cross_entropy(hidden, weight, target, ignore_index, reduction, scale)


class LinearCrossEntropy(nn.Module):
    """``linear_cross_entropy`` with a weight of its own: ``forward(hidden, target)``."""

    def __init__(self, dim, vocab, ignore_index=-100, reduction="mean", scale=1.0, device=None, dtype=None):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(vocab, dim, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=dim ** -0.5)
        self.ignore_index, self.reduction, self.scale = ignore_index, reduction, scale

    def forward(self, hidden, target):
        return linear_cross_entropy(hidden, self.weight, target, self.ignore_index, self.reduction, self.scale)
