"""CPU tests: the derivatives that the head's operators do not have are refused, and none is dropped
without a word.  The refusals come before a device is looked at."""
import warnings

import pytest
import torch
from torch.autograd import forward_ad

from conftest import pkg_mod

DUAL = "forward-mode"


def _calls():
    """Every operator with its differentiable arguments: name -> (call, those arguments)."""
    kd, vl, i8 = (pkg_mod(m) for m in ("keyed_dropout", "vocab_loss", "int8_linear"))
    x, w, t = torch.randn(3, 16), torch.randn(5, 16), torch.zeros(3, dtype=torch.int64)
    wq, q, ws, b, sx = torch.ones(5, 16, dtype=torch.int8), torch.ones(3, 16, dtype=torch.int8), torch.ones(5), torch.ones(5), torch.ones(3)
    return {
        "keyed_dropout": (lambda x, r: kd.keyed_dropout(x, 0.5, 1, residual=r), (x, x.clone())),
        "linear_cross_entropy": (lambda h, w: vl.linear_cross_entropy(h, w, t), (x, w)),
        "int8_linear": (lambda x, s, b: i8.int8_linear(x, wq, s, b), (x, ws, b)),
        "quantize_rows": (lambda x: i8.quantize_rows(x), (x,)),
        "int8_matmul": (lambda s, ws, b: i8.int8_matmul(q, s, wq, ws, b), (sx, ws, b)),
    }


@pytest.mark.parametrize("name", ["keyed_dropout", "linear_cross_entropy", "int8_linear", "quantize_rows", "int8_matmul"])
def test_forward_mode_is_refused(name):
    call, args = _calls()[name]
    for k in range(len(args)):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == k else a for i, a in enumerate(args)]
            with pytest.raises(RuntimeError, match=DUAL):
                call(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match=DUAL):       # which does not stop tangents
                call(*dual)
            # a dual level without a dual tensor, and a tangent that was taken off, are none
            for free in (args, [forward_ad.unpack_dual(a).primal for a in dual]):
                with pytest.raises(RuntimeError, match="CUDA"):
                    call(*free)


@pytest.mark.parametrize("name", ["int8_linear", "quantize_rows", "int8_matmul"])
def test_gradients_of_8_bit_products_are_refused(name):
    call, args = _calls()[name]
    for k in range(len(args)):
        grads = [a.clone().requires_grad_() if i == k else a for i, a in enumerate(args)]
        with pytest.raises(RuntimeError, match="no gradient"):
            call(*grads)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call(*grads)


def test_a_served_layer_says_that_it_cuts_the_graph():
    layer = pkg_mod("int8_linear").Int8Linear.__new__(pkg_mod("int8_linear").Int8Linear)
    torch.nn.Module.__init__(layer)
    layer.wq, layer.wscale, layer.bias = torch.ones(5, 16, dtype=torch.int8), torch.ones(5), None
    x = torch.randn(3, 16, requires_grad=True)
    with pytest.warns(UserWarning, match="cut off"), pytest.raises(RuntimeError, match="CUDA"):
        layer(x)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for y in (x.detach(), x):
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
                layer(y)
        with pytest.raises(RuntimeError, match="CUDA"):
            layer(x.detach())
        with pytest.raises(TypeError, match="x must"):
            layer([1.0] * 16)
