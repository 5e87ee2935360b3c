"""keyed_dropout (po_dropout) against a numpy restatement of its mask and 64-bit
arithmetic.

Tolerance: a kept element is x * s in 32 bits (one rounding, half a step 2^-24
of it), with a residual one more sum (2^-24 of the result), and one rounding to
the type (finfo.eps / 2 of the result; half the smallest subnormal where fp16
ends).  Which elements are dropped is compared exactly."""
import numpy as np
import pytest
import torch

from conftest import pkg_mod
from oracle.draws_ref import philox4x32_10

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TAG = 0x64726F70
TYPES = (torch.float32, torch.float16, torch.bfloat16)


def keep_ref(rows, cols, p, seed, step, row0=0):
    r = np.repeat(np.arange(rows, dtype=np.uint64) + row0, -(-cols // 8))
    g = np.tile(np.arange(-(-cols // 8), dtype=np.uint64), rows)
    w = philox4x32_10(g, r, step & 0xFFFFFFFF, step >> 32, seed & 0xFFFFFFFF, (seed >> 32) ^ TAG)
    u = np.stack(w, -1).astype("<u4").view("<u2").reshape(rows, -1)[:, :cols]
    return torch.from_numpy((u >= round(p * 65536)).astype(np.bool_))


def check(y, x, keep, p, residual=None):
    T = round(p * 65536)
    s = 65536.0 / (65536 - T) if T < 65536 else 0.0
    kept = x.double().cpu() * s
    ref = torch.where(keep, kept, torch.zeros_like(kept))
    tol = torch.where(keep, kept.abs(), torch.zeros_like(kept)) * 2.0 ** -23        # the product and the scale in 32 bits
    if residual is not None:
        ref = ref + residual.double().cpu()
        tol = tol + ref.abs() * 2.0 ** -24
    tol = tol + ref.abs() * torch.finfo(x.dtype).eps / 2 + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    y = y.double().cpu()
    assert torch.equal(y[~keep], ref[~keep].to(x.dtype).double()) if residual is not None else not y[~keep].any()
    assert bool(((y - ref).abs() <= tol).all()), float(((y - ref).abs() - tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (1, 8), (3, 9), (5, 64), (2, 1001), (257, 33), (1, 70000), (70000, 1), (64, 4096)])
@pytest.mark.parametrize("res", [False, True])
def test_forward_and_backward(dtype, rows, cols, res):
    kd = pkg_mod("keyed_dropout").keyed_dropout
    g = torch.Generator(device=DEV).manual_seed(rows * 131 + cols)
    x = torch.randn(rows, cols, generator=g, device=DEV).to(dtype).requires_grad_()
    r = torch.randn(rows, cols, generator=g, device=DEV).to(dtype).requires_grad_() if res else None
    dy = torch.randn(rows, cols, generator=g, device=DEV).to(dtype)
    p, seed, step = 0.3, (7 << 40) + 12345, (3 << 33) + 5
    keep = keep_ref(rows, cols, p, seed, step, row0=11)
    y = kd(x, p, seed, step, row0=11, residual=r)
    check(y.detach(), x.detach(), keep, p, None if r is None else r.detach())
    y.backward(dy)
    check(x.grad, dy, keep, p)
    if res:
        assert torch.equal(r.grad, dy)


@pytest.mark.parametrize("p", [0.0, 1e-6, 2.0 ** -16, 0.1, 0.5, 0.999999, 1.0])
def test_probabilities(p):
    kd = pkg_mod("keyed_dropout").keyed_dropout
    x = torch.randn(300, 500, device=DEV)
    y = kd(x, p, 1, 2)
    check(y, x, keep_ref(300, 500, p, 1, 2), p)
    if p in (0.0, 1e-6):
        assert torch.equal(y, x)             # below half a step of the probability's 2^-16
    if p in (0.999999, 1.0):
        assert not y.any()


def test_share_kept():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    n = 4 << 20
    kept = float((kd(torch.ones(1024, n // 1024, device=DEV), 0.1, 99, 7) != 0).double().mean())
    assert abs(kept - 0.9) < 6 * (0.09 / n) ** 0.5 + 2.0 ** -17


def test_dropped_places_may_hold_anything():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    keep = keep_ref(40, 72, 0.5, 3, 4)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min):
        x = torch.where(keep, torch.ones(()), torch.full((), bad)).to(DEV)
        y = kd(x, 0.5, 3, 4).cpu()
        assert torch.equal(y, 2.0 * keep.float())
        z = kd(torch.where(keep, torch.full((), bad), torch.ones(())).to(DEV), 0.5, 3, 4).cpu()
        assert not z[~keep].any() and not torch.isfinite(z[keep]).any()


def test_rows_of_a_shard_drop_what_the_whole_batch_drops():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    x = torch.randn(96, 40, device=DEV)
    whole = kd(x, 0.4, 5, 6)
    parts = [kd(x[a:a + 32], 0.4, 5, 6, row0=a) for a in (0, 32, 64)]
    assert torch.equal(whole, torch.cat(parts))
    last = (1 << 32) - 3
    check(kd(x[:3], 0.4, 5, 6, row0=last), x[:3], keep_ref(3, 40, 0.4, 5, 6, row0=last), 0.4)


def test_strides_offsets_and_shapes():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    base = torch.randn(50, 200, device=DEV, dtype=torch.float16)
    keep = {c: keep_ref(50, c, 0.25, 1, 1) for c in (64, 63, 200)}
    for v in (base[:, :64], base[:, 1:65], base[:, :63], base[:, 8:72]):
        check(kd(v, 0.25, 1, 1), v, keep[v.shape[1]], 0.25)
        check(kd(v, 0.25, 1, 1, residual=base[:, 100:100 + v.shape[1]]), v, keep[v.shape[1]], 0.25, base[:, 100:100 + v.shape[1]])
    t = torch.randn(200, 50, device=DEV)
    check(kd(t.t(), 0.25, 1, 1), t.t(), keep[200], 0.25)
    e = torch.randn(1, 64, device=DEV).expand(50, 64)
    check(kd(e, 0.25, 1, 1), e, keep[64], 0.25)
    x3 = torch.randn(5, 10, 63, device=DEV)
    assert torch.equal(kd(x3, 0.25, 1, 1).view(50, 63), kd(x3.view(50, 63), 0.25, 1, 1))
    v1 = torch.randn(63, device=DEV)
    assert torch.equal(kd(v1, 0.25, 1, 1), kd(v1[None], 0.25, 1, 1)[0])
    for shape in ((0, 8), (4, 0)):
        assert kd(torch.zeros(shape, device=DEV), 0.25, 1, 1).shape == shape


def test_offsets_past_32_bits():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    rows, cols = 65540, 32777                      # 2.15e9 elements, rows on odd places
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=DEV)
    y = kd(x, 0.5, 6, 7)
    for r in (0, 32767, 65534):
        check(y[r:r + 4], x[r:r + 4], keep_ref(4, cols, 0.5, 6, 7, row0=r), 0.5)
    assert y.view(-1)[2 ** 31 - 5:2 ** 31 + 5].float().max() <= 2.0


def test_gradient_of_a_broadcast_input_and_of_second_order():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    keep = keep_ref(50, 64, 0.5, 8, 9)
    b = torch.randn(64, device=DEV, requires_grad=True)
    y = kd(b.expand(50, 64), 0.5, 8, 9)
    (g,) = torch.autograd.grad((y * y).sum(), b, create_graph=True)
    n = keep.sum(0).to(DEV)
    assert torch.allclose(g, 8 * n * b, rtol=1e-5)
    (gg,) = torch.autograd.grad(g.sum(), b)
    assert torch.equal(gg, 8.0 * n)
    # differences: the map is linear, so they are exact up to the sums' rounding
    x = torch.randn(50, 64, device=DEV, requires_grad=True)
    u = torch.randn(50, 64, device=DEV)
    (gx,) = torch.autograd.grad(kd(x, 0.5, 8, 9), x, u)
    d = torch.randn(50, 64, device=DEV)
    num = ((kd(x + d, 0.5, 8, 9) - kd(x - d, 0.5, 8, 9)).double() * u.double()).sum() / 2
    assert abs(float(num - (gx.double() * d.double()).sum())) < 50 * 64 * 2.0 ** -21 * 16


def test_gradient_of_the_residual_alone_and_inference_mode():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    x, r, dy = (torch.randn(20, 33, device=DEV) for _ in range(3))
    r.requires_grad_()
    y = kd(x, 0.5, 2, 3, residual=r)
    y.backward(dy)
    assert torch.equal(r.grad, dy)
    with torch.inference_mode():
        assert torch.equal(kd(x, 0.5, 2, 3, residual=r), y)
    assert not kd(x, 0.5, 2, 3).requires_grad
    step = torch.tensor([3], device=DEV)
    xx = x.clone().requires_grad_()
    z = kd(xx, 0.5, 2, step, residual=r)
    step += 1
    (dx,) = torch.autograd.grad(z, xx, dy)
    check(dx, dy, keep_ref(20, 33, 0.5, 2, 3), 0.5)


def test_step_on_the_device_in_a_replayed_graph():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    x = torch.randn(33, 65, device=DEV, requires_grad=True)
    dy = torch.randn(33, 65, device=DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(kd(x, 0.5, 21, step), x, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kd(x, 0.5, 21, step)
        step.add_(1)                          # moved on before the backward pass, which keeps the forward's
        (dx,) = torch.autograd.grad(y, x, dy)
    for k in range(4):
        step.fill_(100 + 7 * k)
        graph.replay()
        torch.cuda.synchronize()
        keep = keep_ref(33, 65, 0.5, 21, 100 + 7 * k)
        check(y.detach(), x.detach(), keep, 0.5)
        check(dx, dy, keep, 0.5)
        assert int(step) == 101 + 7 * k
        torch.randn(1000, device=DEV).sum().item()


def test_on_another_stream():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    s = torch.cuda.Stream()
    x = torch.randn(64, 640, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = kd(x, 0.1, 4, 4)
    s.synchronize()
    check(y, x, keep_ref(64, 640, 0.1, 4, 4), 0.1)


def test_apart_from_the_draws_of_the_same_key():
    """The same seed and step give the transformer's noise other numbers than the mask."""
    w = philox4x32_10(np.arange(64), 0, 9, 0, 5, 0)
    v = philox4x32_10(np.arange(64), 0, 9, 0, 5, TAG)
    assert not np.array_equal(w[0], v[0])
