"""The large-vocabulary head as it is used: trained behind keyed dropout with the
linear cross entropy, then served with its weights in 8 bits.  Gradients are held
to the same chain in 64 bits with the mask that the kernels drew."""
import pytest
import torch

from conftest import pkg_mod
from test_gpu_dropout import keep_ref
from test_gpu_int8 import check_product, quant_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_train_then_serve():
    kd, vl, i8 = pkg_mod("keyed_dropout"), pkg_mod("vocab_loss"), pkg_mod("int8_linear")
    N, V, D, p = 200, 1500, 96, 0.25
    torch.manual_seed(5)
    body = torch.nn.Linear(40, D).to(DEV)
    drop = kd.KeyedDropout(p, seed=123)
    head = vl.LinearCrossEntropy(D, V, device=DEV)
    opt = torch.optim.SGD(list(body.parameters()) + list(head.parameters()), lr=0.5)
    x = torch.randn(N, 40, device=DEV)
    res = torch.randn(N, D, device=DEV)
    t = torch.randint(0, V, (N,), device=DEV)
    t[::9] = -100
    for step in range(3):
        drop.step = step
        z = body(x)
        z.retain_grad()
        loss = head(drop(z, residual=res), t)
        opt.zero_grad()
        loss.backward()
        # the same step in 64 bits
        keep = keep_ref(N, D, p, 123, step).to(DEV)
        z64 = z.detach().double().requires_grad_()
        w64 = head.weight.detach().double().requires_grad_()
        y64 = torch.where(keep, z64 / (1 - p), 0.0) + res.double()
        logits = y64 @ w64.t()
        live = t != -100
        l64 = torch.nn.functional.cross_entropy(logits[live], t[live])
        l64.backward()
        assert abs(float(loss.detach()) - float(l64.detach())) < 1e-4
        # the operators' own tests hold single elements to their bounds; here the chain's norms, fp32 through
        # sums of up to 1500 terms: 1500 * 2^-23 of the terms' sizes is 2e-4
        for got, want in ((z.grad, z64.grad), (head.weight.grad, w64.grad)):
            assert float((got.double() - want).norm() / want.norm()) < 2e-4
        opt.step()
    drop.eval()
    served = i8.Int8Linear(head.weight)
    with torch.no_grad():
        y = drop(body(x), residual=res)
        logits = served(y)
    wq, ws = quant_ref(head.weight.detach())
    q, s = quant_ref(y)
    assert torch.equal(served.wq.cpu(), wq)
    check_product(logits, q, s, wq, ws, None, torch.float32)
    one = served(y[7])
    assert torch.equal(one, logits[7])


def test_a_captured_training_step_replays_with_new_masks():
    """Dropout's step on the device, loss and both gradients in one graph; every replay against the eager call."""
    kd, vl = pkg_mod("keyed_dropout"), pkg_mod("vocab_loss")
    N, V, D = 96, 700, 64
    h = torch.randn(N, D, device=DEV).bfloat16().requires_grad_()
    w = (torch.randn(V, D, device=DEV) / 8).bfloat16().requires_grad_()
    t = torch.randint(0, V, (N,), device=DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)

    def go(s):
        loss = vl.linear_cross_entropy(kd.keyed_dropout(h, 0.5, 9, s), w, t)
        return (loss,) + torch.autograd.grad(loss, (h, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go(step)
        step.add_(1)
    seen = []
    for k in range(4):
        graph.replay()
        want = go(k)
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(out, want))
        seen.append(float(out[0].detach()))
    assert len(set(seen)) == 4 and int(step) == 4
