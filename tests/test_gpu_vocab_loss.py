"""linear_cross_entropy (po_linear_ce_fwd / _bwd) against the definition in 64 bits.

Tolerances, from the arithmetic:
 - a logit is a sum of D exact products in 32 bits: off by at most
   eL = (D + 4) * 2^-23 * max_nv sum_k |h w| * scale (fp32 inputs: their three-plane
   products leave out another 2^-22 of each product);
 - a loss takes eL twice (its sum and its target), the sums of exponentials (a lane's
   chain of up to 128 terms, tiles, 2^-23 each), exp2 and log2 (2^-22) and
   arguments of up to 64: 4e-5 in all;
 - a term of dl is off by (2 eL + 1e-4) of its exponential's part, is then rounded to 16
   bits (eps / 2; fp32: 2^-23), and the gradients add their terms in 32 bits
   (length * 2^-23) and are rounded once (eps / 2; half of fp16's smallest
   number).  fp16's dl are kept times 2^14 / max|g|, half their smallest number is
   2^-39 of max|g|."""
import math

import pytest
import torch

from conftest import pkg_mod

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = (torch.float32, torch.float16, torch.bfloat16)
IGN = -100


def inputs(N, V, D, dtype, seed=0, ignored=0.1, dev=DEV):
    g = torch.Generator(device=dev).manual_seed(seed + 1000 * N + 10 * V + D)
    h = torch.randn(N, D, generator=g, device=dev).to(dtype)
    w = (torch.randn(V, D, generator=g, device=dev) / math.sqrt(D) * 1.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[torch.rand(N, generator=g, device=dev) < ignored] = IGN
    return h, w, t


def reference(h, w, t, g=None, scale=1.0):
    """loss [N], and for g [N] = dL/dloss: dh, dw, and the elementwise bounds' sums, all in 64 bits."""
    live = t != IGN
    h64, w64 = torch.where(live[:, None], h.double(), 0.0), w.double()
    logits = scale * (h64 @ w64.t())
    pick = torch.where(live, t, 0)[:, None]
    lse = torch.logsumexp(logits, 1)
    out = {"loss": torch.where(live, lse - logits.gather(1, pick)[:, 0], 0.0)}
    out["S"] = scale * float((h64.abs() @ w64.abs().t()).max())
    if g is not None:
        p = torch.exp(logits - lse[:, None]) * (g.double() * live)[:, None]
        dl = p.clone()
        dl.scatter_add_(1, pick, -(g.double() * live)[:, None])
        dl, p = scale * dl, scale * p.abs()
        out.update(dh=dl @ w64, dw=dl.t() @ h64, ah=p @ w64.abs(), aw=p.t() @ h64.abs(), rh=dl.abs() @ w64.abs(),
                   rw=dl.abs().t() @ h64.abs(), wsum=w64.abs().sum(0), hsum=h64.abs().sum(0), gmax=scale * float((g.abs() * live).max()))
    return out


def bounds(ref, dtype, N, V, D):
    eps = 2.0 ** -22 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    eL = (D + 4) * 2.0 ** -23 * ref["S"] + (2.0 ** -22 * ref["S"] if dtype == torch.float32 else 0.0)
    b = {"loss": 2 * eL + 4e-5}
    if "dh" in ref:
        tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
        under = 2.0 ** -39 * ref["gmax"] if dtype == torch.float16 else 0.0
        for d, a, r, s, n in (("dh", "ah", "rh", "wsum", V), ("dw", "aw", "rw", "hsum", N)):
            b[d] = (2 * eL + 1e-4) * ref[a] + (eps + (n + 4) * 2.0 ** -23) * ref[r] + \
                torch.finfo(dtype).eps / 2 * ref[d].abs() + tiny + under * ref[s]
    return b


def within(got, ref, tol, what):
    d = (got.double() - ref).abs() - tol
    assert not torch.isnan(d).any(), what
    assert float(d.max()) <= 0, "%s: %.3g over a bound of %.3g" % (what, float(d.max()), float(torch.as_tensor(tol).max()))


SIZES = [(1, 1, 1), (1, 2, 3), (2, 7, 8), (3, 255, 40), (5, 257, 64), (31, 300, 65), (32, 128, 128), (33, 129, 72), (64, 1000, 33),
         (127, 513, 136), (129, 2049, 200), (130, 100, 520), (257, 1030, 96), (300, 700, 1001), (1000, 300, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", SIZES)
def test_losses_and_gradients(N, V, D, dtype):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype)
    h.requires_grad_()
    w.requires_grad_()
    g = torch.randn(N, device=DEV) * (64 if dtype == torch.float16 else 1)
    ref = reference(h.detach(), w.detach(), t, g)
    b = bounds(ref, dtype, N, V, D)
    loss = lce(h, w, t, reduction="none")
    assert loss.dtype == torch.float32 and loss.shape == t.shape
    within(loss.detach(), ref["loss"], b["loss"], "loss")
    assert not loss[t == IGN].any()
    loss.backward(g)
    assert h.grad.dtype == w.grad.dtype == dtype
    within(h.grad, ref["dh"], b["dh"], "dh")
    within(w.grad, ref["dw"], b["dw"], "dw")
    assert not h.grad[t == IGN].any()


@pytest.mark.parametrize("N,V,D", [(17, 300, 2056), (20, 5001, 2100), (24, 150001, 1032), (40, 3001, 1123), (65, 2000, 264), (128, 777, 96), (129, 4000, 3001),
                                   (192, 2049, 640), (193, 2049, 640), (192, 33, 8)])
@pytest.mark.parametrize("frozen", ["", "hidden", "weight"])
def test_fp32_of_few_tokens(N, V, D, frozen):
    """The fp32 matrix instructions, rows that serve as they are and others, more than one piece, and the next size."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, torch.float32)
    t[1] = IGN
    h[1] = float("nan")
    t[N - 1] = V - 1
    h.requires_grad_(frozen != "hidden")
    w.requires_grad_(frozen != "weight")
    g = 0.5 + torch.arange(N, device=DEV) % 7 / 7
    loss = lce(h, w, t, reduction="none")
    leaves = [x for x in (h, w) if x.requires_grad]
    grads = torch.autograd.grad(loss, leaves, g)
    ref = reference(h.detach(), w.detach(), t, g)
    b = bounds(ref, torch.float32, N, V, D)
    within(loss.detach(), ref["loss"], b["loss"], "loss")
    for x, got in zip(leaves, grads):
        within(got, ref["dh" if x is h else "dw"], b["dh" if x is h else "dw"], "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(1100, 9001, 513), (2050, 16001, 385), (700, 33001, 520), (300, 20000, 1030)])
def test_large_tiles(N, V, D, dtype):
    """Sizes of whole rounds of the largest tiles with ragged ends, the rest in smaller ones, k cut in slices."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype)
    h.requires_grad_()
    w.requires_grad_()
    g = (64.0 if dtype == torch.float16 else 1.0) * (0.5 + torch.arange(N, device=DEV) % 7 / 7)
    loss = lce(h, w, t, reduction="none")
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    ref = reference(h.detach(), w.detach(), t, g)
    b = bounds(ref, dtype, N, V, D)
    within(loss.detach(), ref["loss"], b["loss"], "loss")
    within(dh, ref["dh"], b["dh"], "dh")
    within(dw, ref["dw"], b["dw"], "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(1, 9001, 793), (1, 33, 2048), (2, 5000, 2047), (3, 7, 5), (4, 1999, 256), (6, 12345, 300), (8, 4096, 512),
                                   (9, 2222, 1024), (13, 8191, 1025), (16, 5001, 2000), (16, 100000, 64), (16, 50, 2049), (17, 3000, 640)])
@pytest.mark.parametrize("frozen", ["", "hidden", "weight"])
def test_few_rows(N, V, D, frozen, dtype):
    """One pass over the vocabulary, its ends in rows and columns; rows that take no part hold NaN."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype)
    if N > 2:
        t[1] = IGN
        h[1] = float("nan")
    if N > 1:
        t[N - 1] = V - 1
    h.requires_grad_(frozen != "hidden")
    w.requires_grad_(frozen != "weight")
    g = (64.0 if dtype == torch.float16 else 1.0) * (0.5 + torch.arange(N, device=DEV) % 7 / 7)
    loss = lce(h, w, t, reduction="none")
    leaves = [x for x in (h, w) if x.requires_grad]
    grads = torch.autograd.grad(loss, leaves, g, retain_graph=True)
    ref = reference(h.detach(), w.detach(), t, g)
    b = bounds(ref, dtype, N, V, D)
    within(loss.detach(), ref["loss"], b["loss"], "loss")
    for x, d, got in zip(leaves, ["dh", "dw"] if len(leaves) == 2 else ["dw" if frozen == "hidden" else "dh"], grads):
        within(got, ref[d], b[d], d)
        if N <= 8 and D <= 2048 and dtype != torch.float32:
            # the gradient of the logits stays in 32 bits there: the one rounding to 16 is the gradient's own, at most half a step
            tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
            own = torch.finfo(dtype).eps / 2 * ref[d].abs() + tiny
            eL = (D + 4) * 2.0 ** -23 * ref["S"]
            a, r, n = (ref["ah"], ref["rh"], V) if d == "dh" else (ref["aw"], ref["rw"], N)
            within(got, ref[d], own + (2 * eL + 1e-4) * a + (n + 4) * 2.0 ** -23 * r, d + ", one rounding")
    for x, y in zip(grads, torch.autograd.grad(loss, leaves, g)):
        assert torch.equal(x, y)


def check_frozen(h, w, t, g, scale=1.0):
    """Loss and gradient against a frozen vocabulary.  Beside the other bounds: blocks of the vocabulary whose
    exponentials stay below 2^-48 of another's are left out of dh."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h = h.detach().requires_grad_()
    loss = lce(h, w, t, reduction="none", scale=scale)
    (dh,) = torch.autograd.grad(loss, h, g, retain_graph=True)
    ref = reference(h.detach(), w, t, g, scale)
    b = bounds(ref, h.dtype, h.shape[0], w.shape[0], h.shape[1])
    within(loss.detach(), ref["loss"], b["loss"] + 2.0 ** -23 * ref["loss"].abs(), "loss")
    within(dh, ref["dh"], b["dh"] + 2.0 ** -48 * ref["gmax"] * ref["wsum"], "dh")
    (again,) = torch.autograd.grad(loss, h, g)
    assert torch.equal(dh, again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", SIZES + [(1100, 9001, 513), (2050, 16001, 640), (300, 20000, 1030), (8192, 12001, 40)])
def test_frozen_vocabulary(N, V, D, dtype):
    h, w, t = inputs(N, V, D, dtype)
    check_frozen(h, w, t, (64.0 if dtype == torch.float16 else 1.0) * (0.5 + torch.arange(N, device=DEV) % 7 / 7))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(70, 5000, 40), (300, 3000, 200), (2100, 9000, 1000)])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_frozen_vocabulary_of_wide_logits(N, V, D, dtype, order):
    """Largest logits that differ by hundreds from one stretch of the vocabulary to the next, targets anywhere."""
    h, w, t = inputs(N, V, D, dtype)
    amp = torch.linspace(0.0, 60.0, V // 128 + 1, device=DEV)
    if order == "down":
        amp = amp.flip(0)
    elif order == "mixed":
        amp = amp[torch.randperm(len(amp), generator=torch.Generator(device=DEV).manual_seed(N), device=DEV)]
    w = (w.float() * amp[torch.arange(V, device=DEV) // 128][:, None]).to(dtype)
    check_frozen(h, w, t, torch.full((N,), 64.0 if dtype == torch.float16 else 1.0, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
def test_frozen_vocabulary_fitted(dtype):
    """Probabilities of the targets next to 1: what is left of them is the gradient."""
    N, V, D = 260, 2000, 64
    h, w, t = inputs(N, V, D, dtype)
    h = (w.float()[t.clamp(min=0)] * torch.linspace(1.0, 40.0, N, device=DEV)[:, None]).to(dtype)
    check_frozen(h, w, t, torch.full((N,), 1024.0 if dtype == torch.float16 else 1.0, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(5, 900, 64), (200, 900, 64), (3000, 9000, 768)])
@pytest.mark.parametrize("mode", ["plain", "frozen", "both"])
def test_small_losses(N, V, D, mode, dtype):
    """With p next to 1 a loss is log(1 + rest): an error of the logits, and of the exponentials, counts as much as the
    rest does, and what is left are the roundings of log2, of 1 + rest and of the target's exponent (an ulp of 1 each)."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype, ignored=0.0)
    w = (w.float() / w.float().norm(dim=1, keepdim=True)).to(dtype)
    h = (w.float()[t] * torch.linspace(14.0, 40.0, N, device=DEV)[:, None]).to(dtype)
    x = h.clone().requires_grad_(mode != "plain")
    loss = lce(x, w.clone().requires_grad_(mode == "both"), t, reduction="none")
    ref = reference(h, w, t)
    b = bounds(ref, dtype, N, V, D)["loss"]
    within(loss.detach(), ref["loss"], -torch.expm1(-ref["loss"]) * b + 3 * 2.0 ** -23, "loss")
    if mode != "plain":
        (dh,) = torch.autograd.grad(loss, x, torch.full((N,), 64.0, device=DEV))
        ref = reference(h, w, t, torch.full((N,), 64.0, device=DEV))
        rest = -torch.expm1(-ref["loss"])[:, None]
        # the target's part, 64 (1 - p) w, is as exact as 1 - p; the others' terms are off by their roundings
        tol = (bounds(ref, dtype, N, V, D)["dh"] - (2 * (b - 4e-5) / 2 + 1e-4) * ref["ah"]).clamp(min=0) + \
            64 * (2 * b * rest + 4 * 2.0 ** -23) * w[t].double().abs() + (2 * b + 1e-4) * (ref["rh"] + 64 * 2.0 ** -48 * ref["wsum"])
        within(dh, ref["dh"], tol, "dh")


@pytest.mark.parametrize("N,V,D", [(90, 700, 64), (2600, 9000, 768)])        # below and above the size that takes a common base
def test_frozen_vocabulary_of_infinite_logits(N, V, D):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, torch.bfloat16)
    w[5], w[V - 2] = 0, 0
    h[:, 0] = 1
    w[:, 0] = 0
    w[5, 0] = -float("inf")                                     # probability 0
    t = torch.where((t == 5) | (t == V - 2), 6, t)
    t[1], t[2], t[3] = 5, V - 2, IGN
    h[4, 1] = float("nan")
    h[4:6, 0] = 1
    x = h.clone().requires_grad_()
    loss = lce(x, w, t, reduction="none")
    plain = lce(h, w, t, reduction="none")
    assert torch.isnan(loss[4]) and torch.isnan(plain[4]) and float(loss[1]) == float("inf") == float(plain[1])
    (dh,) = torch.autograd.grad(loss[torch.arange(N, device=DEV) != 1].sum(), x)
    # 0 * inf in column 0, where the vocabulary is infinite; the rest is the formula's
    live = torch.isfinite(loss.detach()) & (t != IGN)
    assert torch.isfinite(dh[live][:, 1:]).all() and torch.isnan(dh[4]).all() and not dh[3].any() and not dh[1].any()
    w[7, 0] = float("inf")
    x = h.clone().requires_grad_()
    loss = lce(x, w, t, reduction="none")
    assert torch.isnan(loss[t != IGN]).all() and not loss[3].any()
    (dh,) = torch.autograd.grad(loss.sum(), x)
    assert torch.isnan(dh[t != IGN]).all() and not dh[3].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("frozen,N", [("", 150), ("hidden", 150), ("weight", 150), ("", 1), ("", 40), ("weight", 640), ("", 2500)])
def test_reductions_and_frozen_sides(dtype, reduction, frozen, N):
    V, D = 777, 56
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype, ignored=0.3 if N > 1 else 0.0)
    live = t != IGN
    up = -512.0 if N == 40 else 512.0
    each = up / (int(live.sum()) if reduction == "mean" else 1)
    ref = reference(h, w, t, torch.full((N,), each, device=DEV), scale=2.5)
    b = bounds(ref, dtype, N, V, D)
    h.requires_grad_(frozen != "hidden")
    w.requires_grad_(frozen != "weight")
    loss = lce(h, w, t, reduction=reduction, scale=2.5)
    total = ref["loss"].sum() / (int(live.sum()) if reduction == "mean" else 1)
    assert loss.shape == ()
    within(loss.detach(), total, b["loss"] * (1 if reduction == "mean" else N) + abs(float(total)) * 2.0 ** -23, "loss")
    (loss * up).backward()
    for m, d in ((h, "dh"), (w, "dw")):
        if m.requires_grad:
            within(m.grad, ref[d], b[d], d)
        else:
            assert m.grad is None


@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces_of_the_vocabulary(dtype):
    """Sizes at which the backward pass walks more than one piece, the last one ragged."""
    N, V, D = (8192, 12001, 40) if dtype == torch.float32 else (8192, 39999, 72)
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype)
    h.requires_grad_()
    w.requires_grad_()
    g = torch.rand(N, device=DEV) + 0.5
    ref = reference(h.detach(), w.detach(), t, g)
    b = bounds(ref, dtype, N, V, D)
    loss = lce(h, w, t, reduction="none")
    within(loss.detach(), ref["loss"], b["loss"], "loss")
    dh, dw = torch.autograd.grad(loss, (h, w), g, retain_graph=True)
    within(dh, ref["dh"], b["dh"], "dh")
    within(dw, ref["dw"], b["dw"], "dw")
    again = torch.autograd.grad(loss, (h, w), g)
    assert torch.equal(again[0], dh) and torch.equal(again[1], dw)        # sums in one order


@pytest.mark.parametrize("dtype", TYPES)
def test_long_rows_of_many_tokens(dtype):
    """Sizes at which every product takes its largest tile, ragged on all sides."""
    N, V, D = 4090, 8190, 2052
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype)
    h.requires_grad_()
    w.requires_grad_()
    g = (torch.rand(N, device=DEV) + 0.5) * (64 if dtype == torch.float16 else 1)
    ref = reference(h.detach(), w.detach(), t, g)
    b = bounds(ref, dtype, N, V, D)
    loss = lce(h, w, t, reduction="none")
    within(loss.detach(), ref["loss"], b["loss"], "loss")
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    within(dh, ref["dh"], b["dh"], "dh")
    within(dw, ref["dw"], b["dw"], "dw")
    # the elementwise bounds are worst cases of 2052 terms; in the mean the roundings are random: a gradient's
    # norm is off by its two roundings to 16 bits (dl's and its own), each eps / 2 / sqrt(3) rms at most, fp32's by
    # the sums' (a walk of 2^-24 steps over up to 8190 terms: 6e-6)
    tol = 6e-6 if dtype == torch.float32 else 2 * torch.finfo(dtype).eps / 2 / 3 ** 0.5
    for got, want in ((dh, ref["dh"]), (dw, ref["dw"])):
        assert float((got.double() - want).norm() / want.norm()) < tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(70, 300, 64), (4200, 5000, 840)])
def test_frozen_vocabulary_where_ignored_rows_hold_anything(N, V, D, dtype):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype, ignored=0.4)
    clean = h.clone()
    bad = (t == IGN).nonzero()[:, 0]
    h[bad[0::3]] = float("nan")
    h[bad[1::3]] = float("inf")
    h[bad[2::3]] = torch.finfo(dtype).min
    out = []
    for x in (h, clean):
        x = x.clone().requires_grad_()
        loss = lce(x, w, t)
        out.append((loss.detach(),) + torch.autograd.grad(loss * 256, x))
    for a, b in zip(*out):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert not out[0][1][bad].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_ignored_rows_may_hold_anything(dtype):
    N, V, D = 70, 300, 64
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype, ignored=0.4)
    clean = h.clone()
    bad = (t == IGN).nonzero()[:, 0]
    h[bad[0::3]] = float("nan")
    h[bad[1::3]] = float("inf")
    h[bad[2::3]] = torch.finfo(dtype).min
    out = []
    for x in (h, clean):
        x, y = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = lce(x, y, t)
        out.append((loss.detach(),) + torch.autograd.grad(loss * 256, (x, y)))
    for a, b in zip(*out):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_nothing_but_ignored_rows_and_no_rows(reduction):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    for N in (5, 0):
        h = torch.randn(N, 16, device=DEV, requires_grad=True)
        w = torch.randn(20, 16, device=DEV, requires_grad=True)
        loss = lce(h, w, torch.full((N,), IGN, device=DEV), reduction=reduction)
        if reduction == "mean":
            assert torch.isnan(loss)
        else:
            assert loss.shape == ((N,) if reduction == "none" else ()) and not loss.detach().any()
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert not dh.any() and not dw.any() and dh.shape == h.shape and dw.shape == w.shape


def test_another_ignore_index_and_targets_outside():
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(20, 50, 16, torch.float32, ignored=0.0)
    t[3:6] = 7
    loss = lce(h, w, t, ignore_index=7, reduction="none")
    ref = reference(h, w, torch.where(t == 7, IGN, t))
    within(loss, ref["loss"], bounds(ref, torch.float32, 20, 50, 16)["loss"], "loss")
    for bad in (50, -1, 1 << 40, -(1 << 40)):
        u = t.clone()
        u[0] = bad
        loss = lce(h, w, u, ignore_index=7, reduction="none")
        assert torch.isnan(loss[0]) and torch.isfinite(loss[1:]).all()
        assert torch.isnan(lce(h, w, u, ignore_index=7))
        x = h.clone().requires_grad_()
        (dh,) = torch.autograd.grad(lce(x, w, u, ignore_index=7, reduction="sum"), x)
        assert torch.isnan(dh[0]).all() and torch.isfinite(dh[1:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_shapes(dtype):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    N, V, D = 60, 200, 48
    h0, w0, t = inputs(N, V, D, dtype)
    g = torch.randn(N, device=DEV)

    def grads(h, w, target=t, up=g):
        loss = lce(h, w, target, reduction="none")
        return (loss.detach(),) + torch.autograd.grad(loss, (h, w), up)

    want = grads(h0.clone().requires_grad_(), w0.clone().requires_grad_())
    wide_h, wide_w = torch.zeros(N, 200, dtype=dtype, device=DEV), torch.zeros(V, 77, dtype=dtype, device=DEV)
    for off in (0, 1, 8, 13):
        wide_h.fill_(float("nan"))
        wide_w.fill_(float("nan"))
        hv, wv = wide_h[:, off:off + D], wide_w[:, off:off + D]
        hv.copy_(h0)
        wv.copy_(w0)
        for a, b in zip(grads(hv.detach().requires_grad_(), wv.detach().requires_grad_()), want):
            assert torch.equal(a, b)
    ht, wt = h0.t().contiguous().t().requires_grad_(), w0.t().contiguous().t().requires_grad_()
    for a, b in zip(grads(ht, wt), want):
        assert torch.equal(a, b)
    h3, t3 = h0.view(5, 12, D).clone().requires_grad_(), t.view(5, 12)
    got = grads(h3, w0.clone().requires_grad_(), t3, g.view(5, 12))
    assert got[0].shape == (5, 12) and got[1].shape == h3.shape
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    one = lce(h0[0], w0, torch.tensor(3, device=DEV))
    assert one.shape == () and torch.equal(one, lce(h0[:1], w0, torch.tensor([3], device=DEV)))


def test_expanded_inputs_get_summed_gradients():
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h1 = torch.randn(1, 40, device=DEV, requires_grad=True)
    w = torch.randn(90, 40, device=DEV) / 6
    t = torch.randint(0, 90, (17,), device=DEV)
    (dh,) = torch.autograd.grad(lce(h1.expand(17, 40), w, t, reduction="sum"), h1)
    ref = reference(h1.detach().expand(17, 40), w, t, torch.ones(17, device=DEV))
    b = bounds(ref, torch.float32, 17, 90, 40)
    within(dh, ref["dh"].sum(0, keepdim=True), b["dh"].sum(0, keepdim=True) + 1e-5, "dh")


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits_stay_finite(dtype):
    """Logits of +-2e4: only the differences to a row's largest matter."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    N, V, D = 40, 500, 16
    h, w, t = inputs(N, V, D, dtype)
    h = (h * 64).to(dtype).requires_grad_()
    w = (w * 64).to(dtype).requires_grad_()
    ref = reference(h.detach(), w.detach(), t, torch.ones(N, device=DEV))
    eL = (D + 4) * 2.0 ** -23 * ref["S"]
    loss = lce(h, w, t, reduction="none")
    # the loss is as large as the logits' spread: its own rounding too
    within(loss.detach(), ref["loss"], 2 * eL + 4e-5 + ref["loss"] * 2.0 ** -21, "loss")
    dh, dw = torch.autograd.grad(loss.sum(), (h, w))
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("N,frozen", [(3, False), (140, True)])
def test_a_vocabulary_past_4_gib(N, frozen):
    """2.2e9 weights; the reference walks them in 64 bits, piece by piece."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    V, D = 2_150_000, 1032
    g = torch.Generator(device=DEV).manual_seed(N)
    w = (torch.randn(V, D, generator=g, device=DEV, dtype=torch.bfloat16) / 32).requires_grad_(not frozen)
    h = torch.randn(N, D, generator=g, device=DEV).bfloat16().requires_grad_()
    t = torch.randint(0, V, (N,), generator=g, device=DEV)
    t[0], t[-1] = V - 1, 2_100_000
    parts = [(a, min(V, a + 250_000)) for a in range(0, V, 250_000)]
    w64 = lambda a, b: w.detach()[a:b].double()          # noqa: E731
    h64 = h.detach().double()
    lse = torch.logsumexp(torch.stack([torch.logsumexp(h64 @ w64(a, b).t(), 1) for a, b in parts]), 0)
    loss = lce(h, w, t, reduction="none")
    want = lse - (h64 * w.detach()[t].double()).sum(1)
    within(loss.detach(), want, 2 * (D + 4) * 2.0 ** -23 * 60 + 4e-5, "loss")     # sums of |h w| up to 60
    grads = torch.autograd.grad(loss.sum(), [h] if frozen else [h, w])
    dh = -w.detach()[t].double()
    for a, b in parts:
        dh += torch.exp(h64 @ w64(a, b).t() - lse[:, None]) @ w64(a, b)
    # the target's embedding dominates; roundings of 2^-8 to it and to each of the terms
    assert float((grads[0].double() - dh).norm() / dh.norm()) < 2.0 ** -8
    if not frozen:
        for v in (0, 1_040_000, int(t[-1]), int(t[0])):
            p = torch.exp(h64 @ w.detach()[v].double() - lse) - (t == v).double()
            ref = p @ h64
            assert float((grads[1][v].double() - ref).norm() / ref.norm()) < 2.0 ** -7


def test_infinite_logits_are_what_the_formula_says():
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h = torch.ones(3, 8, device=DEV)
    w = torch.zeros(300, 8, device=DEV)
    w[5, 0] = -float("inf")                     # probability 0
    t = torch.tensor([0, 299, 5], device=DEV)
    loss = lce(h, w, t, reduction="none")
    want = math.log(299.0)
    assert abs(float(loss[0]) - want) < 1e-5 and abs(float(loss[1]) - want) < 1e-5 and float(loss[2]) == float("inf")
    w[7, 0] = float("inf")
    assert torch.isnan(lce(h, w, t, reduction="none")).all()
    assert torch.isnan(lce(h, torch.full_like(w, -float("inf")), t, reduction="none")).all()


@pytest.mark.parametrize("N", [9, 40])
def test_gradients_of_second_order_are_refused(N):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, 30, 16, torch.float32)
    h.requires_grad_()
    first = torch.autograd.grad(lce(h, w, t), h)[0]
    (dh,) = torch.autograd.grad(lce(h, w, t), h, create_graph=True)
    assert torch.equal(dh, first)               # the first order itself is there
    with pytest.raises(RuntimeError, match="second order"):
        torch.autograd.grad(dh.sum(), h)


@pytest.mark.parametrize("N", [7, 200])
def test_gradient_against_differences(N):
    """(L(h + e u) - L(h - e u)) / 2e = dh . u + e^2 / 6 L'''; with a = max |w . u| the third cumulant is
    at most (2a)^3, and a loss is off by its own bound."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    V, D = 400, 32
    h, w, t = inputs(N, V, D, torch.float32)
    ref = reference(h, w, t, torch.ones(N, device=DEV))
    b = bounds(ref, torch.float32, N, V, D)["loss"]
    h.requires_grad_()
    w.requires_grad_()
    dh, dw = torch.autograd.grad(lce(h, w, t, reduction="sum"), (h, w))
    e = 2.0 ** -5
    # directions of one length, a = 1, so that the bound (and what the check says) hangs on no draw
    g = torch.Generator(device=DEV).manual_seed(N)
    u = torch.randn(N, D, generator=g, device=DEV)
    v = torch.randn(V, D, generator=g, device=DEV)
    u = u / (u @ w.detach().t()).abs().max()
    v = v / (h.detach() @ v.t()).abs().max()
    a = 1 + 1e-5
    for first, num in (
            ((dh.double() * u).sum(1), lambda s: lce(h + s * u, w, t, reduction="none").detach()),
            ((dw.double() * v).sum(), lambda s: lce(h, w + s * v, t, reduction="sum").detach())):
        d = (num(e).double() - num(-e).double()) / (2 * e)
        rows = N if d.dim() == 0 else 1
        tol = rows * (e * e / 6 * (2 * a) ** 3 + (b + 1e-5) / e)
        want = first if d.dim() == 0 else first          # a row's loss depends on its own h alone
        assert float((d - want).abs().max()) <= tol
        assert tol < 0.2 * max(rows, 1)                   # the check says something


@pytest.mark.parametrize("N,V,D,frozen", [(130, 600, 64, False), (130, 600, 64, True), (2600, 9000, 768, True), (5, 600, 64, False), (1, 600, 64, True)])
def test_forward_and_backward_in_a_replayed_graph(N, V, D, frozen):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, torch.bfloat16)
    h.requires_grad_()
    w.requires_grad_(not frozen)

    def step():
        loss = lce(h, w, t)
        return (loss,) + torch.autograd.grad(loss, (h,) if frozen else (h, w))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):                                    # two graphs: workspaces of their own
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for k in range(3):
        nh, nw, nt = inputs(N, V, D, torch.bfloat16, seed=77 + k)
        with torch.no_grad():
            h.copy_(nh)
            w.copy_(nw)
        t.copy_(nt)
        want = [x.detach().clone() for x in step()]
        for gr, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a.detach(), b)


def test_a_capture_while_an_eager_graph_holds_the_leaves_is_refused():
    """The eager graph's accumulators belong to its stream; capturing a backward pass into them would end the
    process.  The call raises inside the capture, and both go on after it."""
    lce, kd = pkg_mod("vocab_loss").linear_cross_entropy, pkg_mod("keyed_dropout").keyed_dropout
    h, w, t = inputs(60, 400, 40, torch.float32)
    h.requires_grad_()
    w.requires_grad_()
    want = torch.autograd.grad(lce(h, w, t), (h, w))
    eager = lce(h, w, t)
    for call in (lambda: lce(h, w, t), lambda: lce(h.detach(), w, t), lambda: kd(h, 0.5, 1), lambda: kd(h.detach(), 0.5, 1, residual=h)):
        with pytest.raises(RuntimeError, match="outside this capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    late = torch.autograd.grad(eager, (h, w))
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(lce(h, w, t), (h, w))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(got, late, want):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_two_streams_at_once_and_repeats_are_equal():
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    sets = [inputs(260, 3000, 128, torch.bfloat16, seed=k) for k in range(2)]

    def go(k):
        h, w, t = sets[k]
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        loss = lce(h, w, t, reduction="none")
        return (loss.detach(),) + torch.autograd.grad(loss.sum(), (h, w))

    want = [go(0), go(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for k, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[k] = go(k)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
