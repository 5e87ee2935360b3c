"""The head's operators at values and calls that reach few places: gradients that are not
finite, targets outside the vocabulary, weights that are infinite.  References and
bounds of the losses are test_gpu_vocab_loss.py's."""
import pytest
import torch

from conftest import pkg_mod
from test_gpu_vocab_loss import IGN, bounds, inputs, reference, within

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = (torch.float32, torch.float16, torch.bfloat16)
INF, NAN = float("inf"), float("nan")

# few rows' kernels, the smallest tiles (fp32: as it is), one piece in one slice, slices, and a size that
# takes a common base against a frozen vocabulary
HEADS = [(5, 900, 64), (20, 777, 56), (200, 900, 72), (300, 9001, 40), (2600, 9000, 768)]


def _loss_and_grads(h, w, t, up, frozen, reduction="none"):
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w = h.clone().requires_grad_(), w.clone().requires_grad_(not frozen)
    loss = lce(h, w, t, reduction=reduction)
    grads = torch.autograd.grad(loss, [h] if frozen else [h, w], up)
    return loss.detach(), grads[0], None if frozen else grads[1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", HEADS)
@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_one_rows_gradient_that_is_not_finite_stays_its_own(N, V, D, frozen, what, dtype):
    h, w, t = inputs(N, V, D, dtype)
    t[1], t[2], t[3] = 5, 6, IGN
    h[3] = NAN
    up = 0.5 + torch.arange(N, device=DEV) % 7 / 7
    ref = reference(h, w, t, up)                                # of finite gradients
    up[2] = what
    up[3] = what                                                # of a row that takes no part
    loss, dh, dw = _loss_and_grads(h, w, t, up, frozen)
    rest = torch.arange(N, device=DEV) != 2
    b = bounds(ref, dtype, N, V, D)
    within(dh[rest], ref["dh"][rest], (b["dh"] + 2.0 ** -48 * ref["gmax"] * ref["wsum"])[rest], "dh")
    assert not torch.isfinite(dh[2]).any() and not dh[t == IGN].any()
    assert dw is None or not torch.isfinite(dw).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", HEADS)
@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("what", [INF, NAN])
def test_a_sums_gradient_that_is_not_finite_leaves_ignored_rows(N, V, D, frozen, reduction, what, dtype):
    h, w, t = inputs(N, V, D, dtype)
    t[1], t[3] = 5, IGN
    h[3] = NAN
    loss, dh, dw = _loss_and_grads(h, w, t, torch.tensor(what, device=DEV), frozen, reduction)
    assert not dh[t == IGN].any() and not torch.isfinite(dh[t != IGN]).any()
    assert dw is None or not torch.isfinite(dw).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", HEADS)
@pytest.mark.parametrize("frozen", [False, True])
def test_infinite_weights_leave_ignored_rows(N, V, D, frozen, dtype):
    h, w, t = inputs(N, V, D, dtype)
    t[1], t[3] = 5, IGN
    w[7, 0], w[8, 0] = INF, NAN
    loss, dh, dw = _loss_and_grads(h, w, t, torch.tensor(1.0, device=DEV), frozen, "sum")
    assert not dh[t == IGN].any() and torch.isnan(dh[t != IGN]).all() and torch.isnan(loss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(1, 700, 48)] + HEADS)
@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("bad", ["below", "above", "far"])
def test_a_target_outside_the_vocabulary_is_its_rows_alone(N, V, D, frozen, bad, dtype):
    """Its loss, its row of dh and, since every row of dw takes its part, all of dw are NaN; with an upstream gradient
    of 0 it takes no part in the gradients."""
    h, w, t = inputs(N, V, D, dtype, ignored=0.1 if N > 1 else 0.0)
    row = N // 2
    t[row] = IGN                                                # the others' reference
    up = 0.5 + torch.arange(N, device=DEV) % 7 / 7
    ref = reference(h, w, t, up)
    b = bounds(ref, dtype, N, V, D)
    left_out = 2.0 ** -48 * ref["gmax"] * ref["wsum"]
    others = torch.arange(N, device=DEV) != row
    t[row] = {"below": -1, "above": V, "far": 1 << 40}[bad]
    for zero in (False, True):
        up[row] = 0.0 if zero else 0.75
        loss, dh, dw = _loss_and_grads(h, w, t, up, frozen)
        assert torch.isnan(loss[row])
        within(loss[others], ref["loss"][others], b["loss"], "loss") if N > 1 else None
        within(dh[others], ref["dh"][others], (b["dh"] + left_out)[others], "dh") if N > 1 else None
        if zero:
            assert not dh[row].any()
            if not frozen:
                within(dw, ref["dw"], b["dw"], "dw")
        else:
            assert torch.isnan(dh[row]).all() and (frozen or torch.isnan(dw).all())
    for reduction in ("sum", "mean"):
        loss, dh, dw = _loss_and_grads(h, w, t, torch.tensor(1.0, device=DEV), frozen, reduction)
        assert torch.isnan(loss) and torch.isnan(dh[row]).all() and not dh[t == IGN].any()
        assert torch.isfinite(dh[others]).all() and (frozen or torch.isnan(dw).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", HEADS)
@pytest.mark.parametrize("frozen", [False, True])
def test_gradients_of_large_logits(N, V, D, frozen, dtype):
    """Logits of hundreds: exponentials that underflow, targets that are far from the largest."""
    h, w, t = inputs(N, V, D, dtype)
    h = (h.float() * 40).to(dtype)
    up = (16.0 if dtype == torch.float16 else 1.0) * (0.5 + torch.arange(N, device=DEV) % 7 / 7)
    ref = reference(h, w, t, up)
    b = bounds(ref, dtype, N, V, D)
    loss, dh, dw = _loss_and_grads(h, w, t, up, frozen)
    assert float(ref["loss"].max()) > 100
    # arguments of hundreds: a loss and its exponents are rounded to a 2^-23 of their size
    more = 2.0 ** -23 * (ref["loss"].abs() + 2 * ref["S"])
    within(loss, ref["loss"], b["loss"] + more, "loss")
    within(dh, ref["dh"], b["dh"] + float(more.max()) * ref["ah"] + 2.0 ** -48 * ref["gmax"] * ref["wsum"], "dh")
    if not frozen:
        # an exponential below the smallest normal number, 2^-126, is 0, and so is an operand of the matrix cores: a
        # term of dl loses up to 2^-126 of its upstream gradient at each, which counts |h| times
        within(dw, ref["dw"], b["dw"] + float(more.max()) * ref["aw"] + 2 * 2.0 ** -126 * ref["gmax"] * ref["hsum"], "dw")


@pytest.mark.parametrize("K", [3, 40, 5000, 9000])
def test_rows_of_the_smallest_numbers_are_quantised_without_wrapping(K):
    """Row maxima of 1, 2, ... times 2^-149: their scales are whole multiples of 2^-149 as well, up to a third below
    the largest / 127, and the quotients end at 127."""
    m = pkg_mod("int8_linear")
    units = torch.cat([torch.arange(0, 2000), torch.tensor([127 * 127, 127 * 127 + 64, 20000, 65536, 1 << 22, (1 << 23) - 1])])
    R = len(units)
    bits = (torch.arange(K)[None, :] * 7919 + torch.arange(R)[:, None]) % (units[:, None] + 1)
    bits[:, 1] = units                                          # a row's largest
    bits = bits.int()
    bits[:, 2::2] |= -1 << 31                                   # every second number is negative
    bits[0::2, 1] |= -1 << 31                                   # and every second row's largest
    x = bits.view(torch.float32)
    s = (units.double() / 127).round() * 2.0 ** -149            # ties (63.5 and the like) go to the even one, torch.round's rule
    q = torch.where(s[:, None] > 0, torch.round(x.double() / s[:, None]), 0.0).clamp(-127, 127)
    assert float((units.double() * 2.0 ** -149 / s)[s > 0].max()) == 190 and float(q.abs().max()) == 127
    got_q, got_s = m.quantize_rows(x.to(DEV))
    assert torch.equal(got_s.cpu().double(), s) and torch.equal(got_q.cpu().double(), q)
    y = m.int8_linear(x[:4].to(DEV), torch.ones(2, K, dtype=torch.int8, device=DEV), torch.ones(2, device=DEV))
    assert torch.equal(y.cpu().double(), (q.sum(1) * s)[:4, None].expand(4, 2))
    y = m.int8_linear(x[160:162].to(DEV), torch.ones(2, K, dtype=torch.int8, device=DEV), torch.ones(2, device=DEV))
    assert torch.equal(y.cpu().double(), (q.sum(1) * s)[160:162, None].expand(2, 2))


@pytest.mark.parametrize("K", [16, 64, 50, 128])
@pytest.mark.parametrize("rows", [1, 2])
def test_product_of_rows_at_odd_places(K, rows):
    """One row is a matrix of any stride: a view off 16 bytes is copied, and its copy has a stride of its own."""
    m = pkg_mod("int8_linear")
    g = torch.Generator(device=DEV).manual_seed(K)
    buf = torch.randint(-128, 128, (7, 150), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-128, 128, (20, K), generator=g, device=DEV, dtype=torch.int8)
    s, ws = torch.rand(rows, generator=g, device=DEV) + 0.5, torch.ones(20, device=DEV)
    for r in (0, 3):
        for c in (0, 3, 16):
            q = buf[r:r + rows, c:c + K]
            y = m.int8_matmul(q, s, w, ws, dtype=torch.float32)
            assert torch.equal(y, (q.double() @ w.double().t()).float() * s[:, None])
            if rows == 1:
                assert torch.equal(m.int8_matmul(q[0], s[0], w, ws, dtype=torch.float32), y[0])


def _losses_of_a_few_tokens(h, w, t):
    """In 64 bits, the vocabulary in pieces; also the largest sum of a logit's products."""
    m = torch.full((len(h),), -INF, device=DEV, dtype=torch.float64)
    s, S = torch.zeros_like(m), 0.0
    for a in range(0, len(w), 1 << 24):
        x = h.double() @ w[a:a + (1 << 24)].double().t()
        top = torch.maximum(m, x.amax(1))
        s = s * torch.exp(m - top) + torch.exp(x - top[:, None]).sum(1)
        m = top
        S = max(S, float((h.double().abs() @ w[a:a + (1 << 24)].double().abs().t()).max()))
    return m + torch.log(s) - (h.double() * w[t].double()).sum(1), S


@pytest.mark.parametrize("N,V", [(1 << 18, (1 << 20) + 300), (1, (1 << 29) + 1000)])
def test_losses_of_more_tiles_than_a_grid_holds(N, V):
    """More than 2^22 tiles, in a second launch, whose last are ragged: many tokens of few kinds, and one token."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    D, kinds = 8, min(N, 8)
    g = torch.Generator(device=DEV).manual_seed(N)
    w = torch.empty(V, D, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    h = torch.randn(kinds, D, generator=g, device=DEV).bfloat16()
    t = torch.randint(0, V, (kinds,), generator=g, device=DEV)
    t[0] = V - 1                                                # in the last tile
    ref, S = _losses_of_a_few_tokens(h, w, t)
    which = torch.randint(0, kinds, (N,), generator=g, device=DEV)
    which[0] = which[-1] = 0
    with torch.no_grad():
        loss = lce(h[which], w, t[which], reduction="none")
    # the sums of exponentials go over up to 2^22 tiles, 2^14 to a lane's chain (2^-23 each)
    tol = 2 * (D + 4) * 2.0 ** -23 * S + 4e-5 + 2.0 ** -9
    within(loss, ref[which], tol, "loss")


@pytest.mark.parametrize("N", [63, 500, 9000, 200000])
def test_totals_of_many_workgroups(N):
    """The last workgroup to arrive adds up what the others left, on whichever XCD they ran: the sum and the mean are the
    single losses', added in 64 bits and rounded once, on every run, beside another stream's."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    sets = [inputs(N, 300, 16, torch.bfloat16, seed=k) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in sets]
    with torch.no_grad():
        each = [lce(*s, reduction="none").double() for s in sets]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(20):
            for k, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[k].append(torch.stack([lce(*sets[k], reduction=r) for r in ("sum", "mean")]))
        torch.cuda.synchronize()
    for k, e in enumerate(each):
        total = e.sum()
        want = torch.stack([total, total / (sets[k][2] != IGN).sum()])
        for g in got[k]:
            # half a step of 32 bits, and the order of a sum in 64
            assert bool(((g.double() - want).abs() <= want.abs() * (2.0 ** -24 + N * 2.0 ** -53)).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_a_frozen_vocabularys_gradient_made_where_its_sums_are(dtype):
    """256 of the largest tiles, one round: the sums are in one slice, and the gradient takes their place."""
    N, V, D = 4096, 5003, 4095
    h, w, t = inputs(N, V, D, dtype)
    up = (64.0 if dtype == torch.float16 else 1.0) * (0.5 + torch.arange(N, device=DEV) % 7 / 7)
    ref = reference(h, w, t, up)
    b = bounds(ref, dtype, N, V, D)
    loss, dh, _ = _loss_and_grads(h, w, t, up, True)
    within(loss, ref["loss"], b["loss"], "loss")
    within(dh, ref["dh"], b["dh"] + 2.0 ** -48 * ref["gmax"] * ref["wsum"], "dh")


def test_a_capture_is_refused_while_an_eager_graph_holds_leaves_further_up():
    """Inputs that are no leaves themselves: the captured backward pass reaches the leaves they come from."""
    lce, kd = pkg_mod("vocab_loss").linear_cross_entropy, pkg_mod("keyed_dropout").keyed_dropout
    h, w, t = inputs(60, 400, 40, torch.float32)
    h.requires_grad_()
    w.requires_grad_()

    def step():
        hidden = kd(h * 2, 0.25, 3, residual=h + 1)
        return lce(hidden, w * 1.5, t)

    want = torch.autograd.grad(step(), (h, w))
    eager = (h * 3).sum()
    for call in (step, lambda: lce(h * 2, w.detach(), t), lambda: kd(h * 2, 0.5, 1), lambda: kd(h.detach(), 0.5, 1, residual=h * 2)):
        with pytest.raises(RuntimeError, match="outside this capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    late = torch.autograd.grad(eager, h)[0]
    del eager
    assert torch.equal(late, torch.full_like(h, 3.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(step(), (h, w))
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_capture_over_two_streams_is_not_refused():
    """A leaf first used on another stream of the same capture."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(60, 400, 40, torch.float32)
    h.requires_grad_()
    want = [lce(h.detach(), w, t), lce(h.detach(), w, t, reduction="sum")]
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            a = lce(h, w, t)
        main.wait_stream(side)
        b = lce(h, w, t, reduction="sum")
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.detach(), want[0]) and torch.equal(b.detach(), want[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(1, 500, 2049), (3, 700, 4096), (8, 300, 2056), (9, 129, 2049), (5, 40, 70001), (20, 40, 70001), (3000, 1, 40),
                                   (3000, 2, 8), (4097, 17, 1), (200, 4097, 1)])
@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("scale", [1.0, 0.03, 6.0])
def test_sizes_at_the_ends_of_the_paths(N, V, D, frozen, scale, dtype):
    """Few tokens of long rows, one class, one column, rows of 2^17 bytes and more; a class that is the one to ignore."""
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = inputs(N, V, D, dtype)
    up = (64.0 if dtype == torch.float16 else 1.0) * (0.5 + torch.arange(N, device=DEV) % 7 / 7)
    ref = reference(h, w, t, up, scale)
    b = bounds(ref, dtype, N, V, D)
    ignore = V // 2 if V > 2 else IGN                           # its rows are ignored, and so are no others
    if ignore != IGN:
        t = torch.where(t == ignore, IGN, t)
        ref = reference(h, w, t, up, scale)
        b = bounds(ref, dtype, N, V, D)
        t = torch.where(t == IGN, ignore, t)
    h.requires_grad_()
    w.requires_grad_(not frozen)
    loss = lce(h, w, t, ignore_index=ignore, reduction="none", scale=scale)
    grads = torch.autograd.grad(loss, [h] if frozen else [h, w], up)
    within(loss.detach(), ref["loss"], b["loss"] + 2.0 ** -23 * ref["loss"].abs(), "loss")
    within(grads[0], ref["dh"], b["dh"] + 2.0 ** -48 * ref["gmax"] * ref["wsum"], "dh")
    if not frozen:
        # 3000 rows of two classes pass fp16's range.  The rounding to nearest gives the infinity from half a step above
        # the largest number on (65504 + 16), so it is right where the value, within its bound, reaches that.
        want = ref["dw"]
        over = (want.abs() + b["dw"] >= 65520) & (grads[1].double() == torch.copysign(torch.full_like(want, INF), want))
        assert dtype == torch.float16 or not over.any()
        if not over.all():
            within(grads[1][~over], want[~over], b["dw"][~over], "dw")


@pytest.mark.parametrize("N", [1, 5, 20, 300])
@pytest.mark.parametrize("frozen", [False, True])
def test_batches_that_are_ignored_whole(N, frozen):
    h, w, t = inputs(N, 600, 48, torch.bfloat16)
    h[0] = NAN
    for reduction in ("none", "sum", "mean"):
        up = torch.ones(N if reduction == "none" else (), device=DEV)
        loss, dh, dw = _loss_and_grads(h, w, torch.full_like(t, IGN), up, frozen, reduction)
        assert torch.isnan(loss).all() if reduction == "mean" else not loss.any()
        assert not dh.any() and (frozen or not dw.any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(4, 11264, 40), (4, 11265, 40), (1, 45056, 33), (1, 45057, 33), (2, 22528, 20), (3, 8192, 1), (3, 8193, 1),
                                   (1, 131071, 3), (5, 8193, 17), (32, 100, 1), (33, 100, 1), (33, 131071, 2)])
def test_8_bit_products_at_the_ends_of_their_paths(M, K, N, dtype):
    """Tokens that just fit into LDS and those that do not, rows that just stay in registers, one output."""
    from test_gpu_int8 import check_product, quant_ref
    m = pkg_mod("int8_linear")
    g = torch.Generator(device=DEV).manual_seed(M + K)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    w = torch.randint(-128, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    ws, bias = torch.rand(N, generator=g, device=DEV) / 100, torch.randn(N, generator=g, device=DEV)
    y = m.int8_linear(x, w, ws, bias)
    q, s = quant_ref(x)
    check_product(y, q, s, w, ws, bias, dtype)
    assert torch.equal(m.int8_matmul(*m.quantize_rows(x), m.lay_out(w), ws, bias, dtype), y)


def test_calls_of_two_threads():
    """Each on a stream of its own, the calls' workspaces their own."""
    import threading
    lce, kd, i8 = pkg_mod("vocab_loss").linear_cross_entropy, pkg_mod("keyed_dropout").keyed_dropout, pkg_mod("int8_linear")
    sets = [inputs(130, 2500, 96, torch.bfloat16, seed=k) for k in range(2)]
    wq = torch.randint(-127, 128, (50, 96), dtype=torch.int8, device=DEV)
    ws = torch.rand(50, device=DEV)

    def go(k):
        h, w, t = sets[k]
        h = h.detach().requires_grad_()
        hidden = kd(h, 0.3, k, residual=h)
        loss = lce(hidden, w, t)
        (dh,) = torch.autograd.grad(loss, h)
        return loss.detach(), dh, i8.int8_linear(hidden.detach(), wq, ws)

    want = [go(0), go(1)]
    torch.cuda.synchronize()
    got = [[], []]

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k].append(go(k))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 20
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))
