"""quantize_rows, int8_matmul and Int8Linear (po_quantize_rows, po_int8_matmul).

Quantised values and scales are compared exactly (the scale is a 32-bit quotient,
the values the exact quotients' nearest).  A product's sum is exact; it then takes
a conversion, two products and a sum in 32 bits (4 * 2^-24 of |sum| s sw plus 2^-24
of the result) and one rounding to its type (eps / 2, half of fp16's smallest
number)."""
import copy

import pytest
import torch

from conftest import pkg_mod

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = (torch.float32, torch.float16, torch.bfloat16)


def quant_ref(x):
    x = x.double().cpu()
    s = (x.abs().amax(-1) / 127.0).float()
    q = torch.where(s[..., None] > 0, torch.round(x / s.double()[..., None]), torch.zeros(()).double())
    return q.to(torch.int8), s


def check_product(y, q, s, wq, ws, bias, dtype):
    q, s, wq, ws, y = q.double().cpu(), s.double().cpu(), wq.double().cpu(), ws.double().cpu(), y.double().cpu()
    main = (q @ wq.t()) * s[..., None] * ws
    ref = main if bias is None else main + bias.double().cpu()
    tol = main.abs() * 2.0 ** -22 + ref.abs() * (2.0 ** -24 + torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    # Half a step above the largest finite value (fp16: 65504 + 16 = 65520 = 2^16 (1 - eps / 4)) the rounding to
    # nearest gives the infinity, so an infinity is right from there on, less the error before that rounding.
    info = torch.finfo(dtype)
    edge = info.max * (1 - info.eps / 4) / (1 - info.eps / 2)
    before = main.abs() * 2.0 ** -22 + ref.abs() * 2.0 ** -24
    over = (ref.abs() + before >= edge) & (y == torch.copysign(torch.full_like(ref, float("inf")), ref))
    ok = ((y - ref).abs() <= tol) | over
    assert bool(ok.all()), (float(ref[~ok].abs().max()), float((y - ref)[~ok].abs().max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (3, 15), (4, 17), (5, 64), (7, 1000), (2, 1025), (9, 4001), (130, 200), (2, 131071)])
def test_quantize_rows(M, K, dtype):
    m = pkg_mod("int8_linear")
    g = torch.Generator(device=DEV).manual_seed(M * 7 + K)
    x = (torch.randn(M, K, generator=g, device=DEV) * torch.rand(M, 1, generator=g, device=DEV) * 10).to(dtype)
    q, s = m.quantize_rows(x)
    rq, rs = quant_ref(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), rq)
    assert q.shape == x.shape and s.shape == x.shape[:-1]


def test_quantize_ties_and_borders():
    """Halves go to the even neighbour; values next to a border go to their own side."""
    m = pkg_mod("int8_linear")
    s = 0.375                                                   # 127 s is exact, so are the halves
    k = torch.arange(-127, 127, dtype=torch.float64)
    half = (k + 0.5) * s
    x = torch.cat([torch.tensor([127 * s]).double(), half]).float()
    near = torch.stack([x, torch.nextafter(x, torch.full_like(x, -1e9)), torch.nextafter(x, torch.full_like(x, 1e9))])
    near[:, 0] = 127 * s
    q, sc = m.quantize_rows(near.to(DEV))
    rq, rs = quant_ref(near)
    assert torch.equal(sc.cpu(), rs) and float(rs[0]) == s and torch.equal(q.cpu(), rq)
    assert int(q[0, 1 + 127]) == 0 and int(q[0, 1 + 128]) == 2  # 0.5 -> 0, 1.5 -> 2
    # many scales, all values of a 16-bit type next to halves of them
    g = torch.Generator().manual_seed(3)
    top = torch.rand(64, 1, generator=g) + 0.5
    h = ((torch.randint(-126, 126, (64, 500), generator=g) + 0.5).double() * (top.double() / 127)).float()
    for d in (-1e9, 0.0, 1e9):
        v = torch.cat([top, torch.nextafter(h, torch.full_like(h, d)) if d else h], 1)
        q, sc = m.quantize_rows(v.to(DEV))
        rq, rs = quant_ref(v)
        assert torch.equal(sc.cpu(), rs) and torch.equal(q.cpu(), rq)


def test_quantize_extreme_rows():
    m = pkg_mod("int8_linear")
    big, small = torch.finfo(torch.float32).max, 1e-45
    x = torch.zeros(8, 40)
    x[1, 3] = big
    x[2, :4] = torch.tensor([small, 2 * small, 300 * small, -7 * small])
    x[3, :3] = torch.tensor([1e-38, -3e-39, 2e-40])
    x[4, :3] = torch.tensor([3e-29, -1.4e-29, 1e-30])
    x[5, 7] = float("nan")
    x[6, 7] = -float("inf")
    x[7] = -big
    q, s = m.quantize_rows(x.to(DEV))
    ok = [0, 1, 2, 3, 4, 7]
    rq, rs = quant_ref(x)
    assert torch.equal(s.cpu()[ok], rs[ok]) and torch.equal(q.cpu()[ok], rq[ok])
    assert torch.isnan(s[5:7]).all() and not q[5:7].any()
    y = m.int8_linear(x.to(DEV), torch.ones(5, 40, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV))
    # 127 * (largest / 127) rounds past the largest number (row 1), 40 of them pass it (row 7): infinite by the formula
    ref = (rq.double().sum(1) * rs.double())[ok].float()
    assert torch.isnan(y[5:7]).all() and torch.equal(torch.isfinite(y[ok, 0]).cpu(), torch.isfinite(ref)) and not y[0].any()


SIZES = [(1, 1, 1), (1, 16, 5), (1, 4096, 300), (2, 17, 64), (5, 4001, 130), (16, 64, 100), (17, 1000, 257), (32, 129, 128), (33, 31, 65),
         (64, 256, 1000), (130, 2000, 257), (1111, 4001, 1000), (1500, 96, 2500), (2500, 160, 5000), (300, 7, 9), (2000, 100, 4000), (1, 70000, 33), (4, 14336, 50), (3, 20000, 17), (31, 3000, 16), (1100, 300, 1000), (1111, 4001, 500), (2000, 129, 2040)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(M, K, N, dtype):
    m = pkg_mod("int8_linear")
    g = torch.Generator(device=DEV).manual_seed(M + 3 * K + 7 * N)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    w = torch.randint(-128, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    ws = torch.rand(N, generator=g, device=DEV) / 100
    bias = torch.randn(N, generator=g, device=DEV) if N % 2 else None
    q, s = quant_ref(x)
    want = m.int8_linear(x, w, ws, bias)
    assert want.dtype == dtype and want.shape == (M, N)
    check_product(want, q, s, w, ws, bias, dtype)
    laid = m.lay_out(w)
    assert torch.equal(m.int8_linear(x, laid, ws, bias), want)
    store = torch.full((N, laid.stride(0)), 77, dtype=torch.int8, device=DEV)       # what lies behind a weight's row does not count
    store[:, :K] = w
    assert torch.equal(m.int8_linear(x, store[:, :K], ws, bias), want)
    qq, ss = m.quantize_rows(x)
    assert torch.equal(m.int8_matmul(qq, ss, laid, ws, bias, dtype), want)
    qc = torch.full((M, K + 19), -5, dtype=torch.int8, device=DEV)                 # nor behind a token's
    qc[:, :K] = qq
    assert torch.equal(m.int8_matmul(qc[:, :K], ss, w, ws, bias, dtype), want)


def test_sums_past_24_bits_and_at_the_longest_row():
    m = pkg_mod("int8_linear")
    K = m.MAX_INNER
    q = torch.full((2, K), 127, dtype=torch.int8, device=DEV)
    q[1] = -128
    w = torch.full((3, K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(3, device=DEV)
    y = m.int8_matmul(q, one[:2], w, one, dtype=torch.float32)
    ref = (q.double() @ w.double().t()).float()                 # the whole number, rounded once
    assert torch.equal(y, ref)


def test_offsets_past_32_bits():
    m = pkg_mod("int8_linear")
    g = torch.Generator(device=DEV).manual_seed(1)
    # outputs: 2.4e9 of them
    x = torch.randn(40000, 16, generator=g, device=DEV).bfloat16()
    w = torch.randint(-127, 128, (60001, 16), generator=g, device=DEV, dtype=torch.int8)
    ws = torch.rand(60001, generator=g, device=DEV)
    y = m.int8_linear(x, w, ws)
    for r in (0, 35790, 39998):
        q, s = quant_ref(x[r:r + 2])
        check_product(y[r:r + 2], q, s, w, ws, None, torch.bfloat16)
    del y
    # tokens: 2.2e9 bytes of 8 bits
    x = torch.randn(1, 131000, generator=g, device=DEV).half().expand(17000, 131000) * \
        torch.linspace(0.5, 2.0, 17000, device=DEV).half()[:, None]
    w = torch.randint(-127, 128, (40, 131000), generator=g, device=DEV, dtype=torch.int8)
    y = m.int8_linear(x, w, ws[:40])
    for r in (0, 16390, 16998):
        q, s = quant_ref(x[r:r + 2])
        check_product(y[r:r + 2], q, s, w, ws[:40], None, torch.float16)


def test_shapes_strides_and_streams():
    m = pkg_mod("int8_linear")
    w = torch.randint(-127, 128, (70, 96), dtype=torch.int8, device=DEV)
    ws = torch.rand(140, device=DEV)[::2]
    x = torch.randn(6, 4, 96, device=DEV, dtype=torch.bfloat16)
    want = m.int8_linear(x.view(24, 96), w, ws.contiguous())
    assert torch.equal(m.int8_linear(x, w, ws).view(24, 70), want)
    wide = torch.full((24, 300), float("nan"), device=DEV, dtype=torch.bfloat16)
    for off in (0, 1, 8):
        wide[:, off:off + 96] = x.view(24, 96)
        assert torch.equal(m.int8_linear(wide[:, off:off + 96], w, ws), want)
    assert torch.equal(m.int8_linear(x.view(24, 96).t().contiguous().t(), w, ws), want)
    assert torch.equal(m.int8_linear(x[0, 0], w, ws), want[0])
    assert torch.equal(m.int8_linear(x, w.t().contiguous().t(), ws).view(24, 70), want)
    assert m.int8_linear(x[:0], w, ws).shape == (0, 4, 70)
    assert m.quantize_rows(x[:0])[0].shape == (0, 4, 96)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = m.int8_linear(x, w, ws)
    s.synchronize()
    assert torch.equal(y.view(24, 70), want)


def test_in_a_replayed_graph():
    m = pkg_mod("int8_linear")
    layer = m.Int8Linear(torch.randn(200, 130, device=DEV), torch.randn(200, device=DEV))
    for rows in (1, 50):
        x = torch.randn(rows, 130, device=DEV, dtype=torch.float16)
        layer(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x)
        for k in range(3):
            x.copy_(torch.randn(rows, 130, device=DEV))
            want = layer(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_module_of_a_linear_and_its_moves():
    m = pkg_mod("int8_linear")
    lin = torch.nn.Linear(100, 37).to(DEV)
    layer = m.Int8Linear.from_linear(lin)
    x = torch.randn(11, 100, device=DEV, dtype=torch.bfloat16)
    y = layer(x)
    wq, ws = quant_ref(lin.weight.detach())
    q, s = quant_ref(x)
    check_product(y, q, s, wq, ws, lin.bias.detach(), torch.bfloat16)
    layer.half()
    assert layer.wscale.dtype == torch.float32 and layer.wq.stride(0) % 64 == 0 and torch.equal(layer(x), y)
    other = m.Int8Linear(torch.randn(37, 100, device=DEV), torch.zeros(37, device=DEV))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    assert torch.equal(copy.deepcopy(layer)(x), y)
    assert not y.requires_grad and not layer(x.requires_grad_()).requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        m.int8_linear(x, layer.wq, layer.wscale)
