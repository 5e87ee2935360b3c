"""CPU tests of the large-vocabulary head's operators: every argument that the
documentation does not allow is refused with an error that names it, by the
Python entry points and by the C ABI, before anything is launched."""
import ctypes

import pytest
import torch

from conftest import pkg_mod

H = 4          # a small inner dimension


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_dropout_refusals():
    kd = pkg_mod("keyed_dropout").keyed_dropout
    x = _t(2, 8)
    for bad in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="p must"):
            kd(x, bad, 1)
    for kw, what in ((dict(seed=-1), "seed"), (dict(seed=1 << 64), "seed"), (dict(seed=1, step=-1), "step"),
                     (dict(seed=1, step=1 << 64), "step"), (dict(seed=1, row0=-1), "row0"),
                     (dict(seed=1, row0=(1 << 32) - 1), "row0")):
        with pytest.raises(ValueError, match=what):
            kd(x, 0.5, **kw)
    with pytest.raises(TypeError, match="step"):
        kd(x, 0.5, 1, step=torch.zeros(1))
    with pytest.raises(TypeError, match="x must"):
        kd(_t(2, 8, dtype=torch.int32), 0.5, 1)
    with pytest.raises(TypeError, match="x must"):
        kd(_t(2, 8, dtype=torch.float64), 0.5, 1)
    with pytest.raises(ValueError, match="dimension"):
        kd(torch.tensor(1.0), 0.5, 1)
    for res in (_t(8), _t(2, 8, dtype=torch.float16), 3.0):
        with pytest.raises(ValueError, match="residual"):
            kd(x, 0.5, 1, residual=res)
    with pytest.raises(ValueError, match="p must"):
        pkg_mod("keyed_dropout").KeyedDropout(2.0)


def test_loss_refusals():
    lce = pkg_mod("vocab_loss").linear_cross_entropy
    h, w, t = _t(3, H), _t(5, H), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="hidden must"):
        lce(h.double(), w, t)
    with pytest.raises(TypeError, match="weight must"):
        lce(h, w.int(), t)
    with pytest.raises(TypeError, match="hidden is"):
        lce(h.half(), w, t)
    for hh, ww in ((h, _t(5, H + 1)), (h, _t(5)), (torch.tensor(1.0), w)):
        with pytest.raises(ValueError, match="expected"):
            lce(hh, ww, t)
    with pytest.raises(ValueError, match="empty"):
        lce(h, _t(0, H), t)
    with pytest.raises(ValueError, match="empty"):
        lce(_t(3, 0), _t(5, 0), t)
    for tt in (t.int(), t[:2], t[:, None], 0):
        with pytest.raises(ValueError, match="target"):
            lce(h, w, tt)
    with pytest.raises(ValueError, match="reduction"):
        lce(h, w, t, reduction="max")
    for s in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            lce(h, w, t, scale=s)


def test_int8_refusals():
    m = pkg_mod("int8_linear")
    x, wq, ws = _t(2, H), _t(3, H, dtype=torch.int8), _t(3)
    with pytest.raises(TypeError, match="x must"):
        m.quantize_rows(x.double())
    with pytest.raises(ValueError, match="inner"):
        m.quantize_rows(_t(2, 0))
    with pytest.raises(ValueError, match="inner"):
        m.quantize_rows(_t(1, m.MAX_INNER + 1))
    with pytest.raises(RuntimeError, match="no gradient"):
        m.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        m.int8_linear(x.clone().requires_grad_(), wq, ws)
    for w in (wq.float(), wq[:, :2], wq[0], wq[:0]):
        with pytest.raises(ValueError, match="weights"):
            m.int8_linear(x, w, ws)
    for s in (ws.half(), ws[:2]):
        with pytest.raises(ValueError, match="weight scales"):
            m.int8_linear(x, wq, s)
    with pytest.raises(ValueError, match="bias"):
        m.int8_linear(x, wq, ws, bias=_t(2))
    q = _t(2, H, dtype=torch.int8)
    with pytest.raises(TypeError, match="int8 rows"):
        m.int8_matmul(x, ws, wq, ws)
    with pytest.raises(ValueError, match="scale"):
        m.int8_matmul(q, _t(3), wq, ws)
    with pytest.raises(TypeError, match="dtype"):
        m.int8_matmul(q, _t(2), wq, ws, dtype=torch.float64)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg_mod("keyed_dropout").keyed_dropout(_t(2, 8), 0.5, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg_mod("vocab_loss").linear_cross_entropy(_t(3, H), _t(5, H), torch.zeros(3, dtype=torch.int64))
    m = pkg_mod("int8_linear")
    with pytest.raises(RuntimeError, match="CUDA"):
        m.quantize_rows(_t(2, H))
    with pytest.raises(RuntimeError, match="CUDA"):
        m.int8_linear(_t(2, H), _t(3, H, dtype=torch.int8), _t(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        m.int8_matmul(_t(2, H, dtype=torch.int8), _t(2), _t(3, H, dtype=torch.int8), _t(3))


def test_eval_mode_dropout_is_the_identity():
    d = pkg_mod("keyed_dropout").KeyedDropout(0.5).eval()
    x = torch.randn(3, 5)
    assert d(x) is x and torch.equal(d(x, residual=x), 2 * x)


def _buffer():
    """An aligned host address: the entries below refuse before they read it."""
    b = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(b) + 255) // 256 * 256
    return b, at


def test_c_entries_refuse_before_launching():
    import os
    nat = pkg_mod("_native")
    if not os.path.exists(nat.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    lib = nat.load()
    keep, p = _buffer()
    F32, BF16 = 0, 2

    def refused(rc, what):
        assert rc == -1 and what in nat.last_error(), (rc, nat.last_error())

    drop = lambda **k: lib.po_dropout(*[{**dict(x=p, ldx=8, r=None, ldr=0, dt=F32, rows=2, cols=8, seed=1, step=0, sd=None,  # noqa: E731
                                                su=None, row0=0, drop=1, y=p, ldy=8, s=None), **k}[n]
                                        for n in "x ldx r ldr dt rows cols seed step sd su row0 drop y ldy s".split()])
    refused(drop(x=None), "null")
    refused(drop(y=None), "null")
    refused(drop(drop=65537), "drop")
    refused(drop(drop=-1), "drop")
    refused(drop(rows=0), "sizes")
    refused(drop(cols=0), "sizes")
    refused(drop(row0=1 << 32), "sizes")
    refused(drop(ldx=7), "strides")
    refused(drop(r=p, ldr=7), "strides")
    refused(drop(dt=7), "dtype")

    names = "h ldh w ldw dt N V D t ign c red ws wsb stat loss count s".split()
    fwd = lambda **k: lib.po_linear_ce_fwd(*[{**dict(h=p, ldh=8, w=p, ldw=8, dt=BF16, N=4, V=5, D=8, t=p, ign=-100, c=1.0, red=2,  # noqa: E731
                                                     ws=p, wsb=1 << 40, stat=p, loss=p, count=p, s=None), **k}[n] for n in names])
    for n in ("h", "w", "t", "ws", "stat", "loss", "count"):
        refused(fwd(**{n: None}), "null")
    for k in (dict(N=0), dict(V=0), dict(D=0), dict(N=(1 << 21) + 1), dict(V=1 << 31), dict(D=(1 << 20) + 1)):
        refused(fwd(**k), "sizes")
    refused(fwd(ldh=7), "strides")
    refused(fwd(ldw=7), "strides")
    refused(fwd(dt=3), "dtype")
    refused(fwd(red=3), "reduction")
    for c in (0.0, -1.0, float("inf"), float("nan")):
        refused(fwd(c=c), "scale")
    refused(fwd(wsb=0), "workspace")

    names = "h ldh w ldw dt N V D t ign c red stat count g ws wsb dh lddh dw lddw s".split()
    bwd = lambda **k: lib.po_linear_ce_bwd(*[{**dict(h=p, ldh=8, w=p, ldw=8, dt=BF16, N=4, V=5, D=8, t=p, ign=-100, c=1.0, red=2,  # noqa: E731
                                                     stat=p, count=p, g=p, ws=p, wsb=1 << 40, dh=p, lddh=8, dw=p, lddw=8, s=None),
                                               **k}[n] for n in names])
    for n in ("h", "w", "t", "ws", "stat", "count", "g"):
        refused(bwd(**{n: None}), "null")
    refused(bwd(lddh=7), "strides")
    refused(bwd(lddw=7), "strides")
    refused(bwd(wsb=0), "workspace")
    refused(bwd(c=0.0), "scale")
    assert bwd(dh=None, dw=None) == 0                     # nothing is asked for

    names = "h ldh w ldw dt N V D t ign c red ws wsb loss count dhu s".split()
    ffwd = lambda **k: lib.po_linear_ce_frozen_fwd(*[{**dict(h=p, ldh=8, w=p, ldw=8, dt=BF16, N=4, V=5, D=8, t=p, ign=-100, c=1.0,  # noqa: E731
                                                             red=2, ws=p, wsb=1 << 40, loss=p, count=p, dhu=p, s=None), **k}[n]
                                                     for n in names])
    for n in ("h", "w", "t", "ws", "loss", "count", "dhu"):
        refused(ffwd(**{n: None}), "null")
    for k in (dict(N=0), dict(V=0), dict(D=0), dict(N=(1 << 21) + 1), dict(V=1 << 31), dict(D=(1 << 20) + 1)):
        refused(ffwd(**k), "sizes")
    for k, word in ((dict(ldh=7), "strides"), (dict(ldw=7), "strides"), (dict(dt=3), "dtype"), (dict(red=3), "reduction"),
                    (dict(c=0.0), "scale"), (dict(c=float("nan")), "scale"), (dict(wsb=0), "workspace"), (dict(dhu=p + 4), "16 bytes")):
        refused(ffwd(**k), word)
    names = "dhu dt N D t ign red count g dh lddh s".split()
    fbwd = lambda **k: lib.po_linear_ce_frozen_bwd(*[{**dict(dhu=p, dt=BF16, N=4, D=8, t=p, ign=-100, red=2, count=p, g=p, dh=p,  # noqa: E731
                                                             lddh=8, s=None), **k}[n] for n in names])
    for n in ("dhu", "t", "count", "g", "dh"):
        refused(fbwd(**{n: None}), "null")
    for k, word in ((dict(N=0), "sizes"), (dict(D=0), "sizes"), (dict(lddh=7), "strides"), (dict(dt=3), "dtype"),
                    (dict(red=-1), "reduction"), (dict(dhu=p + 8), "16 bytes")):
        refused(fbwd(**k), word)

    qr = lambda **k: lib.po_quantize_rows(*[{**dict(x=p, ldx=20, dt=F32, M=2, K=20, q=p, ldq=32, sc=p, s=None), **k}[n]  # noqa: E731
                                            for n in "x ldx dt M K q ldq sc s".split()])
    for n in ("x", "q", "sc"):
        refused(qr(**{n: None}), "null")
    refused(qr(K=1 << 17, ldx=1 << 17, ldq=1 << 17), "sizes")
    refused(qr(ldq=20), "strides")
    refused(qr(ldq=40), "strides")
    refused(qr(ldx=19), "strides")
    refused(qr(q=p + 4), "strides")
    refused(qr(dt=9), "dtype")

    mm = lambda **k: lib.po_int8_matmul(*[{**dict(q=p, ldq=32, sx=p, w=p, ldw=32, sw=p, b=None, M=2, N=3, K=20, y=p, ldy=3, dt=F32,  # noqa: E731
                                                  s=None), **k}[n] for n in "q ldq sx w ldw sw b M N K y ldy dt s".split()])
    for n in ("q", "sx", "w", "sw", "y"):
        refused(mm(**{n: None}), "null")
    refused(mm(M=0), "sizes")
    refused(mm(K=1 << 17), "sizes")
    for k in (dict(ldq=24), dict(ldw=24), dict(q=p + 8), dict(w=p + 8), dict(ldy=2), dict(ldq=16), dict(ldw=1 << 23)):
        refused(mm(**k), "16")
    refused(mm(dt=-1), "dtype")
    del keep


def test_workspace_sizes_follow_the_work():
    nat = pkg_mod("_native")
    lib = nat.load()
    a, b = ctypes.c_int64(), ctypes.c_int64()

    def sizes(N, V, D, dt, ld, dh, dw):
        assert lib.po_linear_ce_workspace(256, ld, 256, ld, dt, N, V, D, dh, dw, ctypes.byref(a), ctypes.byref(b)) == 0
        return a.value, b.value

    # no logits: far below the N x V numbers of one matrix of them, in either pass
    N, V, D = 8192, 131072, 2048
    f, g = sizes(N, V, D, 2, D, 1, 1)
    assert f < N * V * 4 // 50 and g < N * V * 4 // 4
    # nor with one side frozen (pieces grow to the same bound); a small head needs little; unpadded rows more
    assert max(sizes(N, V, D, 2, D, 1, 0)[1], sizes(N, V, D, 2, D, 0, 1)[1]) < N * V * 4 // 4
    assert sizes(32, 4096, 256, 2, 256, 1, 1)[1] < 64 << 20
    assert sizes(N, V, D, 2, D + 1, 1, 1)[0] > f
    assert sizes(N, V, D, 0, D, 1, 1)[0] > f


def test_frozen_workspace_holds_a_piece():
    lib = pkg_mod("_native").load()
    b = ctypes.c_int64()
    # from small heads to the largest: a piece of 640 MB, its transpose and slabs, never the N x V numbers
    for N, V, D, dt in ((1, 1, 1, 0), (4096, 32768, 1024, 2), (8192, 131072, 2048, 2), (8192, 131072, 2048, 0), (1 << 21, 300000, 64, 1)):
        assert lib.po_linear_ce_frozen_workspace(256, D, 256, D, dt, N, V, D, ctypes.byref(b)) == 0
        slabs = 64 * N * D * 4
        assert 0 < b.value < (900 << 20) + min(slabs, 40 * N * D) + (N * V // 128 * 13 + 64 * N) + (N + 256) * (D + 512) * 12, (N, V, D, dt, b.value)
    assert lib.po_linear_ce_frozen_workspace(256, 8, 256, 8, 7, 1, 1, 8, ctypes.byref(b)) != 0
    assert lib.po_linear_ce_frozen_workspace(256, 8, 256, 8, 2, 1, 1, 8, None) != 0


def test_lay_out_pads_rows():
    m = pkg_mod("int8_linear")
    for K, ld in ((1, 128), (70, 128), (129, 256), (1000, 1152), (4000, 4224), (4001, 4224), (8192, 8320)):
        w = torch.randint(-127, 128, (5, K), dtype=torch.int8)
        v = m.lay_out(w)
        assert torch.equal(v, w) and v.stride() == (ld, 1)
        if v.data_ptr() % 16 == 0:
            assert m._weights(v)[0] is v and m._weights(v)[1] == ld
        assert torch.equal(m._weights(w)[0], w)
