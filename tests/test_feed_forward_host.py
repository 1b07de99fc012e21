"""Refusals of the feed-forward operators, on the host: shapes and types through the Python entry points (fake device tensors,
nothing is launched) and arguments through the C ABI; the shapes that the registered operators promise; the oracle's e4m3."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import verace_amd as va
from oracle import feed_forward as oracle

E4M3 = torch.float8_e4m3fn
BF, F32 = torch.bfloat16, torch.float32


def _e(*s, dtype=BF, device="cuda"):
    return torch.empty(s, dtype=dtype, device=device)


def fake(f):
    def run(*a, **k):
        with FakeTensorMode(allow_non_fake_inputs=True):
            f(*a, **k)
    run.__name__ = f.__name__
    return run


@fake
def test_gated_refusals():
    ok = dict(x=_e(3, 16), w_gate=_e(8, 16), w_up=_e(8, 16))
    eight = dict(x=_e(3, 16, dtype=E4M3), w_gate=_e(8, 16, dtype=E4M3), w_up=_e(8, 16, dtype=E4M3), x_scale=_e(3, dtype=F32),
                 gate_scale=_e(8, dtype=F32), up_scale=_e(8, dtype=F32))
    va.gated_linear(**ok), va.gated_linear(**eight)
    for base, bad in ((ok, dict(x=_e(3, 16, device="cpu"))), (ok, dict(x=_e(3, 16, dtype=torch.float64))), (ok, dict(x=_e(3, 15))),
                      (ok, dict(w_gate=_e(8, 15))), (ok, dict(w_up=_e(9, 16))), (ok, dict(w_up=_e(8, 16, dtype=F32))),
                      (ok, dict(w_gate=_e(16))), (ok, dict(w_gate=_e(8, 16, device="cpu"))), (ok, dict(activation="gelu")),
                      (ok, dict(activation=None)), (ok, dict(beta1=0.0)), (ok, dict(beta2=-1.0)), (ok, dict(beta2=float("inf"))),
                      (ok, dict(beta1=float("nan"))), (ok, dict(beta1=1e-40)), (ok, dict(beta2=1e39)), (ok, dict(x_scale=_e(3, dtype=F32))), (ok, dict(gate_scale=_e(8, dtype=F32))),
                      (ok, dict(out_dtype=F32)), (ok, dict(x=_e())), (eight, dict(x_scale=None)), (eight, dict(x_scale=_e(3))),
                      (eight, dict(x_scale=_e(3, 1, dtype=F32))), (eight, dict(up_scale=None)), (eight, dict(up_scale=_e(1, dtype=F32))),
                      (eight, dict(gate_scale=_e(8, dtype=F32, device="cpu"))), (eight, dict(out_dtype=E4M3)),
                      (eight, dict(out_dtype=torch.float64)), (eight, dict(w_up=_e(8, 16)))):
        with pytest.raises(RuntimeError, match="verace_amd"):
            va.gated_linear(**{**base, **bad})


@fake
def test_linear_refusals():
    ok = dict(x=_e(2, 3, 16), weight=_e(8, 16), bias=_e(8), residual=_e(2, 3, 8))
    eight = dict(x=_e(3, 16, dtype=E4M3), weight=_e(8, 16, dtype=E4M3), x_scale=_e(3, dtype=F32), weight_scale=_e(8, dtype=F32))
    va.linear_add(**ok), va.linear_add(**eight, residual=_e(3, 8)), va.linear_add(**eight, residual=_e(3, 8, dtype=F32), out_dtype=F32)
    for base, bad in ((ok, dict(x=_e(2, 3, 16, device="cpu"))), (ok, dict(weight=_e(16, 8))), (ok, dict(bias=_e(7))), (ok, dict(bias=_e(8, 1))),
                      (ok, dict(bias=_e(8, dtype=F32))), (ok, dict(residual=_e(8))), (ok, dict(residual=_e(3, 8))),
                      (ok, dict(residual=_e(2, 3, 8, dtype=F32))), (ok, dict(residual=_e(2, 3, 8, device="cpu"))),
                      (ok, dict(activation="relu")), (ok, dict(activation="situ")), (ok, dict(weight_scale=_e(8, dtype=F32))),
                      (eight, dict(weight_scale=None)), (eight, dict(residual=_e(3, 8, dtype=F32))), (eight, dict(bias=_e(8, dtype=torch.float16)))):
        with pytest.raises(RuntimeError, match="verace_amd"):
            va.linear_add(**{**base, **bad})


@fake
def test_quant_refusals():
    a = _e(3, 16)
    for bad in (dict(a=_e(3, 16, device="cpu")), dict(a=_e(3, 16, dtype=E4M3)), dict(a=_e()), dict(a=_e(3, 0)), dict(residual=_e(16)),
                dict(residual=_e(3, 16, dtype=F32)), dict(norm_weight=_e(15)), dict(norm_weight=_e(16, dtype=torch.float16)),
                dict(norm_weight=_e(16, device="cpu"))):
        with pytest.raises(RuntimeError, match="verace_amd"):
            va.norm_add_quant(**{**dict(a=a), **bad})
    with pytest.raises(RuntimeError, match="verace_amd"):
        va.quantize_rows(_e(3, 16, device="cpu"))


@fake
def test_no_gradients_through_8_bits():
    w = _e(16, dtype=F32).requires_grad_()
    for call in (lambda: va.norm_add_quant(_e(3, 16), None, w), lambda: va.quantize_rows(_e(3, 16).requires_grad_()),
                 lambda: va.linear_add(_e(3, 16, dtype=E4M3), _e(8, 16, dtype=E4M3), None, _e(3, 8).requires_grad_(), _e(3, dtype=F32),
                                       _e(8, dtype=F32)),
                 lambda: va.gated_linear(_e(3, 16, dtype=E4M3), _e(8, 16, dtype=E4M3), _e(8, 16, dtype=E4M3),
                                         _e(3, dtype=F32).requires_grad_(), _e(8, dtype=F32), _e(8, dtype=F32))):
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
        with torch.no_grad():
            call()
    from verace_amd import feed_forward as ff
    with pytest.raises(RuntimeError, match="no gradients"):
        ff._rows_fit(_e(1, 8), 1 << 23)


@fake
def test_traced_shapes():
    x, w = _e(2, 5, 24), _e(40, 24)
    h = va.gated_linear(x, w, w)
    assert h.shape == (2, 5, 40) and h.dtype == BF
    y = va.linear_add(h, _e(24, 40), _e(24), x, activation="gelu")
    assert y.shape == x.shape and y.dtype == BF
    s, q, scale = va.norm_add_quant(x, x, _e(24))
    assert s.shape == q.shape == x.shape and s.dtype == BF and q.dtype == E4M3 and scale.shape == (2, 5) and scale.dtype == F32
    wq, ws = va.quantize_rows(w)
    assert wq.shape == w.shape and ws.shape == (40,)
    assert va.linear_add(q, wq, x_scale=scale, weight_scale=ws, out_dtype=torch.float16).dtype == torch.float16
    for g, t in zip(torch.ops.verace.gated_linear_bwd(x, w, w, "situ", 4.0, 25.0, h), (x, w, w)):
        assert g.shape == t.shape and g.dtype == t.dtype
    for g, t in zip(torch.ops.verace.linear_add_bwd(x, w, _e(40), "silu", h), (x, w, _e(40))):
        assert g.shape == t.shape and g.dtype == t.dtype


def test_gradient_shapes_are_checked():
    from verace_amd import feed_forward as ff
    with FakeTensorMode(allow_non_fake_inputs=True):
        x, w = _e(3, 16), _e(8, 16)
        for dy in (_e(3, 9), _e(2, 8), _e(3, 8, dtype=F32), _e(3, 8, device="cpu")):
            with pytest.raises(RuntimeError, match="must be"):
                ff._launch_gated_bwd(x, w, w, 1, 4.0, 25.0, dy, (True,) * 3)
            with pytest.raises(RuntimeError, match="must be"):
                ff._launch_linear_bwd(x, w, None, 0, dy, (True,) * 3)


@pytest.fixture(scope="module")
def lib():
    from verace_amd import _lib
    return _lib.load()


def test_c_refusals(lib):
    null, one, odd = None, ctypes.c_void_p(64), ctypes.c_void_p(72)
    INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3

    def linear(x=one, ldx=16, xs=null, w=one, ldw=16, ws=null, dtype=1, bias=null, res=null, ldr=0, act=0, out=one, ldo=8, od=1, M=2, N=8,
               K=16):
        return lib.vmi_linear_add(x, ldx, xs, w, ldw, ws, dtype, bias, res, ldr, act, out, ldo, od, null, M, N, K, null)

    for kw in (dict(x=null), dict(w=null), dict(out=null), dict(ldx=8), dict(ldw=8), dict(ldo=7), dict(res=one, ldr=7), dict(act=3), dict(act=-1),
               dict(dtype=4), dict(dtype=-1), dict(od=0), dict(od=3, dtype=3), dict(dtype=3, ldx=16, ldw=16), dict(M=-1), dict(N=-1), dict(K=-1),
               dict(M=(1 << 30) + 1)):
        assert linear(**kw) == INVALID, kw
    for kw in (dict(x=odd), dict(w=odd), dict(ldx=20), dict(ldw=20), dict(K=15, ldx=15, ldw=16), dict(ldx=1 << 23), dict(ldw=1 << 23)):
        assert linear(**kw) == UNSUPPORTED, kw
    assert linear(M=0, x=null, out=null) == 0 and linear(N=0, w=null, out=null) == 0

    def gated(x=one, ldx=16, xs=null, wg=one, ldg=16, gs=null, wu=one, ldu=16, us=null, dtype=1, act=3, b1=4.0, b2=25.0, out=one, ldo=8, od=1,
              M=2, F=8, K=16):
        return lib.vmi_gated_linear(x, ldx, xs, wg, ldg, gs, wu, ldu, us, dtype, act, b1, b2, out, ldo, od, null, M, F, K, null)

    for kw in (dict(wu=null), dict(act=0), dict(act=2), dict(ldo=7), dict(dtype=3, xs=one, gs=one), dict(F=-1), dict(od=2)):
        assert gated(**kw) == INVALID, kw
    for kw in (dict(ldu=24), dict(wu=odd), dict(x=odd)):
        assert gated(**kw) == UNSUPPORTED, kw
    assert gated(M=0, x=null, out=null) == 0

    n = ctypes.c_size_t(0)
    assert lib.vmi_linear_add_bwd_workspace_bytes(100, 24, 16, 1, 1, ctypes.byref(n)) == 0 and n.value >= 100 * 24 * 2
    assert lib.vmi_linear_add_bwd_workspace_bytes(100, 24, 16, 3, 1, ctypes.byref(n)) == INVALID
    assert lib.vmi_linear_add_bwd_workspace_bytes(100, 24, 16, 1, 1, null) == INVALID
    assert lib.vmi_gated_linear_bwd_workspace_bytes(100, 20, 16, 1, ctypes.byref(n)) == 0 and n.value >= 100 * 48 * 2
    assert lib.vmi_gated_linear_bwd_workspace_bytes(100, 20, -16, 1, ctypes.byref(n)) == INVALID
    bwd = lib.vmi_linear_add_bwd
    assert bwd(one, 16, one, 16, 1, null, 1, null, one, 8, one, one, one, 2, 8, 16, null, 0, null) == WORKSPACE
    assert bwd(one, 16, one, 16, 1, null, 1, null, one, 8, one, one, one, 2, 8, 16, ctypes.c_void_p(8), 1 << 30, null) == WORKSPACE
    assert bwd(one, 16, one, 16, 1, null, 5, null, one, 8, one, one, one, 2, 8, 16, one, 1 << 30, null) == INVALID
    assert bwd(one, 16, one, 16, 1, null, 1, null, odd, 8, one, one, one, 2, 8, 16, one, 1 << 30, null) == UNSUPPORTED
    assert bwd(one, 16, one, 16, 1, null, 1, null, null, 8, one, one, one, 2, 8, 16, one, 1 << 30, null) == INVALID
    assert bwd(one, 16, one, 16, 1, null, 1, null, one, 1 << 23, one, one, one, 0, 1 << 23, 16, one, 1 << 40, null) == UNSUPPORTED
    gb = lib.vmi_gated_linear_bwd
    assert gb(one, 16, one, 16, one, 16, 1, 3, 4.0, 25.0, null, one, 1 << 22, one, one, 0, 1 << 22, 16, one, 1 << 40, null) == UNSUPPORTED
    assert gb(one, 16, one, 16, one, 16, 1, 0, 4.0, 25.0, null, one, 8, one, one, 2, 8, 16, one, 1 << 30, null) == INVALID
    assert gb(one, 16, one, 16, one, 24, 1, 3, 4.0, 25.0, null, one, 8, one, one, 2, 8, 16, one, 1 << 30, null) == UNSUPPORTED
    assert gb(one, 16, one, 16, one, 16, 1, 3, 4.0, 25.0, null, one, 7, one, one, 2, 8, 16, one, 1 << 30, null) == INVALID
    assert gb(one, 16, one, 16, one, 16, 1, 3, 4.0, 25.0, null, one, 8, one, one, 2, 8, 16, one, 16, null) == WORKSPACE

    def quant(a=one, st=16, r=null, rs=0, w=null, dtype=1, wd=1, norm=1, s=one, q=one, scale=one, rows=2, d=16):
        return lib.vmi_norm_add_quant(a, st, r, rs, w, dtype, wd, norm, 1e-6, s, q, scale, rows, d, null)

    for kw in (dict(a=null), dict(q=null), dict(scale=null), dict(dtype=3, wd=3), dict(wd=2), dict(d=0), dict(rows=-1), dict(d=1 << 31)):
        assert quant(**kw) == INVALID, kw
    assert quant(rows=0, a=null, q=null, scale=null) == 0
    assert lib.vmi_pad_rows(null, 16, one, 2, 10, null) == INVALID and lib.vmi_pad_rows(one, 16, odd, 2, 10, null) == INVALID
    assert lib.vmi_pad_rows(one, -1, one, 2, 10, null) == INVALID and lib.vmi_pad_rows(null, 16, null, 0, 10, null) == 0


def test_pad_refusals(lib):
    """Several matrices at once: each is checked before any is copied; none with rows is no launch."""
    from ctypes import c_void_p
    null, one, odd = c_void_p(None), c_void_p(256), c_void_p(260)
    INVALID = 1
    none = (null, 0, null, 0, 0)
    assert lib.vmi_pad_rows_3(*none, *none, *none, null) == 0
    assert lib.vmi_pad_rows_3(null, 16, null, 0, 10, null, 16, null, 0, 10, null, 16, null, 0, 10, null) == 0
    for bad in ((null, 16, one, 2, 10), (one, 16, odd, 2, 10), (one, -1, one, 2, 10), (one, 16, one, -2, 10), (one, 16, one, 2, -10),
                (one, 16, one, 2 ** 62, 2 ** 62)):
        for at in range(3):
            assert lib.vmi_pad_rows_3(*[v for i in range(3) for v in (bad if i == at else none)], null) == INVALID


def test_oracle_e4m3():
    """The oracle's rounding is torch's where torch's input type does not round first."""
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(4000, generator=g) * s for s in (1e-3, 0.1, 1.0, 50.0)] + [torch.linspace(-448, 448, 4097)]).clamp(-448, 448)
    assert torch.equal(oracle.to_e4m3(x.double()), x.to(E4M3).double())


@fake
def test_eps_below_zero():
    for eps in (-1e-6, float("nan")):
        with pytest.raises(RuntimeError, match="eps"):
            va.norm_add_quant(_e(3, 16), eps=eps)
