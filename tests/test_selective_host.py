"""Refusals of the selective scan, the short convolution and the gated norms, on the host: shapes and
types through the Python entry points (fake device tensors, nothing is launched) and arguments through the
C ABI."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import verace_amd as va


@pytest.fixture(scope="module")
def lib():
    from verace_amd import _lib
    return _lib.load()


def _e(*s, dtype=torch.float32, device="cuda"):
    return torch.empty(*s, dtype=dtype, device=device)


def _scan(**kw):
    a = dict(x=_e(2, 5, 4, 16), delta=_e(2, 5, 4), A=_e(4), B=_e(2, 5, 2, 8), C=_e(2, 5, 2, 8))
    a.update(kw)
    return va.selective_scan(**a)


@pytest.mark.parametrize("bad", [
    dict(x=(2, 5, 64)), dict(delta=(2, 5, 3)), dict(delta=(2, 4, 4)), dict(A=(3,)), dict(B=(2, 5, 8)),
    dict(C=(2, 5, 2, 9)), dict(B=(2, 4, 2, 8), C=(2, 4, 2, 8)), dict(B=(2, 5, 3, 8), C=(2, 5, 3, 8)),
    dict(B=(2, 5, 2, 257), C=(2, 5, 2, 257)), dict(D=(5,)), dict(delta_bias=(1,)), dict(initial_state=(2, 4, 16, 9)),
    dict(lengths=(3,)), dict(lengths=(2,)), dict(x=(2, 5, 4, 1025))])
def test_scan_refusals(bad):
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(RuntimeError, match="verace_amd"):
            _scan(**{k: _e(*v) for k, v in bad.items()})


def test_scan_type_refusals():
    with FakeTensorMode(allow_non_fake_inputs=True):
        for kw in (dict(x=_e(2, 5, 4, 16, dtype=torch.float64)), dict(B=_e(2, 5, 2, 8, dtype=torch.bfloat16)),
                   dict(delta=_e(2, 5, 4, dtype=torch.int32)), dict(x=_e(2, 5, 4, 16, device="cpu")),
                   dict(A=_e(4, device="cpu"))):
            with pytest.raises(RuntimeError, match="verace_amd"):
                _scan(**kw)


def test_step_refusals():
    with FakeTensorMode(allow_non_fake_inputs=True):
        ok = dict(x=_e(2, 1, 4, 16), delta=_e(2, 1, 4), A=_e(4), B=_e(2, 1, 2, 8), C=_e(2, 1, 2, 8), state=_e(2, 4, 16, 8))
        for bad in (dict(state=_e(2, 4, 8, 16)), dict(state=_e(2, 4, 16, 8, dtype=torch.bfloat16)),
                    dict(state=_e(2, 4, 8, 16).transpose(2, 3)), dict(A=_e(2)),
                    dict(x=_e(2, 2, 4, 16), delta=_e(2, 2, 4), B=_e(2, 2, 2, 8), C=_e(2, 2, 2, 8))):
            with pytest.raises(RuntimeError, match="verace_amd"):
                va.selective_step_(**{**ok, **bad})


def test_conv_refusals():
    with FakeTensorMode(allow_non_fake_inputs=True):
        ok = dict(x=_e(2, 5, 8), weight=_e(8, 4))
        for bad in (dict(x=_e(2, 8)), dict(weight=_e(4, 8)), dict(weight=_e(8, 5)), dict(weight=_e(8, 1)), dict(bias=_e(7)),
                    dict(bias=_e(8, dtype=torch.bfloat16)), dict(initial_state=_e(2, 4, 8)),
                    dict(initial_state=_e(2, 3, 8, dtype=torch.bfloat16)), dict(activation="relu"), dict(lengths=_e(2)),
                    dict(x=_e(2, 5, 8, device="cpu"))):
            with pytest.raises(RuntimeError, match="verace_amd"):
                va.short_conv(**{**ok, **bad})
        for bad in (dict(state=_e(2, 4, 8)), dict(state=_e(2, 8, 3).transpose(1, 2)), dict(x=_e(2, 2, 8)), dict(x=_e(3, 8))):
            with pytest.raises(RuntimeError, match="verace_amd"):
                va.short_conv_step_(**{**dict(x=_e(2, 8), weight=_e(8, 4), bias=None, state=_e(2, 3, 8)), **bad})


def test_norm_refusals():
    with FakeTensorMode(allow_non_fake_inputs=True):
        ok = dict(y=_e(3, 8), residual=_e(3, 8))
        for bad in (dict(residual=_e(3, 9)), dict(residual=_e(3, 8, dtype=torch.bfloat16)), dict(gate=_e(2, 8)),
                    dict(norm_weight=_e(9)), dict(norm_weight=_e(8, dtype=torch.bfloat16)), dict(activation="tanh"),
                    dict(y=_e(3, 8, device="cpu")), dict(y=_e(2, 8192), residual=_e(2, 8192))):
            with pytest.raises(RuntimeError, match="verace_amd"):
                va.gated_norm_add(**{**ok, **bad})
        y = _e(3, 8, dtype=torch.bfloat16)
        with pytest.raises(RuntimeError, match="one dtype"):
            va.gated_norm_add(y, y, norm_weight=_e(8), scale=_e(8, dtype=torch.bfloat16))


def test_c_refusals(lib):
    n = ctypes.c_size_t(0)
    q = lib.vmi_selective_scan_workspace_bytes
    assert q(1, 10, 2, 16, 1, 16, 1, ctypes.byref(n)) == 0
    assert q(1, 10, 3, 16, 2, 16, 1, ctypes.byref(n)) == 1      # heads that no groups share
    assert q(1, 10, 2, 16, 1, 0, 1, ctypes.byref(n)) == 1
    assert q(1, 10, 2, 16, 1, 257, 1, ctypes.byref(n)) == 2
    assert q(1, 10, 2, 16, 1, 16, 9, ctypes.byref(n)) == 1
    assert q(1, 10, 2, 16, 1, 16, 1, None) == 1
    c = lib.vmi_short_conv_bwd_workspace_bytes
    assert c(2, 100, 8, 4, ctypes.byref(n)) == 0 and n.value > 0
    assert c(2, 100, 8, 5, ctypes.byref(n)) == 2
    assert c(2, -1, 8, 4, ctypes.byref(n)) == 1
    g = lib.vmi_gated_norm_bwd_workspace_bytes
    assert g(10, 64, 0, ctypes.byref(n)) == 0 and n.value > 0
    assert g(10, 5000, 0, ctypes.byref(n)) == 2
    assert g(10, 0, 0, ctypes.byref(n)) == 1
    null = ctypes.c_void_p(0)
    one = ctypes.c_void_p(16)
    assert lib.vmi_short_conv(null, 8, 8, null, null, 0, 0, 1, null, null, 0, null, null, 1, 1, 8, 4, null) == 1
    assert lib.vmi_short_conv(one, 8, 8, one, null, 0, 0, 1, one, null, 0, one, one, 1, 1, 8, 4, null) == 4
    assert lib.vmi_gated_norm(one, 8, one, 8, null, 0, null, null, one, 0, 0, 1, 0.0, 0.0, one, null, null, 1, 8, null) == 1
    assert lib.vmi_gated_norm(one, 8, one, 8, null, 0, null, null, null, 1, 2, 1, 0.0, 0.0, one, null, null, 1, 8, null) == 2


def test_traced_shapes():
    """Fake HIP tensors go through the registered operators: shapes and dtypes, gradients, refusals; no kernel runs."""
    with FakeTensorMode(allow_non_fake_inputs=True):
        bf = torch.bfloat16
        x, delta, bm = _e(2, 40, 4, 16, dtype=bf), _e(2, 40, 4), _e(2, 40, 2, 8, dtype=bf)
        y, state = va.selective_scan(x, delta, _e(4), bm, bm, _e(4), lengths=_e(2, dtype=torch.int32))
        assert y.shape == x.shape and y.dtype == bf and state.shape == (2, 4, 16, 8) and state.dtype == torch.float32
        c, last = va.short_conv(y.flatten(2), _e(64, 4, dtype=bf), _e(64, dtype=bf))
        assert c.shape == (2, 40, 64) and last.shape == (2, 3, 64) and last.dtype == bf
        s, n = va.gated_norm_add(c, c, _e(64), c, None, _e(64))
        assert s.shape == n.shape == c.shape and n.dtype == bf
        assert va.gated_norm_add(c, c, _e(64))[1] is None
        grads = torch.ops.verace.selective_scan_bwd(x, delta, _e(4), bm, bm, y, None, None, True, None, None, None)
        for g, t in zip(grads, (x, delta, _e(4), bm, bm, _e(4), _e(4), _e(0))):
            assert g.shape == t.shape and g.dtype == t.dtype
        with torch.no_grad():
            assert va.selective_step_(x[:, 0], delta[:, 0], _e(4), bm[:, 0], bm[:, 0], state).shape == (2, 1, 4, 16)
            assert va.short_conv_step_(c[:, 0], _e(64, 4), None, last).shape == (2, 1, 64)


def test_gradient_operator_refusals():
    ops = torch.ops.verace
    x, y = torch.zeros(2, 5, 8), torch.zeros(3, 8)
    for call in (lambda: ops.short_conv_bwd(x, torch.zeros(8, 4), None, None, None, "silu", x[:, :4], None),
                 lambda: ops.gated_norm_bwd(y, y, None, None, None, None, torch.zeros(2, 2), "silu", y, None),
                 lambda: ops.selective_scan_bwd(x.view(2, 5, 2, 4), x[..., :2], torch.zeros(2), x.view(2, 5, 2, 4),
                                                x.view(2, 5, 2, 4), x, None, None, True, None, None, None)):
        with pytest.raises(RuntimeError, match="verace_amd"):
            call()
    with FakeTensorMode(allow_non_fake_inputs=True):
        from verace_amd import block_norm, selective
        z = _e(2, 5, 8)
        with pytest.raises(RuntimeError, match="dy must be"):
            selective._launch_conv_bwd(z, _e(8, 4), None, None, None, 1, _e(2, 4, 8), None, (True,) * 4)
        with pytest.raises(RuntimeError, match="d_last must be"):
            selective._launch_conv_bwd(z, _e(8, 4), None, None, None, 1, None, _e(2, 4, 8), (True,) * 4)
        for stats, ds in ((_e(2, 2), _e(3, 8)), (_e(2, 3), _e(3, 4)), (_e(3, 2).t(), _e(3, 8))):
            with pytest.raises(RuntimeError, match="must be"):
                block_norm._launch_bwd(_e(3, 8), _e(3, 8), None, None, None, None, stats, 1, ds, None, (True,) * 6)


def test_backward_refuses_far_and_backward_rows(lib):
    one, null = ctypes.c_void_p(64), None
    for x_t, b_t, y_t in ((-8, 8, 8), (8, -8, 8), (8, 8, -8), ((1 << 23) + 1, 8, 8), (8, (1 << 23) + 1, 8)):
        assert lib.vmi_selective_scan_bwd(one, x_t, 64, one, 1, 8, 0, one, one, b_t, 64, one, 8, 64, null, null, 1, 0, null,
                                          null, 0, one, y_t, 64, null, one, one, one, one, one, null, null, null,
                                          1, 8, 1, 8, 1, 8, one, 1 << 40, null) == 2
