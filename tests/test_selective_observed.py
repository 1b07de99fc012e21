"""What observes torch's operators sees the selective layer's too: jit traces, dispatch and function modes record the
registered operator, forward-mode derivatives raise.  On the host, with stand-ins for the launchers."""
import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

import verace_amd as va
from verace_amd import block_norm, selective


def _conv(x, weight, *rest):
    return 2 * x, x[:, :weight.shape[1] - 1] + 1


def _scan(x, delta, A, B, C, *rest):
    return 3 * x, (x[:, 0].unsqueeze(-1) * B[:, 0, :1].unsqueeze(2)).float()


def _norm(y, residual, gate, w1, scale, w2, *rest):
    return y + residual, None if w2 is None else 2 * y, torch.zeros(2, y.numel() // y.shape[-1])


def _step(x, *rest):
    return x.reshape(x.shape[0], 1, *x.shape[-2:]) + 1


def _conv_step(x, *rest):
    return x.reshape(x.shape[0], 1, x.shape[-1]) + 1


@pytest.fixture
def host(monkeypatch):
    for m in (selective, block_norm):
        monkeypatch.setattr(m, "_require_device", lambda *a: None)
    monkeypatch.setattr(selective, "_launch_conv", _conv)
    monkeypatch.setattr(selective, "launch_selective_hip_scan", _scan)
    monkeypatch.setattr(selective, "_launch_selective_step", _step)
    monkeypatch.setattr(selective, "_launch_conv_step", _conv_step)
    monkeypatch.setattr(block_norm, "_launch", _norm)


W, BM, A, ST = torch.ones(8, 4), torch.ones(2, 5, 1, 3), -torch.ones(2), torch.zeros(2, 2, 4, 3)
CALLS = {
    "short_conv": lambda x: va.short_conv(x, W)[0],
    "short_conv_step_": lambda x: va.short_conv_step_(x[:, :1], W, None, torch.zeros(2, 3, 8)),
    "selective_scan": lambda x: va.selective_scan(x.view(2, 5, 2, 4), x[..., :2], A, BM, BM)[0],
    "selective_step_": lambda x: va.selective_step_(x[:, :1].view(2, 1, 2, 4), x[:, :1, :2], A, BM[:, :1], BM[:, :1], ST.clone()),
    "gated_norm": lambda x: va.gated_norm_add(x, x, W[:, 0])[0],
}


@pytest.mark.parametrize("name", CALLS)
def test_jit_trace(host, name):
    x = torch.randn(2, 5, 8)
    fn = torch.jit.trace(CALLS[name], (x,))
    assert "verace::" + name in str(fn.graph)
    other = torch.randn(2, 5, 8)
    assert torch.equal(fn(other), CALLS[name](other))


@pytest.mark.parametrize("name", CALLS)
def test_modes(host, name):
    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    x = torch.randn(2, 5, 8)
    for mode in (Dispatch, Function):
        seen.clear()
        with mode():
            got = CALLS[name](x)
        assert any("verace." + name in s for s in seen), seen
        assert torch.equal(got, CALLS[name](x))
    with Function(), Dispatch():
        assert torch.equal(CALLS[name](x), CALLS[name](x))


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_raises(host, name):
    x = torch.randn(2, 5, 8)
    with fwad.dual_level():
        CALLS[name](x)  # without a tangent, as ever
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[name](fwad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError):
        torch.func.jvp(CALLS[name], (x,), (x,))


def test_forward_mode_in_any_argument(host):
    x, t = torch.randn(2, 5, 8), torch.ones
    with fwad.dual_level():
        d = lambda v: fwad.make_dual(v, torch.ones_like(v))
        for call in (lambda: va.short_conv(x, d(W)), lambda: va.short_conv(x, W, d(t(8))),
                     lambda: va.short_conv(x, W, None, d(t(2, 3, 8))), lambda: va.gated_norm_add(x, d(x)),
                     lambda: va.gated_norm_add(x, x, None, d(x)), lambda: va.gated_norm_add(x, x, None, None, None, d(t(8))),
                     lambda: va.selective_scan(x.view(2, 5, 2, 4), x[..., :2], d(A), BM, BM),
                     lambda: va.selective_scan(x.view(2, 5, 2, 4), x[..., :2], A, BM, BM, initial_state=d(ST))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
