"""The selective layer's operators where something besides the caller looks on: a jit trace replayed on other inputs, a
function mode, autograd holding a state that a step overwrites."""
import pytest
import torch

from test_gpu_selective import inputs

pytestmark = pytest.mark.gpu


def _calls(device):
    d, state = inputs(device, 2, 40, 2, 32, 1, 16, torch.bfloat16, seed=80)
    w, b = torch.randn(64, 4, device=device).bfloat16(), torch.randn(64, device=device).bfloat16()

    def layer(x):
        from verace_amd import gated_norm_add, selective_scan, selective_step_, short_conv, short_conv_step_
        c, last = short_conv(x, w, b)
        y, S = selective_scan(c.view(2, 40, 2, 32), d["delta"], d["A"], d["B"], d["C"], d["D"], d["delta_bias"], initial_state=state)
        s, n = gated_norm_add(y.flatten(2), x, b, c, None, b)
        t = short_conv_step_(x[:, 0], w, b, last.detach().clone())
        z = selective_step_(t.view(2, 1, 2, 32), d["delta"][:, :1], d["A"], d["B"][:, :1], d["C"][:, :1], S.detach().clone())
        return y, S, s, n, t, z
    return layer, [torch.randn(2, 40, 64, device=device).bfloat16() for _ in range(3)]


def test_jit_trace(device):
    layer, xs = _calls(device)
    with torch.no_grad():
        fn = torch.jit.trace(layer, (xs[0],))
        for x in xs:
            for a, b in zip(fn(x), layer(x)):
                assert torch.equal(a, b)


def test_function_mode(device):
    """A default device is one: results stay the same, and gradients."""
    layer, xs = _calls(device)
    outs = []
    for default in (None, device):
        torch.set_default_device(default)
        try:
            x = xs[0].clone().requires_grad_()
            y, S, s, n, _, _ = layer(x)
            outs.append([y.detach(), S.detach(), *torch.autograd.grad(s.float().sum() + n.float().square().sum() + S.sum(), x)])
        finally:
            torch.set_default_device(None)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_backward_after_a_step(device):
    """The scan's and the convolution's backward read the state they were given: after a step on it they raise."""
    from verace_amd import selective_scan, selective_step_, short_conv, short_conv_step_
    d, state = inputs(device, 2, 40, 2, 32, 1, 16, torch.float32, seed=81)
    x = d["x"].clone().requires_grad_()
    y, _ = selective_scan(**{**d, "x": x}, initial_state=state)
    tok = {k: d[k][:, :1] for k in ("x", "delta", "B", "C")}
    kept = state.clone()
    selective_step_(tok["x"], tok["delta"], d["A"], tok["B"], tok["C"], state)
    assert not torch.equal(kept, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    c, w, s = torch.randn(2, 9, 8, device=device, requires_grad=True), torch.randn(8, 4, device=device), torch.randn(2, 3, 8, device=device)
    y, _ = short_conv(c, w, None, s)
    short_conv_step_(c.detach()[:, 0], w, None, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
