"""The selective layer's operators where something besides the caller looks on: a jit trace replayed on other inputs, a
function mode."""
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
        t = short_conv_step_(x[:, 0], w, b, last.clone())
        z = selective_step_(t.view(2, 1, 2, 32), d["delta"][:, :1], d["A"], d["B"][:, :1], d["C"][:, :1], S.clone())
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
