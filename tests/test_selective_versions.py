"""An in-place step tells autograd: a backward that needs the state from before it raises, and a state that requires grad
is refused.  On the host, with stand-ins for the launchers."""
import pytest
import torch

import verace_amd as va
from verace_amd import selective


def _conv_step(x, weight, bias, state, *rest):
    state.data.add_(1)
    return x.reshape(x.shape[0], 1, -1) + 0


def _step(x, delta, A, B, C, state, *rest):
    state.data.mul_(2)
    return x.reshape(x.shape[0], 1, *x.shape[-2:]) + 0


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(selective, "_require_device", lambda *a: None)
    monkeypatch.setattr(selective, "_launch_conv", lambda x, w, b, state, n, act: (x + 0, x[:, :3] + 0))
    monkeypatch.setattr(selective, "launch_selective_hip_scan", lambda x, d, A, B, *rest: (x + 0, torch.zeros(2, 2, 4, 3)))
    monkeypatch.setattr(selective, "_launch_conv_step", _conv_step)
    monkeypatch.setattr(selective, "_launch_selective_step", _step)


W, BM, A, D1 = torch.ones(8, 4), torch.ones(2, 5, 1, 3), -torch.ones(2), torch.ones(2, 5, 2)


def conv(x, s):
    return va.short_conv(x, W, None, s)[0]


def conv_step(x, s):
    return va.short_conv_step_(x[:, 0].detach(), W, None, s)


def scan(x, s):
    return va.selective_scan(x.view(2, 5, 2, 4), D1, A, BM, BM, initial_state=s)[0]


def step(x, s):
    return va.selective_step_(x[:, 0].detach().view(2, 2, 4), D1[:, 0], A, BM[:, 0], BM[:, 0], s)


@pytest.mark.parametrize("whole,one,shape", [(conv, conv_step, (2, 3, 8)), (scan, step, (2, 2, 4, 3))], ids=["conv", "scan"])
def test_backward_after_a_step(host, whole, one, shape):
    x, state = torch.randn(2, 5, 8, requires_grad=True), torch.zeros(shape)
    y, before = whole(x, state), state._version
    one(x, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        one(torch.zeros(2, 5, 8), torch.zeros(shape))


@pytest.mark.parametrize("one,shape", [(conv_step, (2, 3, 8)), (step, (2, 2, 4, 3))], ids=["conv", "scan"])
def test_a_state_that_requires_grad(host, one, shape):
    x, state = torch.randn(2, 5, 8), torch.zeros(shape, requires_grad=True)
    with pytest.raises(RuntimeError, match="requires grad"):
        one(x, state)
    with torch.no_grad():
        one(x, state)
