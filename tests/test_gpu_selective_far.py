"""The selective scan's backward of tokens that lie far apart: a copy's bits; and of tokens too wide, refused before the
forward."""
import pytest
import torch

from test_gpu_selective import inputs
from test_gpu_selective_bwd import grads_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("which", ["x", "B", "C", "dy"])
def test_backward(device, which, T):
    from verace_amd import launch_selective_hip_scan_bwd
    d, state = inputs(device, 1, T, 2, 32, 1, 16, torch.bfloat16, seed=90)
    dy, dS = grads_of(device, d, state, 91)
    want = launch_selective_hip_scan_bwd(**d, dy=dy, initial_state=state, d_state=dS)
    near = dy if which == "dy" else d[which]
    wide = torch.zeros(1, T, (1 << 23) + 8, device=device, dtype=near.dtype)
    far = wide.as_strided(near.shape, (wide.numel(), wide.shape[2], near.shape[3], 1))
    far.copy_(near)
    assert far.stride(1) > 1 << 23
    if which == "dy":
        got = launch_selective_hip_scan_bwd(**d, dy=far, initial_state=state, d_state=dS)
    else:
        got = launch_selective_hip_scan_bwd(**{**d, which: far}, dy=dy, initial_state=state, d_state=dS)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_gradients_through_the_scan(device):
    from verace_amd import selective_scan
    d, state = inputs(device, 1, 20, 2, 32, 1, 16, torch.float32, seed=92)
    wide = torch.zeros(1, 20, (1 << 23) + 8, device=device)
    wide[..., :64] = d["x"].flatten(2)
    leaf = wide.requires_grad_()
    y, S = selective_scan(**{**d, "x": leaf[..., :64].unflatten(-1, (2, 32))}, initial_state=state)
    y.sum().backward()
    x = d["x"].clone().requires_grad_()
    selective_scan(**{**d, "x": x}, initial_state=state)[0].sum().backward()
    assert torch.equal(leaf.grad[..., :64], x.grad.flatten(2))


def test_wide_tokens_are_refused_before_the_forward(device):
    from verace_amd import selective_scan
    H = 8193
    x, delta, A = torch.zeros(1, 1, H, 1024, device=device), torch.zeros(1, 1, H, device=device), torch.zeros(H, device=device)
    B = torch.zeros(1, 1, 1, 1, device=device)
    assert float(selective_scan(x, delta, A, B, B)[0].abs().sum()) == 0.0
    with pytest.raises(RuntimeError, match="differentiable up to"):
        selective_scan(x.requires_grad_(), delta, A, B, B)
