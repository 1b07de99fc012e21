"""What lies behind a sequence's length is exactly zero in the convolution's outputs and gradients, whatever the weights,
the tokens that count and the state hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", ["x", "weight", "bias", "state"])
def test_conv(device, dtype, bad, at):
    from verace_amd import short_conv
    B, T, C, K = 4, 150, 24, 4
    g = torch.Generator(device).manual_seed(1)
    t = {k: torch.randn(*s, generator=g, device=device).to(dtype)
         for k, s in (("x", (B, T, C)), ("weight", (C, K)), ("bias", (C,)), ("state", (B, K - 1, C)))}
    lens = [5, 70, 149, 0]
    n = torch.tensor(lens, device=device)
    if at == "x":
        for i, m in enumerate(lens):
            if m:
                t["x"][i, m - 1] = bad
    else:
        t[at].view(-1)[:] = bad
    leaf = [v.requires_grad_() for v in t.values()]
    y, last = short_conv(leaf[0], leaf[1], leaf[2], leaf[3], n)
    dx, = torch.autograd.grad((y, last), leaf[:1], (torch.ones_like(y), torch.ones_like(last)))
    for i, m in enumerate(lens):
        assert bool((y[i, m:] == 0).all()) and bool((dx[i, m:] == 0).all()), m
