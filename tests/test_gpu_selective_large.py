"""The selective state space layer's operators on tensors of more than 2^31 elements: their last rows against the
same operators on those rows alone."""
import pytest
import torch

from test_gpu_selective import U
from test_gpu_selective_bwd import magnitudes

pytestmark = pytest.mark.gpu


def _randn(device, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, device=device, dtype=dtype, generator=torch.Generator(device).manual_seed(seed))


def test_scan(device):
    """Steps of 0.5 at a rate of -2: after 600 tokens nothing is left of a state (e^-600), so the last 640 tokens alone
    give the last 40 outputs, and the same gradients of x from the end on.  Either run is within the derived bound of
    the exact value, so within twice that of the other."""
    from oracle import selective as ref
    from verace_amd import selective_scan
    T, H, P, N, last = 1048640, 32, 64, 16, 640
    x = _randn(device, 1, T, H, P)
    assert x.numel() > 2 ** 31
    delta = torch.full((1, T, H), 0.5, device=device)
    A = torch.full((H,), -2.0, device=device)
    B, C = _randn(device, 1, T, 1, N, seed=1), _randn(device, 1, T, 1, N, seed=2)
    dy = _randn(device, 1, T, H, P, seed=3)
    print("[case] scan of", x.numel(), "elements", flush=True)
    x.requires_grad_(True)
    y, S = selective_scan(x, delta, A, B, C, softplus=False)
    dx, = torch.autograd.grad(y, x, dy)
    d = dict(x=x.detach()[:, -last:], delta=delta[:, -last:], A=A, B=B[:, -last:], C=C[:, -last:], D=None, delta_bias=None)
    xs = d["x"].clone().requires_grad_(True)
    ys, Ss = selective_scan(**{**d, "x": xs}, softplus=False)
    dxs, = torch.autograd.grad(ys, xs, dy[:, -last:])
    ym, Sm = ref.selective_scan(**d, softplus=False, magnitude=True)
    h = torch.finfo(x.dtype).eps / 2
    a, b = y[:, -40:].double(), ys[:, -40:].double()
    assert bool(((a - b).abs() <= 2 * (h * b.abs() * 1.01 + ((8 * last + N + 16) * U + 2.0 ** -8) * ym[:, -40:])).all())
    assert bool(((S.double() - Ss.double()).abs() <= 2 * (8 * last + 16) * U * Sm).all())
    m = magnitudes(d, None, dy[:, -last:], None, None, False)["x"]
    a, b = dx[:, -last:].double(), dxs.double()
    assert bool(((a - b).abs() <= 2 * (h * b.abs() * 1.01 + ((8 * last + N + P + 64) * U + 2.0 ** -7) * m)).all())


def test_conv(device):
    """A token's sums run in one order wherever it lies: the same bits."""
    from verace_amd import short_conv
    T, C, last = 933000, 2304, 100
    x, w, b = _randn(device, 1, T, C), _randn(device, C, 4, seed=1), _randn(device, C, seed=2)
    assert x.numel() > 2 ** 31
    print("[case] convolution of", x.numel(), "elements", flush=True)
    dy = _randn(device, 1, T, C, seed=3)
    x.requires_grad_(True)
    y, end = short_conv(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    xs = x.detach()[:, -last:].clone().requires_grad_(True)
    ys, ends = short_conv(xs, w, b, x.detach()[:, -last - 3:-last].contiguous())
    dxs, = torch.autograd.grad(ys, xs, dy[:, -last:].contiguous())
    assert torch.equal(y[:, -last:], ys) and torch.equal(end, ends) and torch.equal(dx[:, -last:], dxs)


def test_norm(device):
    """Rows are independent: the same bits."""
    from verace_amd import gated_norm_add
    rows, d = 2100000, 1024
    t = [_randn(device, rows, d, seed=k) for k in range(5)]
    assert t[0].numel() > 2 ** 31
    w1, sc, w2 = (_randn(device, d, seed=10 + k) for k in range(3))
    print("[case] norm of", t[0].numel(), "elements", flush=True)
    outs = []
    for part in (slice(None), slice(rows - 300, rows)):
        leaf = [v[part].detach().requires_grad_(True) for v in t[:3]]
        s, n = gated_norm_add(leaf[0], leaf[1], w1, leaf[2], sc, w2)
        outs.append([v[-300:].clone() for v in (s.detach(), n.detach(), *torch.autograd.grad((s, n), leaf, (t[3][part], t[4][part])))])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
