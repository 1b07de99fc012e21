"""The feed-forward operators where their arithmetic loses bits, runs out of fp32's range or cancels; each result near its own
value, however small."""

import math

import pytest
import torch

from oracle import feed_forward as oracle
from test_gpu_feed_forward import randn, va, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
E4M3 = oracle.E4M3


@pytest.mark.parametrize("m,n", [(3, 24), (300, 640)])
def test_sums_of_8_bit_rows(m, n):
    """By the kernel for a few rows and by tiles, with a 32-bit result: where one value stands out of a row, its seven neighbours'
    products keep 2^-13 of its power of two; products elsewhere, and rows without one, lose nothing to it."""
    g = torch.Generator().manual_seed(m)
    k = 144
    x, w = (torch.randn(r, k, generator=g).to(E4M3) for r in (m, n))
    x[::2, 21] = 448.0
    one = [torch.ones(r, device="cuda") for r in (m, n)]
    X, W = oracle.values(x), oracle.values(w)
    y = va().linear_add(x.cuda(), w.cuda(), None, None, *one, out_dtype=torch.float32)
    within(y, *oracle.linear(X, W, None, None, None, torch.float32, one))
    h = va().gated_linear(x.cuda(), w.cuda(), w.cuda(), one[0], one[1], one[1], activation="silu", out_dtype=torch.float32)
    within(h, *oracle.gated(X, W, W, "silu", torch.float32, scales=(one[0], one[1], one[1])))
    # the outstanding value's own eight apart: the rest of its row is as exact as a row without it
    rest = X.clone()
    rest[:, 16:24] = 0
    only = va().linear_add(rest.to(E4M3).cuda(), w.cuda(), None, None, *one, out_dtype=torch.float32)
    within(only, *oracle.linear(rest, W, None, None, None, torch.float32, one))


LEAST, MOST = 2.0 ** -64, 2.0 ** 64


@pytest.mark.parametrize("dtype", DTYPES + [E4M3])
@pytest.mark.parametrize("m", [5, 300])
def test_betas_at_their_limits(m, dtype):
    """By the kernel for a few rows and by tiles; u = 0 in one column."""
    g = torch.Generator().manual_seed(m)
    k, f = 64, 600
    x, wg, wu = randn(g, m, k), randn(g, f, k, scale=0.1), randn(g, f, k, scale=0.1)
    wu[7] = 0
    out = torch.bfloat16 if dtype == E4M3 else dtype
    (x, xs), (wg, gs), (wu, us) = ((t.to(dtype), None) if dtype != E4M3 else va().quantize_rows(t) for t in (x, wg, wu))
    X, G, U = oracle.values(x, xs), oracle.values(wg, gs), oracle.values(wu, us)
    for b1 in (LEAST, 4.0, MOST):
        for b2 in (LEAST, 25.0, MOST):
            h = va().gated_linear(x, wg, wu, xs, gs, us, beta1=b1, beta2=b2)
            scales = None if xs is None else (xs, gs, us)
            want, bound = oracle.gated(X, G, U, "situ", out, b1, b2, scales)
            # the least beta makes a step of its factor, on whose other side a projection may come out that is nearer 0 than its error
            (z, ez), (v, ev) = (oracle.product(X, W, None if s is None else (xs, s)) for W, s in ((G, gs), (U, us)))
            bound = bound + 2 * b1 * b2 * ((z.abs() <= ez) & (b1 == LEAST) | (v.abs() <= ev) & (b2 == LEAST)).double()
            within(h, want, bound)
            assert bool((h[:, 7] == 0).all())


def columns(v, dtype):
    """A projection to each value itself: (x, w), and the values in 64 bits."""
    x = torch.zeros(v.numel(), 16, dtype=dtype)
    x[:, 0] = v.to(dtype)
    w = torch.zeros(3, 16, dtype=dtype)
    w[:, 0] = 1
    return x.cuda(), w.cuda(), x[:, :1].double()


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_far_out(dtype, kept, monkeypatch):
    """z Phi(z) and its slope relative to their own values, where 1 + erf would cancel.

    In 16 bits: within 2^-18 (a polynomial of 2^-20, an exponential and a reciprocal of a few 2^-24), and z^2 / 2 itself is off by
    2^-23 of it (two roundings), which goes into the exponential.  fp32: 16 roundings of 2^-23 (the library's own few among them).
    Near the slope's zero (z = -0.75) its two terms cancel: their magnitudes count."""
    monkeypatch.setattr("verace_amd.feed_forward._keeps", lambda *_: kept)
    v = torch.cat([torch.linspace(-13, 13, 1041), torch.tensor([0.0, 1e-6, -1e-6, -1e-3, 40.0, -40.0, 1e4, -1e4])])
    x, w, z = columns(v, dtype)
    x.requires_grad_()
    y = va().linear_add(x, w, activation="gelu")
    phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    density = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    own = 2.0 ** -18 + z * z * 2.0 ** -23 if dtype != torch.float32 else torch.full_like(z, 2.0 ** -19)
    want = z * phi
    within(y, want.expand(-1, 3), (own * want.abs() + z.abs() * oracle.TINY + oracle.rounding(want, dtype)).expand(-1, 3))
    slope = phi + z * density
    dx, = torch.autograd.grad(y, x, torch.cat([torch.ones_like(y[:, :1]), torch.zeros_like(y[:, 1:])], 1))
    # rounded as an operand, and again as the result
    bound = own * (phi + (z * density).abs()) + (1 + z.abs()) * oracle.TINY + 2 * oracle.rounding(slope, dtype)
    within(dx[:, :1], slope, bound)
    if dtype == torch.float32:  # the same through 16-bit rows of a 32-bit result: the values have four bits
        e = torch.tensor([-8.0, -6.5, -6.0, -5.5, -5.0, -4.5, -4.0, -3.0, 2.0, 448.0]).to(E4M3).float()
        x8, w8 = torch.zeros(e.numel(), 16), torch.zeros(3, 16)
        x8[:, 0], w8[:, 0] = e, 1
        one, three = torch.ones(e.numel(), device="cuda"), torch.ones(3, device="cuda")
        y = va().linear_add(x8.to(E4M3).cuda(), w8.to(E4M3).cuda(), None, None, one, three, activation="gelu", out_dtype=torch.float32)
        z = e.double()[:, None]
        want = z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
        within(y, want.expand(-1, 3), (2.0 ** -19 * want.abs() + oracle.rounding(want, torch.float32)).expand(-1, 3))


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_situ_slopes_where_tanh_saturates(dtype, kept, monkeypatch):
    """1 - tanh^2 relative to its own value, where the difference would cancel.

    sech^2 is formed from exp(-2 |x|), x = g / b1 or u / b2: x carries two roundings of 2^-24 (the inverse and the product) and its
    exponent's scale two more, so sech^2 is off by 4 x 2^-23 relative beside 2^-18 for its own operations; each gradient is rounded
    as an operand and as the result.  The gate's slope has a second term, a(g) sigmoid(-g)."""
    monkeypatch.setattr("verace_amd.feed_forward._keeps", lambda *_: kept)
    v = torch.tensor([0.0, 0.3, 0.59, 0.61, 1.0, 2.0, 3.0, 4.0, 5.0, 6.0, 7.0, 8.0, 9.0, 12.0, 30.0])
    v = torch.cat([v, -v])
    n = v.numel()
    x = torch.zeros(n * n, 16, dtype=dtype)
    x[:, 0], x[:, 1] = (4 * v).to(dtype).repeat_interleave(n), (25 * v).to(dtype).repeat(n)
    wg, wu = torch.zeros(1, 16, dtype=dtype), torch.zeros(1, 16, dtype=dtype)
    wg[:, 0], wu[:, 1] = 1, 1
    g, u = x[:, 0].double(), x[:, 1].double()
    x, wg, wu = (t.cuda().requires_grad_() for t in (x, wg, wu))
    h = va().gated_linear(x, wg, wu)
    dx, = torch.autograd.grad(h, x, torch.ones_like(h))

    def sech2(t):
        e = torch.exp(-2 * t.abs())
        return 4 * e / (1 + e) ** 2

    s, ns = torch.sigmoid(g), torch.sigmoid(-g)
    a, b = 4 * torch.tanh(g / 4) * s, 25 * torch.tanh(u / 25)
    one, two = sech2(g / 4) * s * b, a * ns * b
    du = a * sech2(u / 25)
    off_g, off_u = 2.0 ** -18 + (g / 4).abs() * 2.0 ** -21 + g.abs() * 2.0 ** -22, 2.0 ** -18 + (u / 25).abs() * 2.0 ** -21 + g.abs() * 2.0 ** -22
    least = oracle.TINY * 100 * (1 + g.abs())
    within(dx[:, 0], one + two, off_g * (one.abs() + two.abs()) + least + 2 * oracle.rounding(one + two, dtype))
    within(dx[:, 1], du, off_u * du.abs() + least + 2 * oracle.rounding(du, dtype))


@pytest.mark.parametrize("m", [8, 304])
def test_scales_beyond_each_other(m):
    """8-bit rows whose two scales multiply to no normal fp32 number, where their values do not: a sum of 0 stays 0, the others keep
    their precision, down to fp32's own least number and up to its largest."""
    g = torch.Generator().manual_seed(m)
    k, n = 64, 640
    xs = torch.tensor([2.0 ** -126, 2.0 ** -100, 2.0 ** -70, 1e-3, 1.0, 2.0 ** 40, 2.0 ** 90, 2.0 ** 119]).repeat(m // 8)
    ws = torch.tensor([2.0 ** -126, 2.0 ** -75, 2.0 ** -60, 2.0 ** -9, 3.0, 2.0 ** 20, 2.0 ** 60, 2.0 ** 118]).repeat(n // 8)
    x, w = torch.randn(m, k, generator=g) * 30, torch.randn(n, k, generator=g) * 30
    x[:, k // 2:] = 0                                 # the columns below meet only zeros in these rows' values
    w[: n // 2, : k // 2] = 0
    w[n // 2::3, 5:] = 0
    x[::2, 5:] = 0
    x, w = x.to(E4M3), w.to(E4M3)
    X, W = x.double() * xs.double()[:, None], w.double() * ws.double()[:, None]
    args = x.cuda(), w.cuda(), None, None, xs.cuda(), ws.cuda()
    for out in DTYPES:
        y = va().linear_add(*args, out_dtype=out)
        want, bound = oracle.linear(X, W, None, None, None, out, (xs, ws))
        top = torch.finfo(out).max
        fine = want.abs() + bound < top
        assert bool(torch.isfinite(y.cpu())[fine].all()) and bool((y.cpu()[want == 0] == 0).all())
        within(torch.where(fine.cuda(), y, 0), torch.where(fine, want, 0), bound)
        assert bool((y.cpu().double().abs() >= top)[want.abs() - bound > 1.01 * top].all())
    h = va().gated_linear(args[0], args[1], args[1], args[4], args[5], args[5], activation="silu", out_dtype=torch.float32)
    want, bound = oracle.gated(X, W, W, "silu", torch.float32, scales=(xs, ws, ws))
    top = torch.finfo(torch.float32).max
    fine = (want.abs() + bound < top) & ((X @ W.T).abs() < top)  # the projections themselves are fp32
    assert bool((h.cpu()[fine & (want == 0)] == 0).all())
    within(torch.where(fine.cuda(), h, 0), torch.where(fine, want, 0), bound)
