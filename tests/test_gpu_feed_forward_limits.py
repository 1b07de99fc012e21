"""The feed-forward operators where their arithmetic loses bits, runs out of fp32's range or cancels; each result near its own
value, however small."""

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
