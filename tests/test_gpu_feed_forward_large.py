"""The feed-forward operators on tensors of more than 2^31 elements and 2^32 bytes: the rows at both ends, and what lies between in
its sums, against 64 bits."""
import pytest
import torch

from oracle import feed_forward as oracle
from test_gpu_feed_forward import va, within

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def ends(t, n=3):
    return torch.cat([t[:n], t[-n:]])


def test_many_rows():
    """x and dx of 2^31 + 2^21 elements, of few columns each; the weight's gradient over all of them."""
    m, k, n = (1 << 25) + 32771, 64, 8
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.empty(m, k, device="cuda", dtype=BF)
    for i in range(0, m, 1 << 23):
        x[i:i + (1 << 23)] = torch.randn(x[i:i + (1 << 23)].shape, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda").to(BF).requires_grad_()
    x.requires_grad_()
    y = va().linear_add(x, w)
    within(ends(y), *oracle.linear(oracle.values(ends(x)), oracle.values(w), None, None, None, BF))
    dy = torch.ones((), device="cuda", dtype=BF).expand(m, n)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    (want, bound), *_ = oracle.linear_bwd(oracle.values(ends(x)), oracle.values(w), None, None, oracle.values(ends(dy)), BF)
    within(ends(dx), want, bound)
    total = torch.zeros(k, device="cuda", dtype=torch.float64)
    for i in range(0, m, 1 << 23):
        total += x.detach()[i:i + (1 << 23)].double().sum(0)
    # each sum is of m values around 0: their magnitude is sqrt(m), a share's fp32 partial sums' at most that
    assert bool(((dw.double() - total).abs() <= total.abs() * 2.0 ** -8 + m ** 0.5 * 2.0 ** -8).all())


def test_many_columns():
    """h and y of more than 2^31 elements."""
    m, k, n = 4100, 32, 1 << 19
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(m, k, generator=g, device="cuda").to(BF)
    w = torch.randn(n, k, generator=g, device="cuda").to(BF)
    y = va().linear_add(x, w, activation="silu")
    X, W = oracle.values(x), oracle.values(ends(w))
    rows = torch.cat([y[:2], y[-2:]])
    rows = torch.cat([rows[:, :3], rows[:, -3:]], 1)
    within(rows, *oracle.linear(torch.cat([X[:2], X[-2:]]), W, None, None, "silu", BF))
    del y
    h = va().gated_linear(x, w, w, activation="silu")
    rows = torch.cat([h[:2], h[-2:]])
    rows = torch.cat([rows[:, :3], rows[:, -3:]], 1)
    within(rows, *oracle.gated(torch.cat([X[:2], X[-2:]]), W, W, "silu", BF))


def test_many_rows_in_8_bits():
    m, d = (1 << 21) + 5, 1032
    a = torch.randn(1, d, device="cuda").to(BF).expand(m, d)
    s, q, scale = va().norm_add_quant(a, a, None)
    assert torch.equal(s[-1], s[0]) and torch.equal(q[-1].float(), q[0].float()) and bool((scale == scale[0]).all())
    assert torch.equal(q[m // 2].float(), q[0].float())
    want = oracle.norm_quant(oracle.values(a[:1]), oracle.values(a[:1]), None, 1e-6)
    assert torch.equal(q[-1:].cpu().double(), want[1])
