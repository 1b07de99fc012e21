"""The gated projections and the projection with its epilogue against their definitions in 64 bits, forward and backward, at the
sizes where a tile, a row or a contraction ends."""
import pytest
import torch

from oracle import feed_forward as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# (rows, contraction, columns): one of each, less than a piece, not whole pieces, one more than a tile, several tiles
SIZES = [(1, 1, 1), (1, 64, 8), (3, 40, 24), (17, 100, 37), (64, 256, 96), (65, 72, 130), (129, 65, 257), (257, 200, 131),
         (300, 1024, 64)]


def va():
    import verace_amd
    return verace_amd


def randn(g, *shape, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).cuda()


def within(got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    off = (got - want).abs()
    ok = off <= bound
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, the worst {float((off / bound)[~ok].max()):.3g} times its bound"


def make(g, m, k, n, dtype, weights):
    """x and weights; 8-bit ones as (rows, scales)."""
    x = randn(g, m, k)
    ws = [randn(g, n, k, scale=max(k, 1) ** -0.5) for _ in range(weights)]
    if dtype != oracle.E4M3:
        return [(t.to(dtype), None) for t in (x, *ws)]
    return [va().quantize_rows(t) for t in (x, *ws)]


@pytest.mark.parametrize("activation", ["situ", "silu"])
@pytest.mark.parametrize("dtype", DTYPES + [oracle.E4M3])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_gated(m, k, f, dtype, activation):
    g = torch.Generator().manual_seed(m + k + f)
    (x, xs), (wg, gs), (wu, us) = make(g, m, k, f, dtype, 2)
    out = torch.bfloat16 if dtype == oracle.E4M3 else dtype
    h = va().gated_linear(x, wg, wu, xs, gs, us, activation=activation, beta1=2.0, beta2=3.0)
    assert h.dtype == out
    within(h, *oracle.gated(oracle.values(x, xs), oracle.values(wg, gs), oracle.values(wu, us), activation, out, 2.0, 3.0))


@pytest.mark.parametrize("activation,bias,residual", [(None, False, False), (None, False, True), ("silu", True, True), ("gelu", True, False)])
@pytest.mark.parametrize("dtype", DTYPES + [oracle.E4M3])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(m, k, n, dtype, activation, bias, residual):
    g = torch.Generator().manual_seed(m + k + n)
    (x, xs), (w, ws) = make(g, m, k, n, dtype, 1)
    out = torch.bfloat16 if dtype == oracle.E4M3 else dtype
    b = randn(g, n).to(out) if bias else None
    r = randn(g, m, n).to(out) if residual else None
    y = va().linear_add(x, w, b, r, xs, ws, activation=activation)
    assert y.dtype == out
    within(y, *oracle.linear(oracle.values(x, xs), oracle.values(w, ws), None if b is None else oracle.values(b),
                             None if r is None else oracle.values(r), activation, out))


@pytest.mark.parametrize("out", DTYPES)
def test_8_bit_result_types(out):
    g = torch.Generator().manual_seed(5)
    (x, xs), (wg, gs), (wu, us) = make(g, 70, 144, 90, oracle.E4M3, 2)
    b, r = randn(g, 90).to(out), randn(g, 70, 90).to(out)
    X, G, U = oracle.values(x, xs), oracle.values(wg, gs), oracle.values(wu, us)
    h = va().gated_linear(x, wg, wu, xs, gs, us, out_dtype=out)
    y = va().linear_add(x, wg, b, r, xs, gs, activation="silu", out_dtype=out)
    assert h.dtype == out and y.dtype == out
    within(h, *oracle.gated(X, G, U, "situ", out))
    within(y, *oracle.linear(X, G, oracle.values(b), oracle.values(r), "silu", out))


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("activation", ["situ", "silu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,f", SIZES + [(1500, 136, 72)])
def test_gated_backward(m, k, f, dtype, activation, kept, monkeypatch):
    monkeypatch.setattr("verace_amd.feed_forward._keeps", lambda *_: kept)
    g = torch.Generator().manual_seed(m + k + f)
    x, wg, wu = (t.requires_grad_() for t, _ in make(g, m, k, f, dtype, 2))
    dh = randn(g, m, f).to(dtype)
    grads = torch.autograd.grad(va().gated_linear(x, wg, wu, activation=activation), (x, wg, wu), dh)
    want = oracle.gated_bwd(*(oracle.values(t) for t in (x, wg, wu)), activation, oracle.values(dh), dtype)
    for got, w, t in zip(grads, want, (x, wg, wu)):
        assert got.dtype == dtype and got.shape == t.shape
        within(got, *w)


@pytest.mark.parametrize("activation,bias,kept", [(None, False, True), (None, True, True), ("silu", True, True), ("silu", True, False),
                                                  ("gelu", False, True), ("gelu", False, False)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES + [(1500, 136, 72)])
def test_linear_backward(m, k, n, dtype, activation, bias, kept, monkeypatch):
    monkeypatch.setattr("verace_amd.feed_forward._keeps", lambda *_: kept)
    g = torch.Generator().manual_seed(m + k + n)
    x, w = (t.requires_grad_() for t, _ in make(g, m, k, n, dtype, 1))
    b = randn(g, n).to(dtype).requires_grad_() if bias else None
    r = randn(g, m, n).to(dtype).requires_grad_()
    dy = randn(g, m, n).to(dtype)
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = torch.autograd.grad(va().linear_add(x, w, b, r, activation=activation), leaves, dy)
    want = oracle.linear_bwd(oracle.values(x), oracle.values(w), None if b is None else oracle.values(b), activation,
                             oracle.values(dy), dtype)
    if not bias:
        want = want[:2]
    for got, v in zip(grads, want):
        assert got.dtype == dtype
        within(got, *v)
    assert torch.equal(grads[-1], dy)


def test_what_is_kept():
    """Below a length of 1536 a 16-bit forward keeps its inputs alone; from there, and in float32, its sums too."""
    for dtype, k, more in ((torch.bfloat16, 1528, 0), (torch.bfloat16, 1536, 1), (torch.float32, 64, 1)):
        x, w = (torch.zeros(s, k, device="cuda", dtype=dtype, requires_grad=True) for s in (4, 8))
        for y, n, m in ((va().gated_linear(x, w, w), 16, more), (va().linear_add(x, w, activation="silu"), 8, more), (va().linear_add(x, w), 8, 0)):
            saved = [t for t in y.grad_fn.saved_tensors if t is not None and t.shape[1] != k]
            assert [tuple(t.shape) for t in saved] == [(4, n)] * m and all(t.dtype == torch.float32 for t in saved)
    r = torch.zeros(4, 8, device="cuda", requires_grad=True)
    y = va().linear_add(torch.zeros(4, 64, device="cuda"), torch.zeros(8, 64, device="cuda"), None, r, activation="silu")
    assert [t for t in y.grad_fn.saved_tensors if t is not None and t.shape == (4, 8)] == []


# contractions of 32 steps of 128 bytes and more over few tiles, which a tile's waves share: even shares, a last share that ends
# inside a step (33 steps: 9, 9, 9 and 6; 37: 10, 10, 10 and 7), and a last step of one element
LONG = [(130, 32, 0, 1000), (400, 33, -3, 1000), (430, 37, 0, 1040), (450, 34, -31, 1100)]


def long_k(steps, more, dtype):
    each = 128 // torch.empty(0, dtype=dtype).element_size()
    return steps * each + max(more, 1 - each)


@pytest.mark.parametrize("dtype", DTYPES + [oracle.E4M3])
@pytest.mark.parametrize("m,steps,more,n", LONG)
def test_long_contraction(m, steps, more, n, dtype):
    k = long_k(steps, more, dtype)
    g = torch.Generator().manual_seed(m + k + n)
    (x, xs), (w, ws) = make(g, m, k, n, dtype, 1)
    out = torch.bfloat16 if dtype == oracle.E4M3 else dtype
    b, r = randn(g, n).to(out), randn(g, m, n).to(out)
    within(va().linear_add(x, w, b, r, xs, ws, activation="silu"),
           *oracle.linear(oracle.values(x, xs), oracle.values(w, ws), oracle.values(b), oracle.values(r), "silu", out))
    f = n // 2 + 1
    (wg, gs), (wu, us) = make(g, 1, k, f, dtype, 2)[1:]
    within(va().gated_linear(x, wg, wu, xs, gs, us),
           *oracle.gated(oracle.values(x, xs), oracle.values(wg, gs), oracle.values(wu, us), "situ", out))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,steps,more,n", LONG)
def test_long_contraction_backward(m, steps, more, n, dtype):
    """dx contracts over the columns, in one part and (gated) in two."""
    k, n = n, long_k(steps, more, dtype)
    g = torch.Generator().manual_seed(m + k + n)
    x, w = (t.requires_grad_() for t, _ in make(g, m, k, n, dtype, 1))
    dy = randn(g, m, n).to(dtype)
    grads = torch.autograd.grad(va().linear_add(x, w), (x, w), dy)
    for got, v in zip(grads, oracle.linear_bwd(oracle.values(x), oracle.values(w), None, None, oracle.values(dy), dtype)):
        within(got, *v)
    wu = make(g, 1, k, n, dtype, 1)[1][0].requires_grad_()
    grads = torch.autograd.grad(va().gated_linear(x, w, wu), (x, w, wu), dy)
    for got, v in zip(grads, oracle.gated_bwd(*(oracle.values(t) for t in (x, w, wu)), "situ", oracle.values(dy), dtype)):
        within(got, *v)
