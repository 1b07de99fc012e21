"""GPU parity of the gated norms (csrc/gated_norm.hip) with the 64-bit formula, forward and backward.

Tolerances, u = 2^-24 and h the result's half step (finfo.eps / 2).  A mean of d squares carries at most
about 16 + d / 64 roundings a lane and the tree, a norm half of that relatively, sigmoid and the products
a few u: every fp32 intermediate is within (48 + d / 16) u of its row's scale, and each result is rounded
once, h relative.  The backward subtracts two such rows.  Sums over rows add (rows / 8 + 16) u of their
terms' magnitude."""
import pytest
import torch

from oracle import selective as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(device, rows, d, dtype, w_dtype=None, seed=0):
    g = torch.Generator(device).manual_seed(seed + rows * 131 + d)
    y, res, gate = (torch.randn(rows, d, generator=g, device=device).to(dtype) for _ in range(3))
    w1, sc, w2 = ((1 + 0.2 * torch.randn(d, generator=g, device=device)).to(w_dtype or dtype) for _ in range(3))
    return y, res, gate, w1, sc, w2


def _close(got, want, h, d, extra=0.0):
    """Within h of each value, and within the fp32 budget of the row's largest."""
    budget = (48 + d / 16 + extra) * 2.0 ** -24
    err, scale = (got.double() - want).abs(), want.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    bad = err > h * want.abs() + budget * scale
    assert not bool(bad.any()), (float((err / scale).max()), int(bad.sum()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 64), (64, 1024), (33, 1000), (7, 1023), (9, 2048), (2, 4096)])
def test_forward(device, rows, d, dtype):
    from verace_amd import gated_norm_add
    a = _inputs(device, rows, d, dtype)
    y, res, gate, w1, sc, w2 = a
    s, n = gated_norm_add(y, res, w1, gate, sc, w2)
    s64, n64 = ref.gated_norm_add(y, res, w1, gate, sc, w2)
    h = torch.finfo(dtype).eps / 2
    _close(s, s64, h, d)
    _close(n, n64, h, d)


@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.float32), (torch.float32, None), (torch.float16, None)])
@pytest.mark.parametrize("parts", ["y", "gate", "scale", "norm", "next", "sigmoid"])
def test_parts(device, dtype, w_dtype, parts):
    """Each term left out, and the other activation."""
    from verace_amd import gated_norm_add
    y, res, gate, w1, sc, w2 = _inputs(device, 17, 130, dtype, w_dtype)
    kw = {"y": {}, "gate": dict(gate=gate), "scale": dict(scale=sc), "norm": dict(norm_weight=w1, eps=0.5),
          "next": dict(next_weight=w2, next_eps=1e-3), "sigmoid": dict(gate=gate, activation="sigmoid", next_weight=w2)}[parts]
    s, n = gated_norm_add(y, res, **kw)
    s64, n64 = ref.gated_norm_add(y, res, **kw)
    h = torch.finfo(dtype).eps / 2
    _close(s, s64, h, 130)
    assert (n is None) == (n64 is None)
    if n is not None:
        _close(n, n64, h, 130)


@pytest.mark.parametrize("dtype,w_dtype", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32),
                                           (torch.float16, None)])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (130, 64), (600, 1024), (33, 1000), (9, 2048), (2, 4096)])
def test_backward(device, rows, d, dtype, w_dtype):
    from verace_amd import gated_norm_add
    a = _inputs(device, rows, d, dtype, w_dtype, seed=1)
    ds, dn = _inputs(device, rows, d, dtype, seed=2)[:2]
    own = [t.clone().requires_grad_() for t in a]
    y, res, gate, w1, sc, w2 = own
    grads = torch.autograd.grad(gated_norm_add(y, res, w1, gate, sc, w2), own, (ds, dn))
    r = [t.double().requires_grad_() for t in a]
    y, res, gate, w1, sc, w2 = r
    want = torch.autograd.grad(ref.gated_norm_add(y, res, w1, gate, sc, w2), r, (ds.double(), dn.double()))
    for i, (g, w, t) in enumerate(zip(grads, want, a)):
        assert g.dtype == t.dtype and g.shape == t.shape
        h = torch.finfo(g.dtype).eps / 2
        if i < 3:
            # the projections subtract rows of the gradient's size from its parts: twice the budget, and the
            # part left can be small against them (all of it at d = 1)
            scale = max(1.0, float(ds.abs().max() + dn.abs().max())) * 8
            err = (g.double() - w).abs()
            assert bool((err <= h * w.abs() + 2 * (48 + d / 16) * 2.0 ** -24 * scale * (1 + float(
                a[0].double().abs().amax(-1).clamp_min(1e-2).reciprocal().max()))).all()), (i, float(err.max()))
        else:
            m = (rows / 8 + 16 + 48 + d / 16) * 2.0 ** -24 * rows ** 0.5 * 64
            err = (g.double() - w).abs()
            assert bool((err <= h * w.abs() + m).all()), (i, float(err.max()))


def test_gradient_against_differences(device):
    from verace_amd import gated_norm_add
    y, res, gate, w1, sc, w2 = (t.requires_grad_() for t in _inputs(device, 6, 24, torch.float32, seed=5))
    ds, dn = _inputs(device, 6, 24, torch.float32, seed=6)[:2]
    leaves = [y, res, gate, w1, sc, w2]
    grads = torch.autograd.grad(gated_norm_add(y, res, w1, gate, sc, w2), leaves, (ds, dn))
    for i, (t, g) in enumerate(zip(leaves, grads)):
        v = torch.randn_like(t)
        def f(e):
            u = [x.detach().double() for x in leaves]
            u[i] = u[i] + e * v.double()
            s, n = ref.gated_norm_add(u[0], u[1], u[3], u[2], u[4], u[5])
            return float((s * ds).sum() + (n * dn).sum())
        num = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(float((g * v).double().sum()) - num) <= 1e-4 * float((g * v).abs().sum())


def test_strides_broadcast_and_shapes(device):
    """Rows that are slices of a wider tensor, a gate shared by a sequence's tokens, three dimensions, and a
    misaligned start."""
    from verace_amd import gated_norm_add
    g = torch.Generator(device).manual_seed(3)
    wide = torch.randn(2, 5, 200, generator=g, device=device)
    w1 = torch.randn(64, generator=g, device=device)
    gate1 = torch.randn(2, 1, 64, generator=g, device=device, requires_grad=True)
    for off in (0, 3, 8):
        y, res = wide[..., off:off + 64], wide[..., 100:164]
        s, n = gated_norm_add(y, res, w1, gate1, None, w1)
        s64, n64 = ref.gated_norm_add(y, res, w1, gate1.expand(2, 5, 64), None, w1)
        _close(s.detach(), s64.detach(), 2.0 ** -24, 64)
        _close(n.detach(), n64.detach(), 2.0 ** -24, 64)
    dg, = torch.autograd.grad(s.sum(), gate1)
    dg64, = torch.autograd.grad(s64.sum(), gate1)
    assert torch.allclose(dg, dg64, rtol=1e-5, atol=1e-5)


def test_only_one_output_used(device):
    from verace_amd import gated_norm_add
    a = [t.requires_grad_() for t in _inputs(device, 10, 96, torch.float32, seed=7)]
    y, res, gate, w1, sc, w2 = a
    r = [t.detach().double().requires_grad_() for t in a]
    for k in (0, 1):
        got = torch.autograd.grad(gated_norm_add(y, res, w1, gate, sc, w2)[k].sum(), a, allow_unused=True)
        want = torch.autograd.grad(ref.gated_norm_add(r[0], r[1], r[3], r[2], r[4], r[5])[k].sum(), r, allow_unused=True)
        for g, w in zip(got, want):
            if w is None:  # not part of s
                assert g is None or float(g.abs().max()) == 0.0
            else:
                assert torch.allclose(g.double(), w, rtol=2e-5, atol=2e-5)


def test_rows_are_independent(device):
    """A row of NaN, of infinities and of zeros changes no other row; no rows at all."""
    from verace_amd import gated_norm_add
    y, res, gate, w1, sc, w2 = _inputs(device, 9, 256, torch.bfloat16, seed=8)
    s0, n0 = gated_norm_add(y, res, w1, gate, sc, w2)
    y[2], y[4], y[6] = float("nan"), float("inf"), 0.0
    s, n = gated_norm_add(y, res, w1, gate, sc, w2)
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(s[keep], s0[keep]) and torch.equal(n[keep], n0[keep])
    assert torch.isnan(s[2]).all() and torch.equal(s[6], res[6])
    s, n = gated_norm_add(y[:0], res[:0], w1, gate[:0], sc, w2)
    assert s.shape == n.shape == (0, 256)
    w1.requires_grad_()
    s, n = gated_norm_add(y[:0], res[:0], w1, gate[:0], sc, w2)
    assert float(torch.autograd.grad(n.sum(), w1)[0].abs().sum()) == 0.0


def test_repeats_and_other_stream(device):
    """The same bits in every run, and on a side stream."""
    from verace_amd import gated_norm_add
    a = [t.requires_grad_() for t in _inputs(device, 3000, 520, torch.bfloat16, seed=9)]
    y, res, gate, w1, sc, w2 = a

    def run():
        s, n = gated_norm_add(y, res, w1, gate, sc, w2)
        return [s.detach(), n.detach(), *torch.autograd.grad((s, n), a, (s.detach(), n.detach()))]
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, again):
        assert torch.equal(p, q)
