"""GPU parity of the short causal convolution (csrc/short_conv.hip) with the 64-bit formula: prompts,
gradients, single tokens.

Tolerances, u = 2^-24, h the result's half step: z is K + 1 fused steps, (K + 1) u of the terms' magnitude
m; silu's slope is at most 1.1 and its own evaluation a few u of |z| <= m: 16 u m, then one rounding, h.
The gradient of x sums K such products of dz (each a few u, the slope's error included): 32 u of their
magnitude; those of the weights sum B T terms in runs of 32, of 8 and of parts: (64 + parts) u."""
import pytest
import torch

from oracle import selective as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def _inputs(device, B, T, C, K, dtype, seed=0):
    g = torch.Generator(device).manual_seed(seed + B * 7 + T * 31 + C)

    def r(*s):
        return torch.randn(*s, generator=g, device=device).to(dtype)
    return r(B, T, C), r(C, K), r(C), r(B, K - 1, C)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (2, 2, 3), (3, 17, 64), (1, 40, 130), (2, 100, 2304), (2, 33, 8)])
def test_forward(device, B, T, C, K, dtype):
    from verace_amd import short_conv
    x, w, b, st = _inputs(device, B, T, C, K, dtype)
    h = torch.finfo(dtype).eps / 2
    for kw in ({}, dict(initial_state=st), dict(initial_state=st, activation=None)):
        y, last = short_conv(x, w, b, **kw)
        y64, last64 = ref.short_conv(x, w, b, **kw)
        m = ref.short_conv(x, w, b, initial_state=kw.get("initial_state"), magnitude=True)
        assert y.dtype == last.dtype == dtype
        assert bool(((y.double() - y64).abs() <= h * y64.abs() + 16 * U * m).all())
        assert torch.equal(last.double(), last64)
    y, _ = short_conv(x, w, None)
    assert bool(((y.double() - ref.short_conv(x, w)[0]).abs() <= h * y.double().abs() * 1.01 + 16 * U * m).all())


@pytest.mark.parametrize("int_dtype", [torch.int32, torch.int64])
def test_lengths(device, int_dtype):
    """Rows behind a length are not read (NaN there), give zeros and are not part of the state; lengths
    outside the range are clamped."""
    from verace_amd import short_conv
    x, w, b, st = _inputs(device, 6, 20, 24, 4, torch.float32, seed=2)
    n = torch.tensor([0, 1, 2, 20, -3, 99], device=device, dtype=int_dtype)
    y64, last64 = ref.short_conv(x, w, b, st, n)
    for i, k in enumerate([0, 1, 2, 20, 0, 20]):
        x[i, k:] = float("nan")
    y, last = short_conv(x, w, b, st, n)
    assert torch.allclose(y.double(), y64, rtol=1e-5, atol=1e-5) and torch.equal(last.double(), last64)
    assert torch.equal(last[0], st[0]) and float(y[0].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,K", [(1, 1, 1, 4), (2, 2, 3, 3), (3, 30, 64, 4), (1, 300, 40, 2), (2, 600, 136, 4), (2, 65, 2304, 4)])
@pytest.mark.parametrize("ragged", [False, True])
def test_backward(device, B, T, C, K, dtype, ragged):
    from verace_amd import short_conv
    x, w, b, st = _inputs(device, B, T, C, K, dtype, seed=3)
    dy, _, _, dst = _inputs(device, B, T, C, K, dtype, seed=4)
    n = torch.tensor([(T * (i + 1)) // (B + 1) for i in range(B)], device=device) if ragged else None
    own = [t.clone().requires_grad_() for t in (x, w, b, st)]
    y, last = short_conv(own[0], own[1], own[2], own[3], n)
    got = torch.autograd.grad((y, last), own, (dy, dst))
    r = [t.double().requires_grad_() for t in (x, w, b, st)]
    want = torch.autograd.grad(ref.short_conv(r[0], r[1], r[2], r[3], n), r, (dy.double(), dst.double()))
    h = torch.finfo(dtype).eps / 2
    big = float(dy.double().abs().max()) * 1.1
    rows = torch.cat([st, x], 1).double().abs().max()
    m = float(ref.short_conv(x, w, b, st, magnitude=True).max())   # the slope's error scales with z's
    mags = [big * float(w.double().abs().sum(1).max()) * (1 + m) + float(dst.double().abs().max())] * 4
    mags[1], mags[2] = big * float(rows) * (1 + m) * B * T, big * (1 + m) * B * T
    for i, (g, q) in enumerate(zip(got, want)):
        assert g.dtype == dtype
        budget = 32 * U if i in (0, 3) else (64 + B * T / 256) * U
        err = (g.double() - q).abs()
        assert bool((err <= h * q.abs() + budget * mags[i]).all()), (i, float(err.max()), budget * mags[i])
    if ragged:
        for i in range(B):
            assert float(got[0][i, int(n[i]):].abs().sum()) == 0.0


def test_gradient_against_differences(device):
    from verace_amd import short_conv
    leaves = [t.requires_grad_() for t in _inputs(device, 2, 9, 5, 4, torch.float32, seed=5)]
    dy, _, _, dst = _inputs(device, 2, 9, 5, 4, torch.float32, seed=6)
    n = torch.tensor([9, 4], device=device)
    got = torch.autograd.grad(short_conv(*leaves, n), leaves, (dy, dst))
    for i, (t, g) in enumerate(zip(leaves, got)):
        v = torch.randn_like(t)

        def f(e):
            u = [q.detach().double() for q in leaves]
            u[i] = u[i] + e * v.double()
            y, last = ref.short_conv(*u, n)
            return float((y * dy).sum() + (last * dst).sum())
        num = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(float((g * v).double().sum()) - num) <= 1e-4 * float((g * v).abs().sum()) + 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C,K", [(1, 1, 2), (3, 24, 3), (64, 2304, 4), (5, 130, 4)])
def test_steps_are_the_prompt(device, B, C, K, dtype):
    """Token by token from the state of a prompt's first part: the bits of the whole prompt."""
    from verace_amd import short_conv, short_conv_step_
    x, w, b, st = _inputs(device, B, 9, C, K, dtype, seed=7)
    y, last = short_conv(x, w, b, st)
    _, s = short_conv(x[:, :4], w, b, st)
    for t in range(4, 9):
        out = short_conv_step_(x[:, t:t + 1] if t % 2 else x[:, t], w, b, s)
        assert torch.equal(out, y[:, t:t + 1])
    assert torch.equal(s, last)


def test_step_mask(device):
    from verace_amd import short_conv_step_
    x, w, b, st = _inputs(device, 4, 1, 40, 4, torch.bfloat16, seed=8)
    mask = torch.tensor([True, False, True, False], device=device)
    x[1] = float("nan")
    s = st.clone()
    y = short_conv_step_(x, w, b, s, active_mask=mask)
    assert torch.equal(s[1], st[1]) and torch.equal(s[3], st[3]) and float(y[1].abs().sum()) == 0.0
    assert torch.equal(s[0, :2], st[0, 1:]) and torch.equal(s[0, 2], x[0, 0]) and bool(torch.isfinite(y).all())


def test_strided_rows_and_parameters(device):
    """Slices of a wider projection at aligned and odd columns, an expanded item, fp32 parameters."""
    from verace_amd import short_conv
    wide = torch.randn(3, 12, 100, device=device).to(torch.bfloat16)
    w, b = torch.randn(40, 4, device=device), torch.randn(40, device=device)
    for x in (wide[..., 8:48], wide[..., 5:45], wide[:1, :, 16:56].expand(3, 12, 40), wide.transpose(0, 1)[..., :40]):
        got, last = short_conv(x, w, b)
        want, last64 = ref.short_conv(x, w, b)
        m = ref.short_conv(x, w, b, magnitude=True)
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 16 * U * m).all())
        assert torch.equal(last.double(), last64)


def test_no_tokens(device):
    from verace_amd import short_conv
    x, w, b, st = _inputs(device, 2, 0, 16, 4, torch.float32)
    y, last = short_conv(x, w, b, st)
    assert y.shape == (2, 0, 16) and torch.equal(last, st)
    w.requires_grad_(), st.requires_grad_()
    y, last = short_conv(x, w, b, st)
    dw, ds = torch.autograd.grad((y, last), (w, st), (torch.zeros_like(y), torch.ones_like(last)))
    assert float(dw.abs().sum()) == 0.0 and torch.equal(ds, torch.ones_like(ds))
