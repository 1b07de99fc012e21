"""The convolution's weight gradients element by element, over many runs and workgroups, and batches of more tokens than a
grid's second dimension has workgroups for.

Tolerance, u = 2^-24, h the result's half step.  A term of dweight[c, j] is dy act'(z) row: the slope is at most 1.1 and is
off by 16 u of 1 + |z| (z's own K + 1 roundings, sigmoid's few), so the term's magnitude is |dy| (1.1 + |z|) |row| and
carries 20 u of it.  A run adds 32 of them one after the other, a workgroup 4 runs, and the second kernel parts / 4 and 4:
(40 + parts / 4) u of the sum of the magnitudes."""
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
    return r(B, T, C), r(C, K), r(C), r(B, K - 1, C), r(B, T, C), r(B, K - 1, C)


def weight_gradients(x, w, b, st, dy, n=None):
    """dweight, dbias in 64 bits and the sums of their terms' magnitudes."""
    K, T = w.shape[1], x.shape[1]
    rows = torch.cat([st, x], 1).double()
    z = sum(rows[:, j:j + T] * w[:, j].double() for j in range(K)) + b.double()
    sg = torch.sigmoid(z)
    dz = dy.double() * sg * (1 + z * (1 - sg))
    m = dy.double().abs() * (1.1 + sum(rows[:, j:j + T].abs() * w[:, j].double().abs() for j in range(K)) + b.double().abs())
    if n is not None:
        on = (torch.arange(T, device=x.device) < n[:, None]).unsqueeze(-1)
        dz, m = (torch.where(on, t, 0.0) for t in (dz, m))
    dw = torch.stack([(dz * rows[:, j:j + T]).sum((0, 1)) for j in range(K)], 1)
    mw = torch.stack([(m * rows[:, j:j + T].abs()).sum((0, 1)) for j in range(K)], 1)
    return (dw, mw), (dz.sum((0, 1)), m.sum((0, 1)))


def check(got, x, w, b, st, dy, n=None):
    parts = x.shape[0] * -(-(x.shape[1] + w.shape[1] - 1) // 128)
    for name, g, (want, m) in zip(("weight", "bias"), got, weight_gradients(x, w, b, st, dy, n)):
        h = torch.finfo(g.dtype).eps / 2
        err = (g.double() - want).abs()
        bound = h * want.abs() + (40 + parts / 4) * U * m
        assert bool((err <= bound).all()), (name, float((err / bound).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,K", [(1, 31, 8, 2), (2, 600, 136, 4), (2, 65, 2304, 4), (3, 130, 5, 3), (5, 1025, 64, 4)])
@pytest.mark.parametrize("ragged", [False, True])
def test_weights(device, B, T, C, K, dtype, ragged):
    from verace_amd import short_conv
    x, w, b, st, dy, dst = _inputs(device, B, T, C, K, dtype, seed=20)
    n = torch.tensor([(T * (i + 1)) // (B + 1) for i in range(B)], device=device) if ragged else None
    leaf = [w.requires_grad_(), b.requires_grad_()]
    got = torch.autograd.grad(short_conv(x, w, b, st, n), leaf, (dy, dst))
    check(got, x, w.detach(), b.detach(), st, dy, n)


def test_differences_over_runs(device):
    """As in test_gpu_short_conv.py, over several runs and workgroups: T = 300."""
    from verace_amd import short_conv
    x, w, b, st, dy, dst = _inputs(device, 2, 300, 5, 4, torch.float32, seed=21)
    leaves = [t.requires_grad_() for t in (x, w, b, st)]
    n = torch.tensor([300, 161], device=device)
    got = torch.autograd.grad(short_conv(*leaves, n), leaves, (dy, dst))
    for i, (t, g) in enumerate(zip(leaves, got)):
        v = torch.randn(t.shape, generator=torch.Generator(device).manual_seed(i), device=device)

        def f(e):
            u = [q.detach().double() for q in leaves]
            u[i] = u[i] + e * v.double()
            y, last = ref.short_conv(*u, n)
            return float((y * dy).sum() + (last * dst).sum())
        num = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(float((g * v).double().sum()) - num) <= 1e-5 * float((g * v).abs().sum()) + 1e-6, i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_short_sequences(device, dtype):
    """33000 sequences of 128 tokens: 66000 parts, against 64 bits, and single items against themselves alone."""
    from verace_amd import short_conv
    x, w, b, st, dy, dst = _inputs(device, 33000, 128, 4, 4, dtype, seed=22)
    leaf = [t.requires_grad_() for t in (x, w, b, st)]
    got = torch.autograd.grad(short_conv(*leaf), leaf, (dy, dst))
    check(got[1:3], x.detach(), w.detach(), b.detach(), st.detach(), dy)
    for i in (0, 16383, 32767, 32999):
        s = slice(i, i + 1)
        one = [x.detach()[s].clone().requires_grad_(), w, b, st.detach()[s].clone().requires_grad_()]
        dx, ds = torch.autograd.grad(short_conv(*one), (one[0], one[3]), (dy[s], dst[s]))
        assert torch.equal(got[0][s], dx) and torch.equal(got[3][s], ds), i
