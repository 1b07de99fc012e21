"""The selective scan's bf16 results against the 64-bit recurrence term by term: the products' operands that are not
inputs (decayed scores, the carried state and its gradient) are taken in two bf16 parts.

Tolerances: those of test_gpu_selective.py and test_gpu_selective_bwd.py with the bf16 terms' budget cut to what two
parts leave of a value: each part is off by at most 2^-8 of what it rounds, so two by 2^-16.  A term of y, dx, dB or dC
carries one such operand."""
import pytest
import torch

from oracle import selective as ref

from test_gpu_selective import U, inputs
from test_gpu_selective_bwd import grads_of, magnitudes

pytestmark = pytest.mark.gpu
TERM = 2.0 ** -16
SHAPES = [(2, 16, 2, 64, 1, 64), (2, 40, 4, 16, 2, 16), (1, 64, 2, 64, 1, 128), (1, 70, 2, 33, 1, 20), (1, 48, 2, 128, 1, 256),
          (1, 100, 2, 40, 1, 130)]


def near(got, want, m, budget, what):
    h = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    bad = err > h * want.abs() + budget * m.view(want.shape)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((err - h * want.abs()) / m.view(want.shape).clamp_min(1e-30)).max()), budget)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(device, shape, dtype):
    from verace_amd import selective_scan
    d, state = inputs(device, *shape, dtype, seed=60)
    T, N = shape[1], shape[5]
    for s0 in (None, state):
        y, _ = selective_scan(**d, initial_state=s0)
        y64, _ = ref.selective_scan(**d, initial_state=s0)
        m, _ = ref.selective_scan(**d, initial_state=s0, magnitude=True)
        near(y, y64, m, (8 * T + N + 16) * U + (TERM if dtype == torch.bfloat16 else 0.0), "y")


def backward(d, state, dy, dS, lengths=None):
    """All gradients within the budget; returns them."""
    from verace_amd import selective_scan
    own = {k: t.clone().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    got = torch.autograd.grad(selective_scan(**own, lengths=lengths), list(own.values()), (dy, dS))
    r = {k: t.double().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    want = torch.autograd.grad(ref.selective_scan(**r, lengths=lengths), list(r.values()), (dy.double(), dS.double()))
    m = magnitudes(d, state, dy, dS, lengths, True)
    T, P, N = d["x"].shape[1], d["x"].shape[3], d["B"].shape[-1]
    for k, g, w in zip(own, got, want):
        assert g.dtype == own[k].dtype and g.shape == own[k].shape, k
        term = TERM if k in ("x", "B", "C") and g.dtype == torch.bfloat16 else 0.0
        near(g, w, m[k], (8 * T + N + P + 64) * U + term, k)
    return dict(zip(own, got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(device, shape, dtype):
    d, state = inputs(device, *shape, dtype, seed=61)
    backward(d, state, *grads_of(device, d, state, 62))
