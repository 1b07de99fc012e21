"""Decays that leave nothing of a state: rates up to the type's lowest value and below it, infinite step sizes.  The
chunked scan gives what the recurrence gives, token by token or not.

Tolerances: those of test_gpu_selective_terms.py and test_gpu_selective_bwd.py.  Nothing is carried here, so single tokens'
outputs can be as small as their smallest factor: below 2^-14 fp16 has steps of 2^-24, and its rounding is off by up to
2^-25 whatever the value (test_gpu_selective.py's sums over many tokens do not come there)."""
import pytest
import torch

from oracle import selective as ref

from test_gpu_selective import DTYPES, U, inputs
from test_gpu_selective_bwd import grads_of, magnitudes

pytestmark = pytest.mark.gpu
RATES = [-1e30, -3.4e38, -float("inf"), -2.0]


def check(got, d, state):
    (y, S), (T, N, dtype) = got, (d["x"].shape[1], d["B"].shape[-1], d["x"].dtype)
    y64, S64 = ref.selective_scan(**d, initial_state=state)
    ym, Sm = ref.selective_scan(**d, initial_state=state, magnitude=True)
    inner = (8 * T + N + 16) * U + (2.0 ** -16 if dtype == torch.bfloat16 else 0.0)
    step = torch.finfo(dtype).eps / 2 * y64.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert bool(((y.double() - y64).abs() <= step + inner * ym).all())
    assert bool(((S.double() - S64).abs() <= (8 * T + 16) * U * Sm).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [4, 100, 700])
def test_forward(device, T, dtype):
    from verace_amd import selective_scan
    d, state = inputs(device, 2, T, 4, 32, 1, 32, dtype, seed=110, delta_dtype=torch.float32)
    d["A"] = torch.tensor(RATES, device=device)
    got = selective_scan(**d, initial_state=state)
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isfinite(got[1]).all())
    check(got, d, state)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(device, dtype):
    """Finite rates: what crosses such a token has no gradient."""
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 200, 4, 32, 1, 32, dtype, seed=111, delta_dtype=torch.float32)
    d["A"] = torch.tensor([-1e30, -3.4e38, -1e5, -2.0], device=device)
    dy, dS = grads_of(device, d, state, 112)
    leaf = {k: t.clone().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    got = torch.autograd.grad(selective_scan(**leaf), list(leaf.values()), (dy, dS))
    r = {k: t.double().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    want = torch.autograd.grad(ref.selective_scan(**r), list(r.values()), (dy.double(), dS.double()))
    m = magnitudes(d, state, dy, dS, None, True)
    T, P, N = d["x"].shape[1], d["x"].shape[3], d["B"].shape[-1]
    for k, g, w in zip(leaf, got, want):
        inner = (8 * T + N + P + 64) * U + (2.0 ** -16 if k in ("x", "B", "C") and dtype == torch.bfloat16 else 0.0)
        step = torch.finfo(g.dtype).eps / 2 * w.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 0.0)
        assert bool(((g.double() - w).abs() <= step + inner * m[k].view(w.shape)).all()), k  # (false for a NaN)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinite_step(device, dtype):
    """Its head's outputs and states are not finite from there on, as in the recurrence; nothing else changes."""
    from verace_amd import selective_scan
    d, state = inputs(device, 1, 100, 2, 32, 1, 32, dtype, seed=113, delta_dtype=torch.float32)
    d["delta"][0, 40, 1] = float("inf")
    y, S = selective_scan(**d, initial_state=state)
    y64, S64 = ref.selective_scan(**d, initial_state=state)
    assert torch.equal(torch.isfinite(y), torch.isfinite(y64))
    assert torch.equal(torch.isfinite(S), torch.isfinite(S64))
