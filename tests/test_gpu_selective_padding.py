"""What lies behind a sequence's length is exactly zero, in outputs and in gradients, whatever the tokens that count
and the state before them hold."""
import pytest
import torch

from test_gpu_selective import DTYPES, inputs
from test_gpu_selective_bwd import grads_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("at", ["x", "delta", "B", "C", "state"])
def test_scan(device, dtype, bad, at):
    """A length in the first chunk, inside a later one, one short of the whole and of one token; sequences of a few
    tokens (token by token) and of chunks."""
    from verace_amd import selective_scan
    for T, lens in ((9, [1, 5, 8, 0]), (150, [5, 70, 149, 1])):
        d, state = inputs(device, 4, T, 2, 40, 1, 24, dtype, seed=70)
        dy, dS = grads_of(device, d, state, 71)
        n = torch.tensor(lens, device=device)
        if at == "state":
            state[:, :, 3, 5] = bad
        else:
            for i, m in enumerate(lens):
                if m:
                    d[at][i, m - 1].view(-1)[0] = bad
        leaf = {k: t.clone().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
        y, S = selective_scan(**leaf, lengths=n)
        got = dict(zip(leaf, torch.autograd.grad((y, S), list(leaf.values()), (dy, dS))))
        for i, m in enumerate(lens):
            for name, t in (("y", y.detach()), *((k, got[k]) for k in ("x", "delta", "B", "C"))):
                assert bool((t[i, m:] == 0).all()), (name, T, m)
