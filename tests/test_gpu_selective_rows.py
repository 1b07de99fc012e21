"""A head's rows are independent: a NaN or an infinity in one row of x, dy, the state or its gradient leaves the other rows'
y, states and their gradients as they are (dB, dC and the step sizes' gradients are sums over the rows)."""
import pytest
import torch

from test_gpu_selective import DTYPES, inputs
from test_gpu_selective_bwd import grads_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [16, 64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", ["x", "dy", "state", "d_state"])
def test_rows(device, at, bad, N, dtype):
    from verace_amd import launch_selective_hip_scan_bwd, selective_scan
    T, P, row = 150, 40, 6
    d, state = inputs(device, 1, T, 2, P, 1, N, dtype, seed=120)
    dy, dS = grads_of(device, d, state, 121)

    def run(d, state, dy, dS):
        y, S = selective_scan(**d, initial_state=state)
        g = launch_selective_hip_scan_bwd(**d, dy=dy, initial_state=state, d_state=dS)
        return y, S, g[0], g[7]
    want = run(d, state, dy, dS)
    c = {k: v.clone() for k, v in (*d.items(), ("state", state), ("dy", dy), ("d_state", dS))}
    if at in ("x", "dy"):
        c[at][0, 70, 1, row] = bad
    else:
        c[at][0, 1, row, N // 2] = bad
    got = run({k: c[k] for k in d}, c["state"], c["dy"], c["d_state"])
    keep = [p for p in range(P) if p != row]
    h = torch.finfo(dtype).eps
    for name, g, w, dim in zip(("y", "state", "dx", "dstate"), got, want, (3, 2, 3, 2)):
        g, w = g.index_select(dim, torch.tensor(keep, device=device)), w.index_select(dim, torch.tensor(keep, device=device))
        assert bool(torch.isfinite(g).all()), name
        if name == "y":  # the chunk of such a token is summed in another order, then rounded
            assert bool(((g.float() - w.float()).abs() <= 2 * h * w.float().abs() + 1e-3).all())
        else:
            assert torch.equal(g, w), name
