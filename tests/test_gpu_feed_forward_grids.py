"""The feed-forward products of results with more tiles, or more fragments of a few rows, than a grid's 2^32 threads hold in the form
that their shape would take otherwise."""
import pytest
import torch

from oracle import feed_forward as oracle
from test_gpu_feed_forward import va, within

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def counted(n):
    """[n, 8] rows of i % 251."""
    t = torch.empty(n, 8, device="cuda", dtype=BF)
    for i in range(0, n, 251 << 18):
        part = t[i:i + (251 << 18)]
        part.copy_((torch.arange(part.shape[0], device="cuda") % 251).to(BF)[:, None].expand(part.shape))
    return t


def test_many_columns_of_one_row():
    """2^27 + 5 columns: more fragments of 16 columns than a grid holds at 512 threads each."""
    n = (1 << 27) + 5
    w, x = counted(n), torch.ones(1, 8, device="cuda", dtype=BF)
    y = va().linear_add(x, w)
    assert torch.equal(y[0], w[:, 0] * 8)
    h = va().gated_linear(x, w, w, activation="silu")
    at = torch.tensor([0, 1, 250, (1 << 27) - 1, 1 << 27, n - 1], device="cuda")
    want, bound = oracle.gated(oracle.values(x), oracle.values(w[at]), oracle.values(w[at]), "silu", BF)
    within(h[:, at], want, bound)
    assert torch.equal(h[0, 251:502], h[0, :251]) and torch.equal(h[0, n - 502:n - 251], h[0, n - 251:])


@pytest.mark.parametrize("activation", ["situ", "silu"])
def test_many_rows_of_one_column(activation):
    """2^30 rows: more tiles of 64 x 64, and of 128 x 128, than a grid holds."""
    m = 1 << 30
    x, w = counted(m), torch.full((1, 8), 2.0 ** -6, device="cuda", dtype=BF)
    y = va().linear_add(x, w)
    assert torch.equal(y[:, 0], x[:, 0] / 8)
    del y
    h = va().gated_linear(x, w, w, activation=activation)
    at = torch.tensor([0, 1, 250, m // 2, m - 2, m - 1], device="cuda")
    within(h[at], *oracle.gated(oracle.values(x[at]), oracle.values(w), oracle.values(w), activation, BF))
    for i in (251, m // 251 * 251 - 251):
        assert torch.equal(h[i:i + 251], h[:251])
