"""The selective scan's backward where a workgroup walks several heads of a group with dB and dC in accumulators: with and
without partial sums of head blocks, a last block shorter than the others, heads of more than one block of rows (so that
a workgroup's units mix heads and row blocks), 32- and 64-token chunks, ragged lengths.

All gradients against the 64-bit recurrence, within the budget of test_gpu_selective_terms.py."""
import pytest
import torch

from test_gpu_selective import inputs
from test_gpu_selective_bwd import grads_of
from test_gpu_selective_terms import backward

pytestmark = pytest.mark.gpu
# B, T, H, P, G, N, then for chunks of 64 and of 32 tokens: heads a workgroup walks, blocks of heads
SHAPES = [((16, 320, 7, 80, 1, 16), (2, 4), (4, 2)), ((32, 520, 4, 80, 1, 16), (4, 1), (4, 1)),
          ((8, 330, 10, 16, 2, 64), (2, 3), (3, 2)), ((16, 160, 6, 33, 1, 130), None, (2, 3)),
          ((4, 700, 24, 64, 1, 128), (4, 6), (8, 3))]


def blocks(B, T, H, G, L):
    """Heads of a workgroup and blocks of heads of a group: as many blocks as make 256 workgroups."""
    hg, n = H // G, B * -(-T // L) * G
    per = -(-hg // min(hg, -(-256 // n)))
    return per, -(-hg // per)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_backward(device, case, ragged, dtype):
    shape, in64, in32 = SHAPES[case]
    B, T, H, P, G, N = shape
    L = 64 if dtype == torch.bfloat16 and N <= 128 else 32
    assert blocks(B, T, H, G, L) == (in64 if L == 64 else in32)
    d, state = inputs(device, *shape, dtype, seed=100)
    dy, dS = grads_of(device, d, state, 101)
    n = None
    if ragged:
        n = torch.randint(0, T + 1, (B,), generator=torch.Generator(device).manual_seed(102), device=device)
        n[0], n[-1] = 0, T
        for i, m in enumerate(n.tolist()):
            dy[i, m:] = 0  # where the reference's dy meets its own zeros
    got = backward(d, state, dy, dS, n)
    if ragged:
        for k in ("x", "delta", "B", "C"):
            for i, m in enumerate(n.tolist()):
                assert not bool(got[k][i, m:].any()), k
