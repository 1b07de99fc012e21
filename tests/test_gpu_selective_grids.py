"""More workgroups than a grid dimension's 32-bit count of threads: every row is still done."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,d", [(70_000_000, 8), (17_000_000, 1032)])
def test_norm(device, rows, d):
    """Rows are independent: those on either side of the 2^32nd thread and the last ones have the bits of a call on them
    alone."""
    from verace_amd import gated_norm_add
    print("[case] norm of", rows, "rows of", d, flush=True)
    y = torch.empty(rows, d, device=device, dtype=torch.bfloat16).normal_()
    w = torch.randn(d, device=device).bfloat16()
    s, _ = gated_norm_add(y, y, w)
    per = 4 if d == 8 else 1
    first = 2 ** 32 // 256 * per
    assert rows > first
    for r0 in (0, first - 100, rows - 200):
        part = y[r0:r0 + 200]
        assert torch.equal(s[r0:r0 + 200], gated_norm_add(part, part, w)[0]), r0


def test_scan(device):
    """Heads of one row each, in more chunks than the chunk form's first launch has workgroups for, go token by token."""
    from verace_amd import selective_scan
    B, H, T = 1 << 15, 1 << 7, 1100
    print("[case] scan of", B * H * T, "tokens and heads", flush=True)
    x = torch.empty(B, T, H, 1, device=device, dtype=torch.bfloat16).normal_()
    delta = torch.zeros(1, 1, H, device=device, dtype=torch.bfloat16).expand(B, T, H)
    one = torch.ones(1, 1, 1, 1, device=device, dtype=torch.bfloat16)
    A = torch.full((H,), -1.0, device=device)
    y, S = selective_scan(x, delta, A, one.expand(B, T, 1, 1), one.expand(B, T, 1, 1))
    for b in (0, 12345, B - 1):
        s = slice(b, b + 1)
        ys, Ss = selective_scan(x[s], delta[s], A, one.expand(1, T, 1, 1), one.expand(1, T, 1, 1))
        # decays of e^-0.69 a token: sums of about two terms of up to 5; each form rounds y once
        assert bool(((y[s].float() - ys.float()).abs() <= 2.0 ** -7 * ys.float().abs() + 1e-3).all())
        assert bool(((S[s] - Ss).abs() <= 1e-3).all())
