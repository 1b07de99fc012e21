"""The element-wise layer kernels on more rows than a grid dimension's 32-bit count of threads: rows are independent, so
those on either side of the 2^32nd thread and the last ones have the bits of a call on them alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _spans(rows, first):
    assert rows > first
    return [slice(0, 200), slice(first - 100, first + 100), slice(rows - 200, rows)]


def test_norm_add(device):
    from verace_amd.layer_ops import norm_add
    rows, d = 34_000_000, 8
    print("[case] norm_add", rows, flush=True)
    a, c, b = (torch.empty(rows, d, device=device, dtype=torch.bfloat16).normal_() for _ in range(3))
    norm = torch.nn.RMSNorm(d, device=device, dtype=torch.bfloat16)
    with torch.no_grad():
        s, n = norm_add(a, norm, c, b, norm)
        for k in _spans(rows, 2 ** 32 // 128):
            s1, n1 = norm_add(a[k].contiguous(), norm, c[k].contiguous(), b[k].contiguous(), norm)
            assert torch.equal(s[k], s1) and torch.equal(n[k], n1)


def test_mcmoe_coef(device):
    from verace_amd.layer_ops import mcmoe_coef
    n = 17_000_000
    print("[case] mcmoe_coef", n, flush=True)
    logits = torch.empty(n, 2, device=device, dtype=torch.bfloat16).normal_()
    sig, v = (torch.empty(n, 16, device=device, dtype=torch.bfloat16).normal_() for _ in range(2))
    with torch.no_grad():
        y = mcmoe_coef(logits, sig, v, 1)
        for k in _spans(n, 2 ** 32 // 256):
            assert torch.equal(y[k], mcmoe_coef(logits[k].contiguous(), sig[k].contiguous(), v[k].contiguous(), 1))


def test_halting_update(device):
    from verace_amd.layer_ops import HaltingState
    rows, d = 34_000_000, 8
    print("[case] halting", rows, flush=True)
    linear = torch.nn.Linear(d, 1, device=device, dtype=torch.bfloat16)
    out, h = (torch.empty(rows, d, device=device, dtype=torch.bfloat16).normal_() for _ in range(2))
    active = torch.rand(rows, device=device) < 0.7

    def run(out, h, active):
        n = h.shape[0]
        final, acc, depth = torch.zeros_like(h), torch.full((n,), 0.3, device=device).bfloat16(), torch.zeros(n, device=device).bfloat16()
        state = HaltingState.start(linear, 0.9, h, final, acc, depth)
        assert state is not None and state.accepts(out, h)
        nxt, still = state.step(out, h, active, False)
        state.finish(nxt, still)
        return nxt, still, final, acc, depth
    with torch.no_grad():
        whole = run(out, h, active)
        for k in _spans(rows, 2 ** 32 // 128):
            for p, q in zip(whole, run(out[k].contiguous(), h[k].contiguous(), active[k].contiguous())):
                assert torch.equal(p[k], q)


def test_unit_rows(device):
    from verace_amd.hip_kernels import unit_rows
    rows, d = 270_000_000, 64
    print("[case] unit_rows", rows, flush=True)
    x = torch.empty(rows, d, device=device, dtype=torch.bfloat16)
    for i in range(0, rows, 30_000_000):
        x[i:i + 30_000_000].normal_()
    with torch.no_grad():
        y = unit_rows(x)
        for k in _spans(rows, 2 ** 32 // 16):
            assert torch.equal(y[k], unit_rows(x[k].contiguous()))
