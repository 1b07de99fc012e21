"""Rows in 8 bits whose sum with the residual is beyond their type's range."""
import math

import pytest
import torch

from oracle import feed_forward as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def va():
    import verace_amd
    return verace_amd


@pytest.mark.parametrize("d", [8, 100, 1024, 8192, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sums_beyond_the_type(d, dtype):
    """The residual's sum beyond the type's largest number, and in bf16 and fp32 beyond fp32's: s is infinite there, while q and the
    scale come from the sum in 64 bits."""
    g = torch.Generator().manual_seed(d)
    top = torch.finfo(dtype).max
    a, r = torch.randn(6, d, generator=g).to(dtype), torch.randn(6, d, generator=g).to(dtype)
    a[0], r[0] = 0.7 * top, 0.6 * top
    a[1, d // 2], r[1, d // 2] = top, top
    a[2], r[2] = -top, -top
    a[3, 0], r[3, 0] = top, -top
    a[4, d - 1], r[4, d - 1] = math.inf, 1.0
    for w in (None, (0.5 + torch.rand(d, generator=g)).to(dtype).cuda()):
        s, q, scale = va().norm_add_quant(a.cuda(), r.cuda(), w, eps=1e-6)
        ws, wq, wscale = oracle.norm_quant(oracle.values(a), oracle.values(r), None if w is None else oracle.values(w),
                                           float(torch.tensor(1e-6, dtype=torch.float32)))
        assert torch.equal(s.cpu(), ws.to(dtype))
        assert torch.equal(q.cpu().double().nan_to_num(nan=-1000.0), wq.nan_to_num(nan=-1000.0))
        nan = torch.isnan(wscale)
        assert nan.tolist() == [False] * 4 + [True, False] and torch.equal(torch.isnan(scale.cpu()), nan)
        off = (scale.cpu().double() - wscale)[~nan].abs()
        assert bool((off <= wscale[~nan] * 2.0 ** -23).all())  # its own rounding, and that of a 16-bit row's terms in the sum of squares
