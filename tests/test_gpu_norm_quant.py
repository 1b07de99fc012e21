"""Rows in 8 bits, with and without the norm, against their definition in 64 bits: q has to be the same value everywhere."""
import math

import pytest
import torch

from oracle import feed_forward as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# one value, less than a piece, odd, a wave's and a workgroup's limits, and rows that are read twice
WIDTHS = [1, 5, 8, 63, 256, 257, 512, 1000, 1024, 2048, 4001, 4096, 4104, 8192, 16384, 20000]


def va():
    import verace_amd
    return verace_amd


def check(got, want, dtype):
    s, q, scale = got
    ws, wq, wscale = want
    assert q.dtype == oracle.E4M3 and scale.dtype == torch.float32
    assert torch.equal(q.cpu().double().nan_to_num(nan=-1000.0), wq.nan_to_num(nan=-1000.0))
    nan = torch.isnan(wscale)
    assert torch.equal(torch.isnan(scale.cpu()), nan)
    off = (scale.cpu().double() - wscale)[~nan].abs()
    # its own rounding, and that of the sum of squares (64 bits)
    assert bool((off <= wscale[~nan] * 2.0 ** -24 * 1.001).all())
    if s is not None:
        assert s.dtype == dtype
        fine = torch.isfinite(ws)
        assert bool(((s.cpu().double() - ws)[fine].abs() <= oracle.rounding(ws, dtype)[fine]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_norm_add_quant(d, dtype):
    g = torch.Generator().manual_seed(d)
    rows = 9
    a, r = (torch.randn(rows, d, generator=g).mul(s).to(dtype).cuda() for s in (1.0, 2.0))
    w = (1 + 0.1 * torch.randn(d, generator=g)).to(dtype).cuda()
    for residual, weight in ((r, w), (None, w.float()), (r, None)):
        got = va().norm_add_quant(a, residual, weight, eps=1e-6)
        want = oracle.norm_quant(oracle.values(a), None if residual is None else oracle.values(residual),
                                 None if weight is None else oracle.values(weight), float(torch.tensor(1e-6, dtype=torch.float32)))
        check(got, want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_quantize_rows(d, dtype):
    g = torch.Generator().manual_seed(d)
    x = torch.randn(2, 3, d, generator=g).to(dtype).cuda()
    q, scale = va().quantize_rows(x)
    assert q.shape == x.shape and scale.shape == (2, 3)
    check((None, q, scale), oracle.norm_quant(oracle.values(x), None, None, 0.0, norm=False), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(dtype):
    """Rows that hold every tie between two neighbours of e4m3, with 448 as the largest: ties go to even."""
    top = torch.finfo(oracle.E4M3).max
    v = torch.arange(0, 127, dtype=torch.uint8).view(oracle.E4M3).double()
    v = v[torch.isfinite(v)]
    ties = (v[1:] + v[:-1]) / 2
    row = torch.cat([v, ties, -ties, torch.tensor([top], dtype=torch.float64)])
    if dtype == torch.float16:
        row = row / 8
    x = torch.stack([row, row * 2, row / 4, torch.zeros_like(row)]).to(dtype).cuda()
    q, scale = va().quantize_rows(x)
    check((None, q, scale), oracle.norm_quant(oracle.values(x), None, None, 0.0, norm=False), dtype)
    assert float(q[3].float().abs().sum()) == 0


@pytest.mark.parametrize("d", [100, 1024, 8192, 20000])
def test_extremes(d):
    """Subnormal and huge rows, rows of zeros, a NaN or an infinity: the scale stays a normal number, or says so."""
    g = torch.Generator().manual_seed(d)
    base = torch.randn(8, d, generator=g)
    base[0] *= 1e-42
    base[1] *= 1e-37
    base[2] = base[2].clamp(-3, 3) * 1e38
    base[3] = 0
    base[4, d // 2] = math.nan
    base[5, d - 1] = math.inf
    base[6, 1:] = 0
    x = base.cuda()
    q, scale = va().quantize_rows(x)
    check((None, q, scale), oracle.norm_quant(oracle.values(x), None, None, 0.0, norm=False), torch.float32)
    s, q, scale = va().norm_add_quant(x, None, None, eps=1e-6)
    check((s, q, scale), oracle.norm_quant(oracle.values(x), None, None, float(torch.tensor(1e-6, dtype=torch.float32))), torch.float32)
    assert torch.equal(torch.isnan(s), torch.isnan(x)) and torch.equal(torch.isinf(s), torch.isinf(x))


def test_layouts():
    """Slices of wider rows, rows that lie backwards in memory order, a broadcast residual, odd addresses, three dimensions."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(6, 5, 700, generator=g).to(torch.bfloat16).cuda()
    one = torch.randn(700, generator=g).to(torch.bfloat16).cuda()
    for a, r in ((wide[..., :264], wide[..., 300:564]), (wide[..., 1:258], wide[..., 3:260]), (wide.transpose(0, 1), None),
                 (wide.permute(2, 0, 1), None), (wide, one.expand(6, 5, 700)), (wide.flip(0), wide)):
        got = va().norm_add_quant(a, r, None)
        check(got, oracle.norm_quant(oracle.values(a), None if r is None else oracle.values(r), None,
                                     float(torch.tensor(1e-6, dtype=torch.float32))), torch.bfloat16)


def test_empty():
    for shape in ((0, 16), (2, 0, 16)):
        x = torch.empty(shape, device="cuda", dtype=torch.float16)
        s, q, scale = va().norm_add_quant(x, x, None)
        assert s.shape == x.shape and q.shape == x.shape and scale.shape == shape[:-1]
