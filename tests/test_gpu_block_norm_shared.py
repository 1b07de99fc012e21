"""A gate that several rows or columns share: its gradient is summed in fp32 and rounded once.

Tolerance: the same chain in plain fp32 makes the same roundings in another order: 8 times its own distance to 64 bits and
2^-20 of the sum of the terms' absolute values (16 more roundings of each), and the result's half step."""
import pytest
import torch

from oracle import selective as ref

pytestmark = pytest.mark.gpu


def _f32(y, res, w1, gate, sc, w2):
    """The oracle's formula in fp32."""
    r = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * w1 * torch.nn.functional.silu(gate)
    s = res + sc * r
    return s, s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + 1e-6) * w2


@pytest.mark.parametrize("traced", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,gate_shape", [((4, 300, 64), (4, 1, 64)), ((4, 300, 64), (64,)), ((2, 70, 96), (2, 70, 1)),
                                              ((1200, 40), (1, 1)), ((3, 5, 1030), (3, 1, 1030)), ((6, 33), (1, 33))])
def test_gradient(device, shape, gate_shape, dtype, traced):
    from verace_amd import gated_norm_add
    g = torch.Generator(device).manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device=device).to(dtype)
    d = shape[-1]
    y, res, gate, ds, dn = r(*shape), r(*shape), r(*gate_shape), r(*shape), r(*shape)
    w1, sc, w2 = (1 + r(d) / 8 for _ in range(3))
    leaf = [t.requires_grad_() for t in (y, res, gate, w1, sc, w2)]

    def own(*t):
        return gated_norm_add(t[0], t[1], t[3], t[2], t[4], t[5])
    torch._dynamo.reset()
    out = (torch.compile(own, backend="aot_eager", fullgraph=True) if traced else own)(*leaf)
    got = torch.autograd.grad(out, leaf, (ds, dn))
    for a, b in zip(got, leaf):
        assert a.shape == b.shape and a.dtype == dtype

    def grad(fn, dt, full):
        t = [v.detach().to(dt).requires_grad_() for v in (y, res, gate.expand(shape) if full else gate, w1, sc, w2)]
        return torch.autograd.grad(fn(t[0], t[1], t[3], t[2], t[4], t[5]), t[2], (ds.to(dt), dn.to(dt)))[0]
    want, terms = grad(ref.gated_norm_add, torch.float64, False), grad(ref.gated_norm_add, torch.float64, True)
    f32 = grad(_f32, torch.float32, False)
    bound = (torch.finfo(dtype).eps / 2 * want.abs() + 8 * (f32.double() - want).abs()
             + 2.0 ** -20 * terms.abs().sum_to_size(gate_shape) + (2.0 ** -25 if dtype == torch.float16 else 0.0))
    assert bool(((got[2].double() - want).abs() <= bound).all()), float(((got[2].double() - want).abs() / bound).max())
