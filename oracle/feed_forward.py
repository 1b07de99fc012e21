"""The feed-forward operators from their definitions in 64 bits, with a bound for each result of what rounding can do to it.

A sum of K products in fp32 is off by at most (K + 8) 2^-23 of the sum of their magnitudes (every partial sum rounded, by at
most a whole step where the matrix cores cut instead of rounding); an activation evaluated in fp32 by at most 2^-18 of its
terms' magnitude (an exponential and a reciprocal of a few 2^-23 each, their differences from 1 no closer than 2^-3); a result
rounded to its type by half a step, ``eps / 2`` relative, or half the smallest subnormal.  A gradient of a projection is rounded to
x's type between the backward's products, half a step of each term.

The matrix cores' products of 8-bit rows are rounded before they are added: of eight consecutive ones each is cut to a multiple of
2^-13 of the power of two of the largest, which those with an exponent of eight less and lower can lose a part to (seven at most);
the sums of eight then add up in fp32.

An fp32 number below 2^-126, the least normal one, may be taken as 0: an exponential (the sigmoid of -90 is 8e-40; what it
multiplies, at most the larger of |g| and b1 and the other factor, scales that), an operand of a product, a result.
"""
import math

import torch

E4M3 = torch.float8_e4m3fn
ACT_ERROR = 2.0 ** -18
TINY = 2.0 ** -126


def values(t, scale=None):
    """What a tensor stands for, in 64 bits."""
    t = t.detach().to("cpu").to(torch.float64)
    return t if scale is None else t * scale.detach().cpu().double().unsqueeze(-1)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(x, dtype):
    """How far rounding x to dtype may take it."""
    return x.abs() * half_step(dtype) * (1 + 1e-6) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 + TINY


def product(x, w, scales=None):
    """x w^T and its fp32 sum's bound; scales: of the rows of both, for values that were held in 8 bits."""
    K = x.shape[-1]
    e = (K + 8) * 2.0 ** -23 * (x.abs() @ w.abs().T)
    if scales is not None:
        # a value's power of two is at most the value, and e4m3's least exponent (a zero's too) is -6
        a, b = (torch.maximum(t.abs(), s.detach().to(t.device).double().unsqueeze(-1) * 2.0 ** -6) for t, s in zip((x, w), scales))
        for k in range(0, K, 8):
            most = torch.zeros_like(e)
            for j in range(k, min(k + 8, K)):
                most = torch.maximum(most, a[:, j, None] * b[:, j])
            e = e + 7 * 2.0 ** -13 * most
    return x @ w.T, e


def gate_terms(g, u, activation, b1=4.0, b2=25.0):
    """a(g), a'(g), b(u), b'(u)."""
    s = torch.sigmoid(g)
    if activation == "silu":
        return g * s, s * (1 + g * (1 - s)), u, torch.ones_like(u)
    t1, t2 = torch.tanh(g / b1), torch.tanh(u / b2)
    return b1 * t1 * s, (1 - t1 * t1) * s + b1 * t1 * s * (1 - s), b2 * t2, 1 - t2 * t2


def flushed(g, b1):
    """What a sigmoid taken as 0 may take from a(g) or a'(g)."""
    return TINY * (1 + g.abs().clamp_min(b1))


def gated(x, wg, wu, activation, dtype, b1=4.0, b2=25.0, scales=None):
    """(h, bound) of gated_linear for values in 64 bits; scales: of x, wg and wu where they were held in 8."""
    of_g, of_u = (None, None) if scales is None else ((scales[0], scales[1]), (scales[0], scales[2]))
    (g, eg), (u, eu) = product(x, wg, of_g), product(x, wu, of_u)
    a, da, b, db = gate_terms(g, u, activation, b1, b2)
    h = a * b
    e = (da * b).abs() * eg + (a * db).abs() * eu + 2 * eg * eu + ACT_ERROR * h.abs() + flushed(g, b1) * b.abs()
    return h, e + rounding(h, dtype)


def gated_dz(x, wg, wu, activation, dh, dtype, b1=4.0, b2=25.0):
    """[(dg, bound), (du, bound)], rounded to dtype as operands of products."""
    (g, eg), (u, eu) = product(x, wg), product(x, wu)
    a, da, b, db = gate_terms(g, u, activation, b1, b2)
    dg, du = dh * da * b, dh * a * db
    # slopes change by at most twice their argument's error and the other factor's
    edg = dh.abs() * (2 * b.abs() * eg + da.abs() * eu + 2 * eg * eu) + (ACT_ERROR + flushed(g, b1)) * dh.abs() * b.abs() + rounding(dg, dtype)
    edu = dh.abs() * (2 * a.abs() * eu + da.abs() * eg + 2 * eg * eu) + (ACT_ERROR * a.abs() + flushed(g, b1)) * dh.abs() + rounding(du, dtype)
    return [(dg, edg), (du, edu)]


def gated_bwd(x, wg, wu, activation, dh, dtype, b1=4.0, b2=25.0):
    """[(gradient, bound)] of x, wg, wu."""
    (dg, edg), (du, edu) = gated_dz(x, wg, wu, activation, dh, dtype, b1, b2)
    out = []
    n = 2 * dg.shape[1] + 8
    dx = dg @ wg + du @ wu
    ex = edg @ wg.abs() + edu @ wu.abs() + n * 2.0 ** -23 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    out.append((dx, ex + rounding(dx, dtype)))
    for d, e in ((dg, edg), (du, edu)):
        dw = d.T @ x
        out.append((dw, e.T @ x.abs() + (x.shape[0] + 8) * 2.0 ** -23 * (d.abs().T @ x.abs()) + rounding(dw, dtype)))
    return out


def act(z, activation):
    """act(z), act'(z)."""
    if activation == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if activation == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def linear(x, w, bias, residual, activation, dtype, scales=None):
    """(y, bound) of linear_add; scales: of x and w where they were held in 8 bits."""
    z, e = product(x, w, scales)
    if bias is not None:
        z = z + bias
        e = e + 2.0 ** -23 * z.abs()
    a, da = act(z, activation)
    y = a if residual is None else a + residual
    return y, 1.2 * e + ACT_ERROR * (a.abs() if activation else 0) + 2.0 ** -23 * y.abs() + rounding(y, dtype)


def linear_dz(x, w, bias, activation, dy, dtype):
    """(dz, bound), rounded to dtype as an operand of products where there is an activation."""
    z, e = product(x, w)
    if bias is not None:
        z = z + bias
    _, da = act(z, activation)
    dz = dy * da
    if activation is None:
        return dz, torch.zeros_like(dz)
    # the slopes' own slopes are at most 1
    return dz, dy.abs() * (e + 2.0 ** -23 * z.abs() + ACT_ERROR) + rounding(dz, dtype)


def linear_bwd(x, w, bias, activation, dy, dtype):
    """[(gradient, bound)] of x, weight, bias."""
    dz, edz = linear_dz(x, w, bias, activation, dy, dtype)
    dx, dw, db = dz @ w, dz.T @ x, dz.sum(0)
    M, N = dz.shape
    return [(dx, edz @ w.abs() + (N + 8) * 2.0 ** -23 * (dz.abs() @ w.abs()) + rounding(dx, dtype)),
            (dw, edz.T @ x.abs() + (M + 8) * 2.0 ** -23 * (dz.abs().T @ x.abs()) + rounding(dw, dtype)),
            (db, edz.sum(0) + (M + 8) * 2.0 ** -23 * dz.abs().sum(0) + rounding(db, dtype))]


def to_e4m3(r):
    """64-bit values of at most 448 to the nearest of e4m3, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(r.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(r / step) * step


def norm_quant(a, residual, weight, eps, norm=True):
    """(s, q, scale) in 64 bits; q is exact."""
    s = a if residual is None else a + residual
    p = s if weight is None else s * weight
    rms = torch.sqrt(s.pow(2).mean(-1, keepdim=True) + eps) if norm else torch.ones_like(s[..., :1])
    top = torch.maximum(p.abs().amax(-1, keepdim=True), 448 * 2.0 ** -126 * rms)
    q = to_e4m3(448 * p / top)
    scale = top / (448 * rms)
    lost = ~torch.isfinite(p).all(-1, keepdim=True)
    return s, torch.where(lost, math.nan, q), torch.where(lost, math.nan, scale).squeeze(-1)
