"""Every form that a feed-forward product can take (tiles of 256 x 256, 256 x 128, 128 x 128 and 64 x 64, the last also by four groups
of waves, and 16, 32 or 64 of a few rows a workgroup), in every kind and type, each element of the result against 64 bits.  The sizes
end inside a tile and the contractions inside a step; which form each case takes is asked of the library (and on the host, without a
device, by test_feed_forward_forms_host.py), so that a change of the rule does not leave a form untested.

The backward's dz is read from its workspace, where it lies first, and is the operand from which dx and dW are then expected."""
import ctypes

import pytest
import torch

from oracle import feed_forward as oracle
from test_gpu_feed_forward import make, randn, va

pytestmark = pytest.mark.gpu

BF, FP, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, oracle.E4M3
CODE = {F32: 0, BF: 1, FP: 2, E4M3: 3}
SIZE = {F32: 4, BF: 2, FP: 2, E4M3: 1}
NAME = {F32: "fp32", BF: "bf16", FP: "fp16", E4M3: "e4m3"}
ACT = {None: 0, "silu": 1, "gelu": 2, "situ": 3}
LARGE, TALL, MIDDLE, SMALL, SMALL_BY_FOUR, ROWS_16, ROWS_32, ROWS_64 = range(8)
LINEAR, GATED, LINEAR_DZ, GATED_DZ, LINEAR_DX, GATED_DX, LINEAR_DW, GATED_DW = range(8)
# rows and columns of the result (gated: of both projections together)
RESULT = {LARGE: (4090, 4085), TALL: (4090, 2045), MIDDLE: (2045, 2043), SMALL: (1020, 1021), SMALL_BY_FOUR: (1020, 1021),
          ROWS_16: (13, 301), ROWS_32: (31, 2101), ROWS_64: (45, 2101)}


def long(steps, more, dtype):
    """A contraction of that many steps of 128 bytes and so many elements."""
    return steps * (128 // SIZE[dtype]) + more


def cases():
    """(product, form, type, M, N, K), N of a gated product F."""
    for form, (m, n) in RESULT.items():
        for dtype in (BF, FP, F32, E4M3):
            rows = form >= ROWS_16
            k = long(33, 5, dtype) if rows or form == SMALL_BY_FOUR else long(2, 3, dtype)
            yield LINEAR, form, dtype, m, n, k
            if form == ROWS_64 and dtype != F32:
                continue  # none that large has more columns than compute units
            if rows and form > ROWS_16:
                gm, f = (m, n) if dtype == F32 else (45, 1101)
            else:
                gm, f = m, n // 2
            yield GATED, form, dtype, gm, f, k if rows or form == SMALL_BY_FOUR else long(9, 3, dtype)
            if dtype == E4M3 or rows:
                continue
            if form != SMALL_BY_FOUR:
                yield LINEAR_DZ, form, dtype, m, n, long(2, 3, dtype)
                yield GATED_DZ, form, dtype, m, n // 2, long(9, 3, dtype)
                yield LINEAR_DW, form, dtype, long(3, 5, dtype), m, n
                yield GATED_DW, form, dtype, long(3, 5, dtype), m // 2, n
            c = long(33, 5, dtype) if form == SMALL_BY_FOUR else long(2, 3, dtype)
            yield LINEAR_DX, form, dtype, m, c, n
            yield GATED_DX, form, dtype, m, c, n
    for dtype in (BF, FP, F32):  # dW in shares of its contraction, which are joined
        yield LINEAR_DW, SMALL if dtype == F32 else MIDDLE, dtype, 1100, 1010, 1021
        yield GATED_DW, SMALL if dtype == F32 else MIDDLE, dtype, 1100, 505, 1021
        yield LINEAR_DW, TALL, dtype, 3000, 1010, 4085
        yield GATED_DW, TALL, dtype, 3000, 505, 4085


def form_of(product, dtype, m, n, k):
    from verace_amd import _lib
    form = ctypes.c_int(-1)
    act = ACT["situ" if product & 1 else "gelu"]
    assert _lib.load().vmi_feed_forward_form(product, CODE[dtype], act, m, n, k, ctypes.byref(form)) == 0
    return form.value


def chosen(*products):
    each = [c for c in cases() if c[0] in products]
    return pytest.mark.parametrize("product,form,dtype,m,n,k", each, ids=[f"{c[0]}-{c[1]}-{NAME[c[2]]}-{c[3]}x{c[5]}x{c[4]}" for c in each])


def all_within(got, want, bound):
    got = got.detach().double()
    assert got.shape == want.shape
    ok = (got - want).abs() <= bound
    if not bool(ok.all()):
        bad = (~ok).nonzero()
        at = tuple(bad[0].tolist())
        assert False, f"{len(bad)} of {ok.numel()} off, the first at {at}, the last at {bad[-1].tolist()}: {got[at]} for {want[at]} +- {bound[at]}"


def wide(t, s=None):
    t = t.detach().double()
    return t if s is None else t * s.double()[:, None]


@chosen(LINEAR, GATED)
def test_forward(product, form, dtype, m, n, k):
    assert form_of(product, dtype, m, n, k) == form
    g = torch.Generator().manual_seed(m + n + k)
    (x, xs), (w, ws), (wu, us) = make(g, m, k, n, dtype, 2)
    out = BF if dtype == E4M3 else dtype
    X, W, U = wide(x, xs), wide(w, ws), wide(wu, us)
    if product == LINEAR:
        b, r = randn(g, n).to(out), randn(g, m, n).to(out)
        y = va().linear_add(x, w, b, r, xs, ws, activation="gelu")
        all_within(y, *oracle.linear(X, W, wide(b), wide(r), "gelu", out, None if xs is None else (xs, ws)))
    else:
        h = va().gated_linear(x, w, wu, xs, ws, us, beta1=2.0, beta2=3.0)
        all_within(h, *oracle.gated(X, W, U, "situ", out, 2.0, 3.0, None if xs is None else (xs, ws, us)))


class Backward:
    """One backward pass, its dz too."""

    def __init__(self, monkeypatch, product, dtype, m, n, k, activation):
        from verace_amd import feed_forward as ff
        monkeypatch.setattr(ff, "_keeps", lambda *_: False)
        real, self.ws = ff._workspace, None

        def workspace(*sizes, **where):
            found = real(*sizes, **where)
            self.ws = found[0]
            return found

        monkeypatch.setattr(ff, "_workspace", workspace)
        g = torch.Generator().manual_seed(m + n + k)
        gated = bool(product & 1)
        self.dtype, self.n = dtype, n
        ts = [t.requires_grad_() for t, _ in make(g, m, k, n, dtype, 2 if gated else 1)]
        self.dy = randn(g, m, n).to(dtype)
        if gated:
            self.grads = torch.autograd.grad(va().gated_linear(*ts, activation=activation, beta1=2.0, beta2=3.0), ts, self.dy)
        else:
            self.b = randn(g, n).to(dtype).requires_grad_()
            self.grads = torch.autograd.grad(va().linear_add(*ts, self.b, activation=activation), (*ts, self.b), self.dy)
        self.x, *self.w = (wide(t) for t in ts)

    def dz(self, parts):
        """[dz] or [dg, du] as they lie, and whether the rest of their rows is zeros."""
        whole = -(-self.n * SIZE[self.dtype] // 16) * 16 // SIZE[self.dtype]
        m = self.dy.shape[0]
        rows = self.ws[:m * parts * whole * SIZE[self.dtype]].view(self.dtype).view(m, parts, whole)
        return [rows[:, i, :self.n] for i in range(parts)], bool((rows[:, :, self.n:] == 0).all())


def sums(a, b, dtype):
    """a b and the bound of fp32 sums of exact operands, rounded once."""
    want = a @ b
    return want, (a.shape[1] + 8) * 2.0 ** -23 * (a.abs() @ b.abs()) + oracle.rounding(want, dtype)


@chosen(LINEAR_DZ, GATED_DZ)
def test_dz(product, form, dtype, m, n, k, monkeypatch):
    assert form_of(product, dtype, m, n, k) == form
    gated = product == GATED_DZ
    t = Backward(monkeypatch, product, dtype, m, n, k, "situ" if gated else "gelu")
    dz, clear = t.dz(2 if gated else 1)
    assert clear
    if gated:
        want = oracle.gated_dz(t.x, *t.w, "situ", wide(t.dy), dtype, 2.0, 3.0)
    else:
        want = [oracle.linear_dz(t.x, *t.w, wide(t.b), "gelu", wide(t.dy), dtype)]
        db = wide(dz[0]).sum(0)
        all_within(t.grads[2], db, (m + 8) * 2.0 ** -23 * wide(dz[0]).abs().sum(0) + oracle.rounding(db, dtype))
    for got, w in zip(dz, want):
        all_within(got, *w)


@chosen(LINEAR_DX, GATED_DX, LINEAR_DW, GATED_DW)
def test_products_of_dz(product, form, dtype, m, n, k, monkeypatch):
    assert form_of(product, dtype, m, n, k) == form
    gated = bool(product & 1)
    t = Backward(monkeypatch, product, dtype, m, n, k, "silu" if gated else None)
    dz = [wide(d) for d in t.dz(2)[0]] if gated else [wide(t.dy)]
    if product in (LINEAR_DX, GATED_DX):
        all_within(t.grads[0], *sums(torch.cat(dz, 1), torch.cat(t.w), dtype))
    else:
        for got, d in zip(t.grads[1:], dz):
            all_within(got, *sums(d.T, t.x, dtype))
