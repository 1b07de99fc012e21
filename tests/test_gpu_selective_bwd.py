"""GPU parity of the selective scan's backward (csrc/selective_bwd.hip) with the 64-bit recurrence.

Tolerances, u = 2^-24, h the result's half step.  Each gradient is a sum of products along paths through the
recurrence; m is the same gradient with every factor's absolute value (A's sign kept: decays shrink), which is
what each rounding scales with.  fp32 arithmetic: a path carries at most 8 roundings a token and N + P + 64 from
its products: (8 T + N + P + 64) u m.  With bf16 inputs every term of dx, dB and dC may carry one rounding to
bf16 of a score and one of the carried gradient: 2^-7 m; the step sizes' gradients, dA, dD, dbias and the
initial state's carry none."""
import pytest
import torch

from oracle import selective as ref

from test_gpu_selective import DTYPES, SHAPES, U, inputs

pytestmark = pytest.mark.gpu
NAMES = ("x", "delta", "A", "B", "C", "D", "delta_bias", "initial_state")


def magnitudes(d, state, dy, dS, lengths, softplus):
    """The gradients of the sum of absolute values: x, B, C, states, dy positive, the step sizes' own sign
    irrelevant (positive), the decays as they are.  A token's log decay takes the paths across it."""
    with torch.no_grad():
        x, B, C, D = (None if d[k] is None else d[k].double().abs() for k in ("x", "B", "C", "D"))
        z = d["delta"].double() + (0 if d["delta_bias"] is None else d["delta_bias"].double())
        if z.dim() == 4:
            z = z.squeeze(-1)
        b, T, H, P = x.shape
        r = H // B.shape[2]
        G, N = B.shape[2:]
        on = torch.arange(T, device=x.device) < (torch.full((b,), T, device=x.device) if lengths is None else lengths)[:, None]
        st = torch.logaddexp(z, torch.zeros_like(z)) if softplus else z
        st = st * on.unsqueeze(-1)
        a, st, A = torch.exp(st * d["A"].double()), st.abs(), d["A"].double().abs()
        B, C = B.repeat_interleave(r, 2), C.repeat_interleave(r, 2)
        live = on.view(b, T, 1, 1).double()
        x, B, C, dy = (torch.nan_to_num(t * live, 0, 0, 0) for t in (x, B, C, dy.double().abs()))
        S = torch.zeros(b, H, P, N, dtype=torch.float64, device=x.device) if state is None else state.double().abs()
        states = [S]
        for t in range(T):
            states.append(a[:, t, :, None, None] * states[-1] + st[:, t, :, None, None] * x[:, t].unsqueeze(-1) * B[:, t].unsqueeze(2))
        g = torch.zeros_like(S) if dS is None else dS.double().abs()
        m = {k: torch.zeros_like(t) for k, t in (("x", x), ("delta", st), ("B", B), ("C", C))}
        mA = torch.zeros_like(A)
        for t in range(T - 1, -1, -1):
            m["C"][:, t] = (dy[:, t].unsqueeze(-1) * states[t + 1]).sum(2)
            g = g + dy[:, t].unsqueeze(-1) * C[:, t].unsqueeze(2)
            gB = (g * B[:, t].unsqueeze(2)).sum(-1)
            m["x"][:, t] = st[:, t, :, None] * gB
            m["B"][:, t] = st[:, t, :, None] * (g * x[:, t].unsqueeze(-1)).sum(2)
            # a token's own term also appears in, and cancels out of, the sums over its chunk
            la = (g * states[t + 1]).sum((-1, -2))
            m["delta"][:, t] = (x[:, t] * gB).sum(-1) + A * la
            mA += (st[:, t] * la).sum(0)
            g = g * a[:, t, :, None, None]
        if D is not None:
            m["x"] += D[:, None] * dy
        # the sums of a chunk of up to 64 tokens share their roundings: its largest
        c = m["delta"]
        pad = torch.cat([c, c.new_zeros(b, -T % 64, H)], 1).view(b, -1, 64, H)
        m["delta"] = pad.amax(2, keepdim=True).expand(pad.shape).reshape(b, -1, H)[:, :T] + c
        m["B"], m["C"] = (m[k].view(b, T, G, r, N).sum(3) for k in ("B", "C"))
        m["A"], m["D"], m["delta_bias"], m["initial_state"] = mA, (x * dy).sum((0, 1, 3)), m["delta"].sum((0, 1)), g
        return m


def check(d, state, dy, dS, lengths=None, softplus=True, clean=None, clean_dy=None):
    from verace_amd import selective_scan
    own = {k: None if t is None else t.clone().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    names = [k for k in NAMES if own[k] is not None]
    y, S = selective_scan(**own, softplus=softplus, lengths=lengths)
    outs, grads = (y, S) if dS is not None else (y,), (dy, dS) if dS is not None else (dy,)
    got = dict(zip(names, torch.autograd.grad(outs, [own[k] for k in names], grads)))
    d, dy = clean or d, dy if clean_dy is None else clean_dy
    r = {k: None if t is None else t.double().requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    y, S = ref.selective_scan(**r, softplus=softplus, lengths=lengths)
    want = torch.autograd.grad((y, S), [r[k] for k in names],
                               (dy.double(), torch.zeros_like(S) if dS is None else dS.double()), allow_unused=True)
    want = {k: torch.zeros_like(r[k]) if w is None else w for k, w in zip(names, want)}
    m = magnitudes(d, state, dy, dS, lengths, softplus)
    T, P, N = d["x"].shape[1], d["x"].shape[3], d["B"].shape[-1]
    for k in names:
        assert got[k].dtype == own[k].dtype and got[k].shape == own[k].shape, k
        h = torch.finfo(got[k].dtype).eps / 2
        inner = (8 * T + N + P + 64) * U
        if k in ("x", "B", "C") and d["x"].dtype == torch.bfloat16:
            inner += 2.0 ** -7
        err = (got[k].double() - want[k]).abs()
        bad = err > h * want[k].abs() + inner * m[k].view(want[k].shape)
        assert not bool(bad.any()), (k, float((err / m[k].view(want[k].shape).clamp_min(1e-30)).max()), inner)
    return got


def grads_of(device, d, state, seed):
    g = torch.Generator(device).manual_seed(seed)
    return (torch.randn(d["x"].shape, generator=g, device=device).to(d["x"].dtype),
            torch.randn(state.shape, generator=g, device=device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(device, shape, dtype):
    d, state = inputs(device, *shape, dtype, seed=11)
    dy, dS = grads_of(device, d, state, 12)
    check(d, state, dy, dS)
    check(d, None, dy, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_heads_and_segments(device, dtype):
    """More heads than a workgroup walks, and enough chunks to be split along time."""
    d, state = inputs(device, 1, 640, 12, 64, 2, 64, dtype, seed=13)
    dy, dS = grads_of(device, d, state, 14)
    check(d, state, dy, dS)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_options(device, dtype):
    d, state = inputs(device, 2, 100, 4, 64, 2, 64, dtype, seed=15, delta_dtype=torch.float32)
    dy, dS = grads_of(device, d, state, 16)
    e = dict(d, D=None, delta_bias=None)
    check(e, state, dy, dS)
    e = dict(e, delta=torch.rand_like(d["delta"]) * 0.1)
    check(e, state, dy, dS, softplus=False)
    check(dict(e, delta=e["delta"].unsqueeze(-1)), state, dy, dS, softplus=False)
    check(dict(e, A=torch.zeros(4, device=device)), state, dy, dS, softplus=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths(device, dtype):
    """Nothing behind a length is used, and its gradients are zero."""
    d, state = inputs(device, 5, 140, 2, 64, 1, 64, dtype, seed=17)
    dy, dS = grads_of(device, d, state, 18)
    n = torch.tensor([0, 1, 64, 140, 65], device=device)
    clean = {k: None if v is None else v.clone() for k, v in d.items()}
    for k in ("x", "delta", "B", "C"):
        for i, q in enumerate(n.tolist()):
            d[k][i, q:] = float("nan")
            clean[k][i, q:] = 0.0
    zero = dy.clone()
    for i, q in enumerate(n.tolist()):
        dy[i, q:] = float("nan")
        zero[i, q:] = 0.0
    got = check(d, state, dy, dS, n, clean=clean, clean_dy=zero)
    for k in ("x", "delta", "B", "C"):
        for i, q in enumerate(n.tolist()):
            assert float(got[k][i, q:].abs().sum()) == 0.0, k
    assert torch.equal(got["initial_state"][0], dS[0])


def test_gradient_against_differences(device):
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 70, 2, 16, 1, 16, torch.float32, seed=19)
    dy, dS = grads_of(device, d, state, 20)
    leaves = {k: t.requires_grad_() for k, t in {**d, "initial_state": state}.items()}
    got = torch.autograd.grad(selective_scan(**leaves), list(leaves.values()), (dy, dS))
    for (k, t), g in zip(leaves.items(), got):
        v = torch.randn_like(t)

        def f(e):
            u = {n: q.detach().double() for n, q in leaves.items()}
            u[k] = u[k] + e * v.double()
            y, S = ref.selective_scan(**u)
            return float((y * dy).sum() + (S * dS).sum())
        num = (f(1e-6) - f(-1e-6)) / 2e-6
        assert abs(float((g * v).double().sum()) - num) <= 1e-4 * float((g * v).abs().sum()) + 1e-6, k


def test_strided_and_expanded_gradients(device):
    """x, B, C as slices of one projection (its gradient collects all three), a gradient expanded from a sum."""
    from verace_amd import selective_scan
    H, P, N = 2, 32, 48
    wide = torch.randn(2, 90, H * P + 2 * N, device=device, requires_grad=True)
    d, _ = inputs(device, 2, 90, H, P, 1, N, torch.float32, seed=21)

    def split(w):
        return dict(d, x=w[..., :H * P].unflatten(-1, (H, P)), B=w[..., H * P:H * P + N].unsqueeze(2),
                    C=w[..., H * P + N:].unsqueeze(2))
    got, = torch.autograd.grad(selective_scan(**split(wide))[0].sum(), wide)
    w64 = wide.detach().double().requires_grad_()
    want, = torch.autograd.grad(ref.selective_scan(**split(w64))[0].sum(), w64)
    assert float((got.double() - want).norm() / want.norm()) < 1e-5


def test_repeats(device):
    """The same bits in every run."""
    from verace_amd import launch_selective_hip_scan_bwd
    d, state = inputs(device, 2, 500, 16, 64, 1, 128, torch.bfloat16, seed=22)
    dy, dS = grads_of(device, d, state, 23)
    first = launch_selective_hip_scan_bwd(**d, dy=dy, initial_state=state, d_state=dS)
    for _ in range(3):
        for p, q in zip(first, launch_selective_hip_scan_bwd(**d, dy=dy, initial_state=state, d_state=dS)):
            assert torch.equal(p, q)


def test_no_tokens(device):
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 0, 2, 16, 1, 16, torch.float32)
    A, state = d["A"].requires_grad_(), state.requires_grad_()
    y, S = selective_scan(**d, initial_state=state)
    dA, d0 = torch.autograd.grad(S.sum(), (A, state))
    assert float(dA.abs().sum()) == 0.0 and torch.equal(d0, torch.ones_like(d0))
