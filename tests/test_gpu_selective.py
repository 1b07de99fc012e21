"""GPU parity of the selective scan (csrc/selective*.hip) with the 64-bit recurrence: prompts and the
in-place step.

Tolerances, u = 2^-24, h the result's half step, M the same recurrence of absolute values (what each
rounding scales with).  fp32 arithmetic: a token's decay and input carry at most 8 roundings and the decays
only shrink them, so a state is within 8 T u of its M; a readout adds N + 16 of them.  With bf16 inputs the
matrix products take the decayed scores and the carried state rounded to bf16 once each, every term of y by
at most 2^-8: 2^-8 M on top of the result's own rounding; the states themselves are carried exactly as in
fp32."""
import pytest
import torch

from oracle import selective as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def inputs(device, B, T, H, P, G, N, dtype, seed=0, delta_dtype=None):
    g = torch.Generator(device).manual_seed(seed + T * 13 + H * 7 + P + N)

    def r(*s):
        return torch.randn(*s, generator=g, device=device)
    d = dict(x=r(B, T, H, P).to(dtype), delta=r(B, T, H).to(delta_dtype or dtype),
             A=-(0.5 + 8 * torch.rand(H, generator=g, device=device)), B=r(B, T, G, N).to(dtype),
             C=r(B, T, G, N).to(dtype), D=r(H), delta_bias=-3 + r(H))
    return d, r(B, H, P, N)


def check(got, d, state, lengths=None, softplus=True):
    y, S = got
    T, N, dtype = d["x"].shape[1], d["B"].shape[-1], d["x"].dtype
    kw = dict(softplus=softplus, initial_state=state, lengths=lengths)
    y64, S64 = ref.selective_scan(**d, **kw)
    ym, Sm = ref.selective_scan(**d, **kw, magnitude=True)
    h = torch.finfo(dtype).eps / 2
    assert y.dtype == dtype and S.dtype == torch.float32 and y.shape == y64.shape and S.shape == S64.shape
    inner = (8 * T + N + 16) * U + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    ey, es = (y.double() - y64).abs(), (S.double() - S64).abs()
    assert bool((ey <= h * y64.abs() + inner * ym).all()), float((ey / ym.clamp_min(1e-30)).max())
    assert bool((es <= (8 * T + 16) * U * Sm).all()), float((es / Sm.clamp_min(1e-30)).max())


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 2, 64, 1, 128), (2, 5, 4, 16, 2, 16), (1, 64, 2, 64, 1, 64), (1, 65, 2, 24, 1, 20),
          (2, 130, 4, 64, 2, 128), (1, 200, 2, 128, 1, 128), (3, 77, 3, 40, 3, 48), (1, 70, 2, 33, 1, 7),
          (1, 150, 1, 64, 1, 256), (1, 90, 2, 200, 1, 130), (2, 16, 2, 64, 1, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(device, shape, dtype):
    from verace_amd import selective_scan
    d, state = inputs(device, *shape, dtype)
    check(selective_scan(**d), d, None)
    check(selective_scan(**d, initial_state=state), d, state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_options(device, dtype):
    """Without D or bias, the step size itself, fp32 step sizes, growing states, no decay."""
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 100, 4, 64, 2, 64, dtype, seed=3, delta_dtype=torch.float32)
    e = dict(d, D=None, delta_bias=None)
    check(selective_scan(**e), e, None)
    e = dict(e, delta=torch.rand_like(d["delta"]) * 0.1)
    check(selective_scan(**e, softplus=False, initial_state=state), e, state, softplus=False)
    check(selective_scan(**dict(e, delta=e["delta"].unsqueeze(-1)), softplus=False), e, None, softplus=False)
    e = dict(e, A=0.1 * torch.rand(4, device=device))
    check(selective_scan(**e, softplus=False), e, None, softplus=False)
    e = dict(e, A=torch.zeros(4, device=device))
    check(selective_scan(**e, softplus=False), e, None, softplus=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths(device, dtype):
    """Nothing behind a length is used (NaN and infinities there), y is 0 there, an empty sequence keeps its
    state; lengths are clamped."""
    from verace_amd import selective_scan
    d, state = inputs(device, 6, 140, 2, 64, 1, 64, dtype, seed=4)
    n = torch.tensor([0, 1, 64, 140, 65, 500], device=device)
    for k in ("x", "delta", "B", "C"):
        for i, m in enumerate(n.tolist()):
            d[k][i, m:] = float("nan") if i % 2 else float("inf")
    y, S = selective_scan(**d, initial_state=state, lengths=n.int())
    clean = {k: (torch.nan_to_num(v, 0.0, 0.0, 0.0) if k in ("x", "delta", "B", "C") else v) for k, v in d.items()}
    check((y, S), clean, state, n.clamp(max=140))
    assert torch.equal(S[0], state[0]) and float(y[0].abs().sum()) == 0.0
    y2, S2 = selective_scan(**d, lengths=n)
    check((y2, S2), clean, None, n.clamp(max=140))


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_are_the_whole(device, dtype):
    """A prompt in pieces, each from the state the last one left."""
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 300, 4, 64, 1, 128, dtype, seed=5)
    S, ys = state, []
    for a, b in ((0, 1), (1, 70), (70, 198), (198, 300)):
        part = {k: (v[:, a:b] if k in ("x", "delta", "B", "C") else v) for k, v in d.items()}
        y, S = selective_scan(**part, initial_state=S)
        ys.append(y)
    check((torch.cat(ys, 1), S), d, state)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,P,G,N", [(1, 1, 1, 1, 1), (2, 4, 64, 1, 128), (3, 2, 24, 2, 20), (2, 2, 33, 1, 7),
                                       (64, 32, 64, 1, 128), (2, 2, 128, 1, 256)])
def test_step(device, B, H, P, G, N, dtype):
    from verace_amd import selective_step_
    d, state = inputs(device, B, 4, H, P, G, N, dtype, seed=6)
    S, ys = state.clone(), []
    for t in range(4):
        sl = slice(t, t + 1) if t % 2 else t
        ys.append(selective_step_(d["x"][:, sl], d["delta"][:, sl], d["A"], d["B"][:, sl], d["C"][:, sl], S, D=d["D"],
                                  delta_bias=d["delta_bias"]))
    check((torch.cat(ys, 1), S), d, state)


def test_step_mask(device):
    from verace_amd import selective_step_
    d, state = inputs(device, 4, 1, 2, 64, 1, 128, torch.bfloat16, seed=7)
    for k in ("x", "delta", "B", "C"):
        d[k][1] = float("nan")
    S = state.clone()
    y = selective_step_(d["x"], d["delta"], d["A"], d["B"], d["C"], S, active_mask=torch.tensor([1, 0, 1, 0], device=device))
    assert torch.equal(S[1], state[1]) and torch.equal(S[3], state[3]) and not torch.equal(S[0], state[0])
    assert float(y[1].abs().sum()) == 0.0 and float(y[3].abs().sum()) == 0.0 and bool(torch.isfinite(S).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_strided_rows(device, dtype, off):
    """x, B and C as slices of one wide row, at aligned and odd columns; delta as a slice of another."""
    from verace_amd import selective_scan
    B, T, H, P, G, N = 2, 90, 2, 32, 1, 48
    wide = torch.randn(B, T, H * P + 2 * G * N + 16, device=device).to(dtype)
    d, _ = inputs(device, B, T, H, P, G, N, dtype, seed=8)
    d["x"] = wide[..., off:off + H * P].unflatten(-1, (H, P))
    d["B"] = wide[..., off + H * P:off + H * P + N].unsqueeze(2)
    d["C"] = wide[..., off + H * P + N:off + H * P + 2 * N].unsqueeze(2)
    d["delta"] = torch.randn(B, T, 7, device=device).to(dtype)[..., 3:5]
    check(selective_scan(**d), d, None)


def test_no_tokens_and_no_items(device):
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 0, 2, 16, 1, 16, torch.float32)
    y, S = selective_scan(**d, initial_state=state)
    assert y.shape == (2, 0, 2, 16) and torch.equal(S, state)
    assert float(selective_scan(**d)[1].abs().sum()) == 0.0
    d, _ = inputs(device, 0, 5, 2, 16, 1, 16, torch.float32)
    assert selective_scan(**d)[0].shape == (0, 5, 2, 16)
