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
@pytest.mark.parametrize("T,P,N", [(150, 33, 20), (230, 64, 128), (300, 64, 64), (530, 33, 20), (700, 64, 128), (705, 20, 7)])
def test_segments(device, T, P, N, dtype):
    """Long enough to be cut into segments, few (the last pass joins them) and more (a kernel does); sequences that
    end in the first segment, inside a later one and before the first token."""
    from verace_amd import selective_scan
    d, state = inputs(device, 3, T, 2, P, 1, N, dtype, seed=40)
    check(selective_scan(**d, initial_state=state), d, state)
    lengths = torch.tensor([T - 170, 0, 5], device=device)
    check(selective_scan(**d, lengths=lengths), d, None, lengths)


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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_tokens_reach_no_earlier_one(device, dtype, bad):
    """A NaN or an infinity in a token's x, delta, B or C leaves every earlier token's y as it is, and the
    other heads' (x, delta) and channels' (x)."""
    from verace_amd import selective_scan
    d, state = inputs(device, 2, 100, 4, 32, 2, 64, dtype, seed=30)
    y0, S0 = selective_scan(**d, initial_state=state)
    ym, Sm = ref.selective_scan(**d, initial_state=state, magnitude=True)
    # the chunk of such a token is summed in another order: both results are within check()'s bound of the exact
    # one, and so within twice that of each other
    bound = 2 * (torch.finfo(dtype).eps / 2 * y0.double().abs() +
                 ((8 * 100 + 64 + 16) * U + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)) * ym)

    def same(y, part):
        return bool(((y.double() - y0.double()).abs() <= bound)[part].all())
    for k in ("x", "delta", "B", "C"):
        e = {n: None if v is None else v.clone() for n, v in d.items()}
        at = {"x": (1, 45, 2, 7), "delta": (1, 45, 2), "B": (1, 45, 1, 7), "C": (1, 45, 1, 7)}[k]
        e[k][at] = bad
        y, S = selective_scan(**e, initial_state=state)
        assert torch.equal(y[0], y0[0]) and torch.equal(S[0], S0[0]), k
        assert same(y, (1, slice(0, 45))), k
        assert not bool(torch.isfinite(y[1, 45, 2]).all()), k
        assert torch.equal(y[1, :, :2], y0[1, :, :2]), k           # the first group's heads
        if k in ("x", "delta"):
            assert torch.equal(y[1, :, 3], y0[1, :, 3]), k         # the other head of the group
        if k == "x":
            keep = [p for p in range(32) if p != 7]
            assert same(y, (1, slice(None), 2, keep)) and torch.equal(S[1, 2][keep], S0[1, 2][keep])
        if k == "C":
            assert torch.equal(y[1, 46:], y0[1, 46:]) and torch.equal(S, S0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strong_decays(device, dtype):
    """Log decays of hundreds a token and of none at all: differences of a chunk's sums keep their accuracy."""
    from verace_amd import selective_scan
    d, state = inputs(device, 1, 150, 4, 32, 1, 32, dtype, seed=31, delta_dtype=torch.float32)
    d["A"] = torch.tensor([-1e-6, -3.0, -200.0, -1e4], device=device)
    check(selective_scan(**d, initial_state=state), d, state)


def test_graph_replays(device):
    """Scan, convolution, norm and both steps captured in one graph with states updated in place: each replay,
    between eager work, gives the eager bits."""
    from verace_amd import gated_norm_add, selective_scan, selective_step_, short_conv, short_conv_step_
    g = torch.Generator(device).manual_seed(40)

    def r(*s):
        return torch.randn(*s, generator=g, device=device).to(torch.bfloat16)
    B, H, P, N = 2, 4, 64, 128
    x, w, b, cs = r(B, 300, H * P), r(H * P, 4), r(H * P), r(B, 3, H * P)
    delta, Bm, Cm = r(B, 300, H), r(B, 300, 1, N), r(B, 300, 1, N)
    A, nw = -torch.rand(H, generator=g, device=device), r(H * P)
    S = torch.randn(B, H, P, N, generator=g, device=device)
    tok = r(B, 1, H * P)

    def run(cs, S):
        y, last = short_conv(x, w, b)
        o, fin = selective_scan(y.view(B, 300, H, P), delta, A, Bm, Cm)
        s, n = gated_norm_add(o.reshape(B, 300, H * P), x, nw, y, nw, nw)
        t = short_conv_step_(tok, w, b, cs)
        z = selective_step_(t.view(B, 1, H, P), delta[:, :1], A, Bm[:, :1], Cm[:, :1], S)
        return last, fin, s, n, t, z
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(cs.clone(), S.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    cs1, S1, cs2, S2 = cs.clone(), S.clone(), cs.clone(), S.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(cs1, S1)
    cs1.copy_(cs), S1.copy_(S)
    for i in range(4):
        x.add_(0.125 * i)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, run(cs2, S2)):
            assert torch.equal(p, q), i
        assert torch.equal(cs1, cs2) and torch.equal(S1, S2)


def test_other_streams_at_once(device):
    """Two calls on two streams at the same time, each with its own workspace."""
    from verace_amd import selective_scan
    d1, s1 = inputs(device, 1, 700, 4, 64, 1, 128, torch.bfloat16, seed=50)
    d2, s2 = inputs(device, 2, 500, 2, 64, 2, 64, torch.float32, seed=51)
    want1, want2 = selective_scan(**d1, initial_state=s1), selective_scan(**d2, initial_state=s2)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got1, got2 = [], []
    for _ in range(5):
        with torch.cuda.stream(a):
            got1.append(selective_scan(**d1, initial_state=s1))
        with torch.cuda.stream(b):
            got2.append(selective_scan(**d2, initial_state=s2))
    torch.cuda.synchronize()
    for got, want in ((got1, want1), (got2, want2)):
        for y, S in got:
            assert torch.equal(y, want[0]) and torch.equal(S, want[1])
