"""The operators of a selective state space layer used together on the GPU: a projection's row [gate | x | B | C | delta]
through the short convolution, the scan and the gated norm with the next block's norm, as prompt, token by token,
in training, captured into a graph and through torch.compile (aot_eager: operator by operator).

Tolerance: the same formulas in plain fp32 make the same roundings, in another order, so an fp32 chain may be off by a
small multiple of the plain chain's own distance to 64 bits (norms over a tensor): 8 times it, and 2^-20 for sums that
the plain form happens to round exactly."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H, P, G, N, K = 4, 32, 2, 16, 4
INNER, CONV = H * P, H * P + 2 * G * N
PARAMS = ("w", "b", "A", "D", "dt", "norm", "scale", "next")


def _params(device, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    p = dict(w=0.5 * r(CONV, K), b=0.1 * r(CONV), A=-torch.exp(r(H)), D=r(H), dt=r(H) - 2, norm=1 + 0.1 * r(INNER),
             scale=1 + 0.1 * r(INNER), next=1 + 0.1 * r(INNER))
    f32 = ("A", "D", "dt")
    return {k: v.to(torch.float32 if k in f32 else dtype).to(device) for k, v in p.items()}


def _rows(device, B, T, dtype=torch.float32, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, T, INNER + CONV + H, generator=g).to(dtype).to(device),
            torch.randn(B, T, INNER, generator=g).to(dtype).to(device))


def _split(c):
    B, T = c.shape[:2]
    x, bm, cm = c.split([INNER, G * N, G * N], -1)
    return x.reshape(B, T, H, P), bm.reshape(B, T, G, N), cm.reshape(B, T, G, N)


def layer(p, rows, res, lengths=None, conv=None, state=None):
    import verace_amd as va
    gate, c, delta = rows.split([INNER, CONV, H], -1)
    c, conv = va.short_conv(c, p["w"], p["b"], conv, lengths)
    x, bm, cm = _split(c)
    y, state = va.selective_scan(x, delta, p["A"], bm, cm, p["D"], p["dt"], True, state, lengths)
    s, n = va.gated_norm_add(y.flatten(2), res, p["norm"], gate, p["scale"], p["next"])
    return s, n, conv, state


def plain(p, rows, res, lengths=None):
    """In rows' dtype: fp32 or 64 bits."""
    gate, c, delta = rows.split([INNER, CONV, H], -1)
    B, T = rows.shape[:2]
    n = [T] * B if lengths is None else lengths.tolist()
    on = torch.tensor([[t < v for t in range(T)] for v in n], device=rows.device)
    c = torch.where(on[..., None], c, torch.zeros_like(c))
    full = torch.cat([c.new_zeros(B, K - 1, CONV), c], 1)
    z = sum(full[:, j:j + T] * p["w"][:, j] for j in range(K)) + p["b"]
    conv = torch.stack([full[i, v:v + K - 1] for i, v in enumerate(n)])
    x, bm, cm = _split(z * torch.sigmoid(z))
    bm, cm = bm.repeat_interleave(H // G, 2), cm.repeat_interleave(H // G, 2)
    step = torch.nn.functional.softplus(delta + p["dt"])
    S, ys = x.new_zeros(B, H, P, N), []
    for t in range(T):
        live = on[:, t].view(B, 1, 1, 1)
        d = step[:, t]
        S1 = torch.exp(d * p["A"])[..., None, None] * S + (d[..., None] * x[:, t])[..., None] * bm[:, t].unsqueeze(2)
        S = torch.where(live, S1, S)
        y = (S * cm[:, t].unsqueeze(2)).sum(-1) + p["D"][:, None] * x[:, t]
        ys.append(torch.where(live[..., 0], y, torch.zeros_like(y)))
    y = torch.stack(ys, 1).flatten(2)
    r = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * p["norm"] * torch.nn.functional.silu(gate)
    s = res + p["scale"] * r
    return s, s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + 1e-6) * p["next"], conv, S


def _close(got, p32, p64, what):
    off = (got.double() - p64).norm()
    allowed = 8 * (p32.double() - p64).norm() + 2.0 ** -20 * p64.norm()
    assert off <= allowed, (what, float(off), float(allowed))


def _double(p):
    return {k: v.double() for k, v in p.items()}


LENGTHS = [None, [70, 33, 1, 0]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=["full", "ragged"])
def test_prompt_then_tokens(device, lengths):
    """A prompt, and 5 more tokens one at a time from its states, against the whole at once."""
    import verace_amd as va
    T, more = 70, 5
    p = _params(device)
    rows, res = _rows(device, 4, T + more)
    n = torch.tensor(lengths or [T] * 4)
    # each sequence's tokens behind its own length
    at = [torch.stack([t[i, v:v + more] for i, v in enumerate(n.tolist())]) for t in (rows, res)]
    print("[case] prompt then tokens", lengths, flush=True)
    got = layer(p, rows[:, :T], res[:, :T], None if lengths is None else n.to(device))
    whole = n + more
    a32 = plain(p, rows, res, whole)
    a64 = plain(_double(p), rows.double(), res.double(), whole)
    b32, b64 = plain(p, rows[:, :T], res[:, :T], n), plain(_double(p), rows[:, :T].double(), res[:, :T].double(), n)
    for name, g, x, y in zip(("s", "n", "conv", "state"), got, b32, b64):
        _close(g, x, y, name)
    conv, state = got[2].clone(), got[3].clone()
    for t in range(more):
        r, q = at[0][:, t], at[1][:, t:t + 1]
        gate, c, delta = r.split([INNER, CONV, H], -1)
        c = va.short_conv_step_(c, p["w"], p["b"], conv)
        x, bm, cm = _split(c)
        y = va.selective_step_(x, delta.unsqueeze(1), p["A"], bm, cm, state, p["D"], p["dt"])
        s, m = va.gated_norm_add(y.flatten(2), q, p["norm"], gate.unsqueeze(1), p["scale"], p["next"])
        pick = lambda k: [torch.stack([o[k][i, v + t] for i, v in enumerate(n.tolist())]).unsqueeze(1) for o in (a32, a64)]
        _close(s, *pick(0), ("s", t))
        _close(m, *pick(1), ("n", t))
    assert torch.equal(conv, a32[2])
    _close(state, a32[3], a64[3], "state")


@pytest.mark.parametrize("lengths", LENGTHS, ids=["full", "ragged"])
def test_gradients(device, lengths):
    p = _params(device)
    rows, res = _rows(device, 4, 70)
    n = None if lengths is None else torch.tensor(lengths, device=device)
    g = torch.Generator().manual_seed(5)
    w = [torch.randn(s, generator=g).to(device) for s in ((4, 70, INNER), (4, 70, INNER), (4, H, P, N))]
    print("[case] gradients", lengths, flush=True)

    def grads(fn, dt):
        q = {k: v.to(dt).requires_grad_(True) for k, v in p.items()}
        r, t = rows.to(dt).requires_grad_(True), res.to(dt).requires_grad_(True)
        s, m, _, st = fn(q, r, t, n)
        loss = sum((a * b.to(dt)).sum() for a, b in zip((s, m, st), w))
        return torch.autograd.grad(loss, [r, t] + [q[k] for k in PARAMS])
    got, p32, p64 = grads(layer, torch.float32), grads(plain, torch.float32), grads(plain, torch.float64)
    for name, a, b, c in zip(("rows", "res") + PARAMS, got, p32, p64):
        _close(a, b, c, name)
    if n is not None:
        off = torch.arange(70, device=device) >= n[:, None]
        assert not got[0][off][:, INNER:].any()


def test_prompt_and_gradients_in_a_graph(device):
    """Forward and backward captured once and replayed on new contents, eager work between the replays."""
    p = {k: v.requires_grad_(True) for k, v in _params(device, torch.bfloat16).items()}
    rows, res = _rows(device, 2, 100, torch.bfloat16)
    n = torch.tensor([100, 41], device=device)
    leaf = [rows.clone().requires_grad_(True), res.clone().requires_grad_(True)]

    def run(r, t):
        s, m, _, st = layer(p, r, t, n)
        loss = s.float().square().mean() + m.float().sum() + st.square().sum()
        grads = torch.autograd.grad(loss, [r, t] + [p[k] for k in PARAMS])
        return (s.detach(), m.detach(), st.detach(), *grads)  # no autograd graph outlives a run
    print("[case] graph", flush=True)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        run(*leaf)
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*leaf)
    for seed, lens in ((11, [100, 41]), (12, [3, 100]), (13, [0, 64])):
        new = _rows(device, 2, 100, torch.bfloat16, seed)
        n.copy_(torch.tensor(lens))
        with torch.no_grad():
            for a, b in zip(leaf, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = run(*(t.requires_grad_(True) for t in new))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_opcheck(device):
    import verace_amd  # noqa: F401
    ops = torch.ops.verace
    p = _params(device)
    rows, res = _rows(device, 2, 40)
    gate, c, delta = (t.contiguous() for t in rows.split([INNER, CONV, H], -1))
    x, bm, cm = (t.contiguous() for t in _split(c))
    y = x.flatten(2)
    n = torch.tensor([40, 7], device=device)
    st, cs = torch.randn(2, H, P, N, device=device), torch.randn(2, K - 1, CONV, device=device)
    leaf = lambda t: t.detach().clone().requires_grad_(True)
    cases = [
        (ops.short_conv, (leaf(c), leaf(p["w"]), leaf(p["b"]), leaf(cs), n, "silu")),
        (ops.short_conv, (leaf(c), leaf(p["w"]), None, None, None, None)),
        (ops.short_conv_bwd, (c, p["w"], p["b"], cs, n, "silu", torch.randn_like(c), None)),
        (ops.short_conv_step_, (c[:, 0].clone(), p["w"], p["b"], cs.clone(), "silu", None)),
        (ops.selective_scan, (leaf(x), leaf(delta), leaf(p["A"]), leaf(bm), leaf(cm), leaf(p["D"]), leaf(p["dt"]), True,
                              leaf(st), n)),
        (ops.selective_scan, (leaf(x), leaf(delta), leaf(p["A"]), leaf(bm), leaf(cm), None, None, True, None, None)),
        (ops.selective_scan_bwd, (x, delta, p["A"], bm, cm, torch.randn_like(x), p["D"], p["dt"], True, st, n, st.clone())),
        (ops.selective_step_, (x[:, :1].clone(), delta[:, :1].clone(), p["A"], bm[:, :1].clone(), cm[:, :1].clone(),
                               st.clone(), p["D"], p["dt"], True, torch.tensor([True, False], device=device))),
        (ops.gated_norm, (leaf(y), leaf(res), leaf(gate), leaf(p["norm"]), leaf(p["scale"]), leaf(p["next"]), 1e-6, 1e-5,
                          "silu")),
        (ops.gated_norm, (leaf(y), leaf(res), None, leaf(p["norm"]), None, None, 1e-6, 1e-6, "sigmoid")),
        (ops.gated_norm_bwd, (y, res, gate, p["norm"], p["scale"], p["next"], torch.rand(2, 80, device=device), "silu",
                              torch.randn_like(y), None)),
    ]
    for op, args in cases:
        print("[case] opcheck", op, flush=True)
        torch.library.opcheck(op.default, args)


def test_compile_fullgraph(device):
    """The traced layer, forward and gradients, has the eager one's bits (fp32 sums in one order either way)."""
    p = {k: v.requires_grad_(True) for k, v in _params(device).items()}
    rows, res = _rows(device, 2, 50)
    n = torch.tensor([50, 20], device=device)

    def loss(r, t):
        s, m, conv, st = layer(p, r, t, n)
        return s.sum() + (m * m).sum() + st.sum() + conv.sum()
    print("[case] compile", flush=True)
    outs = []
    for fn in (loss, torch.compile(loss, fullgraph=True, backend="aot_eager")):
        r, t = rows.clone().requires_grad_(True), res.clone().requires_grad_(True)
        v = fn(r, t)
        outs.append((v.detach(), *torch.autograd.grad(v, [r, t] + [p[k] for k in PARAMS])))
    for a, b in zip(*outs):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)
