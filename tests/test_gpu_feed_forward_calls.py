"""The feed-forward operators as programs call them: larger tiles of every kind, rows that lie anywhere, non-finite values, other
streams, captured graphs, traces, and a run of them together."""
import pytest
import torch

from oracle import feed_forward as oracle
from test_gpu_feed_forward import make, randn, va, within

pytestmark = pytest.mark.gpu
E4M3 = oracle.E4M3


def rel(got, want):
    got, want = got.detach().double(), want.double()
    return float((got - want).norm() / want.norm())


def wide(t, s=None):
    t = t.detach().double()
    return t if s is None else t * s.double()[:, None]


# Results of 192 and more tiles of 256 x 256, of 256 x 128 and of 128 x 128, each with a ragged edge, and a contraction that ends
# inside a step; on the device in 64 bits.  The bound is of the whole result's norm: half a step (relative, rms below it) of the
# result and of dz, and (K + 8) 2^-23 sqrt(K) at most of a sum's terms.
SHAPES = [(4000, 200, 4200), (4000, 136, 2100), (1500, 72, 1300), (700, 520, 600)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, E4M3])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_tiles(m, k, n, dtype):
    if dtype == torch.float32 and m > 2000:
        m, n = m // 2, n
    g = torch.Generator().manual_seed(m + n)
    (x, xs), (w, ws), (wu, us) = make(g, m, k, n, dtype, 2)
    out = torch.bfloat16 if dtype == E4M3 else dtype
    r = randn(g, m, n).to(out)
    u = oracle.half_step(out) + (k + 8) * 2.0 ** -23
    y = va().linear_add(x, w, None, r, xs, ws)
    X, W, U = wide(x, xs), wide(w, ws), wide(wu, us)
    z = X @ W.T
    assert rel(y, z + wide(r)) < u
    f = n // 2
    h = va().gated_linear(x, w[:f], wu[:f], xs, None if ws is None else ws[:f], None if us is None else us[:f], activation="silu")
    G, V = z[:, :f], (X @ U.T)[:, :f]
    assert rel(h, G * torch.sigmoid(G) * V) < u + 4 * (k + 8) * 2.0 ** -23
    if dtype == E4M3:
        return
    x, w, wu = (t.requires_grad_() for t in (x, w, wu))
    dy = randn(g, m, n).to(dtype)
    b = randn(g, n).to(dtype).requires_grad_()
    grads = torch.autograd.grad(va().linear_add(x, w, b, activation="silu"), (x, w, b), dy)
    z = z + wide(b)
    s = torch.sigmoid(z)
    dz = wide(dy) * s * (1 + z * (1 - s))
    for got, want in zip(grads, (dz @ W, dz.T @ X, dz.sum(0))):
        assert rel(got, want) < 2 * u + max(m, n) * 2.0 ** -23
    dh = dy[:, :f]
    grads = torch.autograd.grad(va().gated_linear(x, w[:f], wu[:f], activation="silu"), (x, w, wu), dh)
    s = torch.sigmoid(G)
    dg, du = wide(dh) * V * s * (1 + G * (1 - s)), wide(dh) * G * s
    for got, want in zip(grads, (dg @ W[:f] + du @ U[:f], torch.cat([dg.T @ X, torch.zeros_like(W[f:])]),
                                 torch.cat([du.T @ X, torch.zeros_like(W[f:])]))):
        assert rel(got, want) < 2 * u + max(m, n) * 2.0 ** -23


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_differences(dtype):
    """The gradients as the change of the result along a direction, in 64 bits from the result's formula: a second proof beside
    the formula's own."""
    g = torch.Generator().manual_seed(2)
    x, wg, wu = (t.requires_grad_() for t, _ in make(g, 33, 48, 40, dtype, 2))
    dh = randn(g, 33, 40).to(dtype)
    grads = torch.autograd.grad(va().gated_linear(x, wg, wu), (x, wg, wu), dh)
    at = [oracle.values(t) for t in (x, wg, wu)]
    for i, got in enumerate(grads):
        v = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        e = 1e-5
        moved = [[t + (s * e * v if j == i else 0) for j, t in enumerate(at)] for s in (1, -1)]
        h = [oracle.gated(*p, "situ", dtype)[0] for p in moved]
        want = float(((h[0] - h[1]) / (2 * e) * oracle.values(dh)).sum())
        # the directional sum: half a step of each gradient and of dz, over independent terms
        scale = float((oracle.values(got) * v).norm())
        assert abs(float((oracle.values(got) * v).sum()) - want) < 8 * oracle.half_step(dtype) * scale + 1e-4 * abs(want) + 1e-6


def test_layouts():
    """Rows of a wider tensor, a transposed weight, odd addresses, expanded rows, three dimensions: the same bits as contiguous
    copies of them."""
    g = torch.Generator().manual_seed(4)
    bf = torch.bfloat16
    base, wbase = randn(g, 6, 7, 400).to(bf), randn(g, 300, 400).to(bf)
    res = randn(g, 6, 7, 500).to(bf)
    one = randn(g, 264).to(bf)
    xs = [base[..., :264], base[..., 8:272], base[..., 1:265], base[..., :264].transpose(0, 1), base[:, :, :264].flip(2),
          one.expand(6, 7, 264), base[::2, :, :264], base[2, 3, :264]]
    ws = [wbase[:96, :264], wbase[:96, 3:267], wbase[:264, :96].t(), wbase[::3, :264], wbase[:1, :264].expand(96, 264), wbase[:96, 8:272]]
    for x in xs:
        for w in ws:
            n = w.shape[0]
            r = res[..., 5:5 + n]
            r = r.transpose(0, 1) if x.shape[0] == 7 else r[:x.shape[0]] if x.dim() == 3 else r[0, 0]
            a = va().linear_add(x, w, None, r)
            assert torch.equal(a, va().linear_add(x.contiguous(), w.contiguous(), None, r.contiguous()))
            a = va().gated_linear(x, w, wbase[:n, :264])
            assert torch.equal(a, va().gated_linear(x.contiguous(), w.contiguous(), wbase[:n, :264].contiguous()))
    # gradients that arrive broadcast, or as slices
    x, w = base[..., :264].contiguous().requires_grad_(), wbase[:96, :264].contiguous().requires_grad_()
    for dy in (torch.ones((), device="cuda", dtype=bf).expand(6, 7, 96), res[..., 3:99], res.transpose(0, 1)[..., :96].transpose(0, 1)):
        a = torch.autograd.grad(va().linear_add(x, w, activation="silu"), (x, w), dy)
        b = torch.autograd.grad(va().linear_add(x, w, activation="silu"), (x, w), dy.contiguous())
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        a = torch.autograd.grad(va().gated_linear(x, w, w), (x, w), dy)
        b = torch.autograd.grad(va().gated_linear(x, w, w), (x, w), dy.contiguous())
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_shared_and_needed_gradients():
    """One tensor as both weights and as x and residual: the sum of its gradients; only what is needed comes back."""
    g = torch.Generator().manual_seed(6)
    x, w, r = (randn(g, *s).requires_grad_() for s in ((20, 64), (64, 64), (20, 64)))
    dy = randn(g, 20, 64)
    a, b = w.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    dw, = torch.autograd.grad(va().gated_linear(x, w, w, activation="silu"), w, dy)
    da, db = torch.autograd.grad(va().gated_linear(x, a, b, activation="silu"), (a, b), dy)
    assert torch.equal(dw, da + db)
    dx, = torch.autograd.grad(va().linear_add(x, w, None, x), x, dy)
    dx0, = torch.autograd.grad(va().linear_add(x, w, None, r), x, dy)
    assert torch.equal(dx, dx0 + dy)
    only, = torch.autograd.grad(va().linear_add(x.detach(), w.detach(), None, r, activation="gelu"), r, dy)
    assert torch.equal(only, dy)
    only, = torch.autograd.grad(va().linear_add(x.detach(), w, None, r), w, dy)
    assert torch.equal(only, torch.autograd.grad(va().linear_add(x, w, None, r), (x, w), dy)[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_empty(dtype):
    for m, k, n in ((0, 16, 8), (5, 0, 8), (5, 16, 0), (0, 0, 0), (5, 3, 0)):
        x, w, u = (torch.ones(s, device="cuda", dtype=dtype, requires_grad=True) for s in ((m, k), (n, k), (n, k)))
        b = torch.full((n,), 2.0, device="cuda", dtype=dtype, requires_grad=True)
        y = va().linear_add(x, w, b)
        assert y.shape == (m, n) and bool((y == (2 + k)).all())
        h = va().gated_linear(x, w, u)
        assert h.shape == (m, n) and (k > 0 or bool((h == 0).all()))
        for t, gt in zip((x, w, b), torch.autograd.grad(y, (x, w, b), torch.ones_like(y))):
            assert gt.shape == t.shape
        db, = torch.autograd.grad(va().linear_add(x, w, b), b, torch.ones_like(y))
        assert torch.equal(db, torch.full_like(db, float(m)))
        for t, gt in zip((x, w, u), torch.autograd.grad(h, (x, w, u), torch.ones_like(h))):
            assert gt.shape == t.shape and (m > 0 and n > 0 and k > 0 or bool((gt == 0).all()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [5, 300, 3000])
def test_non_finite_stays_in_its_row_and_column(m, dtype):
    """A NaN or an infinity in a row of x reaches that row of y, in a row of the weight that column; both gradients likewise."""
    g = torch.Generator().manual_seed(m)
    x, w = randn(g, m, 100).to(dtype), randn(g, 150, 100).to(dtype)
    clean = va().linear_add(x, w)
    x[m // 2, 99] = float("nan")
    w[149, 0] = float("inf")
    y = va().linear_add(x, w)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[m // 2] = True
    hit[:, 149] = True
    assert not bool(torch.isfinite(y[hit]).any()) and torch.equal(y[~hit], clean[~hit])
    h = va().gated_linear(x, w[:75], w[75:])
    assert bool(torch.isfinite(h[~hit[:, 75:]]).all()) and bool(torch.isnan(h[m // 2]).all())
    # an infinite row of the gradient
    x, w = (randn(g, *s).to(dtype).requires_grad_() for s in ((m, 100), (150, 100)))
    dy = randn(g, m, 150).to(dtype)
    a = torch.autograd.grad(va().linear_add(x, w), (x, w), dy)
    dy[m - 1] = float("nan")
    b = torch.autograd.grad(va().linear_add(x, w), (x, w), dy)
    assert bool(torch.isnan(b[0][m - 1]).all()) and torch.equal(a[0][:m - 1], b[0][:m - 1]) and bool(torch.isnan(b[1]).all())


@pytest.mark.parametrize("activation", ["situ", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_activations_far_out(dtype, activation):
    """Arguments from the smallest to where everything saturates; the projections are the values themselves."""
    v = torch.tensor([0.0, 1e-30, 1e-6, 1e-4, 3e-3, 0.05, 0.39, 0.41, 1.0, 3.0, 14.9, 15.1, 60.0, 90.0, 3e3, 6e4])
    v = torch.cat([v, -v]).to(dtype)
    n = v.numel()
    x = torch.zeros(n * n, 16, dtype=dtype)
    x[:, 0], x[:, 1] = v.repeat_interleave(n), v.repeat(n)
    wg, wu = torch.zeros(3, 16, dtype=dtype), torch.zeros(3, 16, dtype=dtype)
    wg[:, 0], wu[:, 1] = 1, 1
    x, wg, wu = (t.cuda().requires_grad_() for t in (x, wg, wu))
    h = va().gated_linear(x, wg, wu, activation=activation)
    X, G, U = (oracle.values(t) for t in (x, wg, wu))
    want, bound = oracle.gated(X, G, U, activation, dtype)
    top = torch.finfo(dtype).max
    fine = want.abs() < top
    assert bool(torch.isfinite(h.cpu())[fine].all())
    within(torch.where(fine.cuda(), h.detach(), 0), torch.where(fine, want, 0), bound)
    dh = torch.ones_like(h)
    dx, = torch.autograd.grad(h, x, dh)
    (want, bound), *_ = oracle.gated_bwd(X, G, U, activation, oracle.values(dh), dtype)
    fine = want.abs() < top / 4
    within(torch.where(fine.cuda(), dx, 0), torch.where(fine, want, 0), bound)


def block(x, r, wg, wu, wd, b, norm):
    """The 16-bit feed-forward block, differentiable."""
    h = va().gated_linear(x, wg, wu)
    return va().linear_add(h, wd, b, r)


def block8(a, r, w8, norm):
    """The same on rows in 8 bits."""
    s, q, scale = va().norm_add_quant(a, r, norm)
    (wg, sg), (wu, su), (wd, sd) = w8
    h, hs = va().quantize_rows(va().gated_linear(q, wg, wu, scale, sg, su, out_dtype=a.dtype))
    return va().linear_add(h, wd, None, s, hs, sd, out_dtype=a.dtype)


@pytest.mark.parametrize("m", [1, 64, 500])
def test_block_in_8_bits(m):
    """The whole serving path against 64 bits of the same 8-bit rows and weights."""
    g = torch.Generator().manual_seed(m)
    bf = torch.bfloat16
    a, r, norm = randn(g, m, 256).to(bf), randn(g, m, 256).to(bf), (1 + 0.1 * randn(g, 256)).to(bf)
    w8 = [va().quantize_rows(randn(g, *s, scale=s[1] ** -0.5).to(bf)) for s in ((512, 256), (512, 256), (256, 512))]
    y = block8(a, r, w8, norm)
    S, Q, scale = oracle.norm_quant(oracle.values(a), oracle.values(r), oracle.values(norm), 1e-6)
    W = [oracle.values(*w) for w in w8]
    h, _ = oracle.gated(Q * scale[:, None], W[0], W[1], "situ", bf)
    h8 = va().quantize_rows(h.to(bf).cuda())
    want = oracle.values(*h8) @ W[2].T + S.to(bf).double()
    # h may fall on the other side of a step of e4m3 (an eighth) where its own rounding to bf16 does: of a hundredth of its values
    assert rel(y.cpu(), want) < oracle.half_step(bf) + 0.1 * 2.0 ** -4


def test_streams():
    """Work on a side stream, and tensors made on it."""
    g = torch.Generator().manual_seed(9)
    bf = torch.bfloat16
    args = [randn(g, *s).to(bf) for s in ((300, 128), (300, 128), (256, 128), (256, 128), (128, 256))]
    x, r, wg, wu, wd = args
    norm = torch.ones(128, device="cuda", dtype=bf)
    w8 = [va().quantize_rows(w) for w in (wg, wu, wd)]
    want = block8(x, r, w8, norm), block(x, r, wg, wu, wd, None, norm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block8(x.clone(), r.clone(), w8, norm), block(x.clone(), r.clone(), wg, wu, wd, None, norm)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_graphs():
    """Two captured graphs, a forward with its backward and the 8-bit block, replayed in turn with eager work between: every
    replay gives the eager result on the inputs that it finds."""
    g = torch.Generator().manual_seed(10)
    bf = torch.bfloat16
    x, r = randn(g, 200, 128).to(bf), randn(g, 200, 128).to(bf)
    wg, wu, wd = (randn(g, *s, scale=0.1).to(bf) for s in ((264, 128), (264, 128), (128, 264)))
    norm = torch.ones(128, device="cuda", dtype=bf)
    w8 = [va().quantize_rows(w) for w in (wg, wu, wd)]

    def train(x, r):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
        y = va().linear_add(va().gated_linear(*leaves[:3]), leaves[3], None, r, activation="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]

    def serve(x, r):
        with torch.no_grad():
            return [block8(x, r, w8, norm)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train(x, r), serve(x, r)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for f in (train, serve):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(x, r)
        graphs.append((graph, f, out))
    for i in range(4):
        x.copy_(randn(g, 200, 128))
        r.copy_(randn(g, 200, 128))
        for graph, f, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            want = f(x, r)
            for a, b in zip(out, want):
                assert torch.equal(a, b), i


def test_same_bits_every_time():
    g = torch.Generator().manual_seed(12)
    x, wg, wu = (t.requires_grad_() for t, _ in make(g, 3000, 192, 200, torch.bfloat16, 2))
    dh = randn(g, 3000, 200).to(torch.bfloat16)
    runs = [torch.autograd.grad(va().gated_linear(x, wg, wu), (x, wg, wu), dh) for _ in range(3)]
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_registered_operators():
    g = torch.Generator().manual_seed(13)
    bf = torch.bfloat16
    x, w, b, r = randn(g, 10, 32).to(bf), randn(g, 24, 32).to(bf), randn(g, 24).to(bf), randn(g, 10, 24).to(bf)
    grad = [t.clone().requires_grad_() for t in (x, w, b, r)]
    ops = torch.ops.verace
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(ops.gated_linear, (grad[0], grad[1], grad[1].detach().clone().requires_grad_(), None, None, None, "situ", 4.0, 25.0, bf),
                          test_utils=checks)
    torch.library.opcheck(ops.linear_add, (*grad, None, None, "gelu", bf), test_utils=checks)
    # the schema's check multiplies its tensors, which torch does not do in 8 bits
    torch.library.opcheck(ops.norm_add_quant, (x, x, None, 1e-6), test_utils=checks[1:2])
    torch.library.opcheck(ops.quantize_rows, (x,), test_utils=checks[1:2])
    xq, wq = va().quantize_rows(x), va().quantize_rows(w)
    torch.library.opcheck(ops.linear_add, (xq[0], wq[0], b, r, xq[1], wq[1], None, bf), test_utils=checks[1:2])
    with torch.no_grad():
        def f(x):
            s, q, scale = va().norm_add_quant(x, x, None)
            return va().linear_add(va().gated_linear(x, w, w), w.t(), None, s), va().linear_add(q, wq[0], None, r, scale, wq[1])
        fn = torch.jit.trace(f, (x,))
        for t in (x, x * 2, x.neg()):
            assert all(torch.equal(a, c) for a, c in zip(fn(t), f(t)))
    # under a function mode: the registered operators, with their gradients
    outs = []
    for device in (None, "cuda"):
        torch.set_default_device(device)
        try:
            y = va().linear_add(*grad, activation="silu")
            h = va().gated_linear(grad[0], grad[1], grad[1])
            outs.append([*torch.autograd.grad((y, h), grad, (r, r))])
        finally:
            torch.set_default_device(None)
    assert all(torch.equal(a, c) for a, c in zip(*outs))


def test_forward_mode_is_refused():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: va().linear_add(d, w), lambda: va().gated_linear(d, w, w), lambda: va().norm_add_quant(d), lambda: va().quantize_rows(d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_a_second_derivative_is_refused():
    x, w = torch.randn(4, 16, device="cuda", requires_grad=True), torch.randn(8, 16, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(va().linear_add(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_on_the_fused_products(dtype):
    """SiTUGLU with its products fused, in training, against the separate ops."""
    torch.manual_seed(0)
    m = va().SiTUGLU(96, 160).cuda().to(dtype)
    x = torch.randn(2, 50, 96, device="cuda").to(dtype)
    dy = torch.randn(2, 50, 160, device="cuda").to(dtype)
    outs = []
    for fused in (False, True):
        m.fuse_products = fused
        t = x.clone().requires_grad_()
        y = m(t)
        outs.append([y.detach(), *torch.autograd.grad(y, (t, *m.parameters()), dy)])
    for a, b in zip(*outs):
        # the separate ops round five times in between, each at most a half step of a factor near 1
        assert a.dtype == b.dtype and rel(b, a) < 8 * oracle.half_step(dtype) + 1e-5
    assert m.state_dict().keys() == {"w_gate.weight", "w_up.weight"}


def test_model_in_8_bits():
    """A model's feed-forward base path in 8 bits: prompts and single tokens run, near the 16-bit ones; off again, the same bits."""
    config = va().VeraceV1Config(vocab_size=128, hidden_dim=256, num_layers=2, num_heads=2, head_dim=128, chams_holographic_dim=64,
                                 mcmoe_rank=8, mcmoe_num_components=8)
    torch.manual_seed(0)
    model = va().VeraceV1Model(config).cuda().to(torch.bfloat16)
    ids = torch.randint(0, 128, (2, 40), device="cuda")
    keys = set(model.state_dict())
    with torch.no_grad():
        want, state = model.prefill(ids, static_depth=True)
        model.quantize_feed_forward_()
        assert set(model.state_dict()) == keys
        got, state8 = model.prefill(ids, static_depth=True)
        step = model.decode_step(ids[:, :1], state8, static_depth=True)
        assert bool(torch.isfinite(step).all())
        # two layers' base paths, each from rows and weights with relative errors of up to 2^-4 (rms a third of it)
        assert 0 < rel(got, want) < 0.1
        model.quantize_feed_forward_(False)
        assert torch.equal(model.prefill(ids, static_depth=True)[0], want)
    model.quantize_feed_forward_()
    with pytest.raises(RuntimeError, match="no gradients"):
        model.layers[0].mcmoe(torch.randn(1, 4, 256, device="cuda", dtype=torch.bfloat16))


def test_under_autocast():
    """The fused products give way to the separate ops, and the path in 8 bits gives what they would: autocast's dtype."""
    torch.manual_seed(1)
    m = va().ManifoldContinuousMoE(128, rank=8, num_components=8).cuda()
    x = torch.randn(2, 20, 128, device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = m.base_situ_glu(x)
        base = m.parts(x)[0]
        m.base_situ_glu.fuse_products = True
        assert torch.equal(m.base_situ_glu(x), want)
        m.quantize_base_()
        got = m.parts(x)[0]
    assert got.dtype == base.dtype == torch.bfloat16
    # as for the model: relative errors of up to 2^-4 in each of rows and weights, twice
    assert 0 < rel(got, base) < 0.1


def test_decode_graph_in_8_bits():
    """A decode step captured with the base path in 8 bits: its replays keep to 8 bits after the model has gone back, and take
    weights that are quantized anew."""
    config = va().VeraceV1Config(vocab_size=128, hidden_dim=256, num_layers=2, num_heads=2, head_dim=128, chams_holographic_dim=64,
                                 mcmoe_rank=8, mcmoe_num_components=8)
    torch.manual_seed(2)
    model = va().VeraceV1Model(config).cuda().to(torch.bfloat16).eval()
    ids = torch.randint(0, 128, (4, 12), device="cuda")
    nxt = torch.randint(0, 128, (4, 1), device="cuda")

    with torch.no_grad():
        for renew in (False, True):
            model.quantize_feed_forward_()
            held, state = (model.prefill(ids, static_depth=True)[1] for _ in range(2))  # the graph's states are its caller's to keep
            graph = va().DecodeGraph(model, held, 4, static_depth=True)
            if renew:
                for layer in model.layers:
                    layer.mcmoe.base_w_down.weight.mul_(0.5)
                model.quantize_feed_forward_()
            want = model.decode_step(nxt, state, static_depth=True, static_control=True)
            model.quantize_feed_forward_(renew)
            junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
            assert torch.equal(graph.step(nxt), want)
            del junk
            model.quantize_feed_forward_(False)
