"""The layer's feed-forward on the fused products and in 8 bits, where a program has changed the modules, the weights or the mode
around it."""
import copy

import pytest
import torch
import torch.nn as nn

from test_gpu_feed_forward import va

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def model(layers=2):
    config = va().VeraceV1Config(vocab_size=128, hidden_dim=256, num_layers=layers, num_heads=2, head_dim=128, chams_holographic_dim=64,
                                 mcmoe_rank=8, mcmoe_num_components=8)
    torch.manual_seed(3)
    return va().VeraceV1Model(config).cuda().to(BF).eval()


def moe():
    torch.manual_seed(4)
    return va().ManifoldContinuousMoE(128, rank=8, num_components=8).cuda().to(BF)


def test_decode_graph_with_another_feed_forward():
    """A layer whose feed-forward is a module of the caller's own decodes in a graph as it does without."""
    m = model()
    m.layers[1].mcmoe = nn.Sequential(nn.Linear(256, 64), nn.SiLU(), nn.Linear(64, 256)).cuda().to(BF)
    ids, nxt = (torch.randint(0, 128, s, device="cuda") for s in ((4, 12), (4, 1)))
    with torch.no_grad():
        held, state = (m.prefill(ids, static_depth=True)[1] for _ in range(2))
        graph = va().DecodeGraph(m, held, 4, static_depth=True)
        for _ in range(3):
            assert torch.equal(graph.step(nxt), m.decode_step(nxt, state, static_depth=True, static_control=True))


class Wider(nn.Linear):
    """A projection with more than its weight (as an adapter adds)."""

    def forward(self, x):
        return super().forward(x) + 1


def test_fused_products_leave_other_modules_to_themselves():
    """A hook, a bias, a replaced module or method on a projection has its effect with fuse_products as without."""
    torch.manual_seed(0)
    x = torch.randn(3, 7, 96, device="cuda").to(BF)
    wide = Wider(96, 160, bias=False).cuda().to(BF)

    def hook(m):
        m.w_gate.register_forward_hook(lambda mod, a, y: y + 1)

    def bias(m):
        m.w_up = nn.Linear(96, 160).cuda().to(BF)

    def replaced(m):
        m.w_gate = wide

    def method(m):
        m.w_up.forward = lambda t: nn.functional.linear(t, m.w_up.weight) * 2

    for change in (hook, bias, replaced, method):
        m = va().SiTUGLU(96, 160).cuda().to(BF)
        plain = m(x)
        change(m)
        want = m(x)
        assert not torch.equal(want, plain)
        m.fuse_products = True
        assert torch.equal(m(x), want), change.__name__


@torch.no_grad()
def test_8_bits_refuse_other_modules():
    """What the 8-bit path would pass by is refused: before a weight is held where it is known then, else by the call."""
    x = torch.randn(1, 5, 128, device="cuda").to(BF)

    def hook(m):
        return m.base_w_down.register_forward_hook(lambda mod, a, y: y + 1)

    def gate_hook(m):
        return m.base_situ_glu.register_forward_pre_hook(lambda mod, a: None)

    def bias(m):
        m.base_w_down = nn.Linear(*m.base_w_down.weight.shape[::-1]).cuda().to(BF)

    def replaced(m):
        m.base_situ_glu.w_up = Wider(*m.base_situ_glu.w_up.weight.shape[::-1], bias=False).cuda().to(BF)

    for change in (hook, gate_hook, bias, replaced):
        m = moe()
        change(m)
        with pytest.raises(RuntimeError, match="plain"):
            m.quantize_base_()
        m(x)  # as it was
        m = moe().quantize_base_()
        want = m(x)
        handle = change(m)
        with pytest.raises(RuntimeError, match="plain"):
            m(x)
        if handle is not None:
            handle.remove()
            assert torch.equal(m(x), want)


@torch.no_grad()
def test_a_model_is_quantized_whole_or_not():
    ids = torch.randint(0, 128, (2, 9), device="cuda")
    for change in (lambda m: m.layers[1].mcmoe.base_w_down.register_forward_hook(lambda mod, a, y: y),
                   lambda m: setattr(m.layers[1], "mcmoe", nn.Linear(256, 256).cuda().to(BF))):
        m = model()
        change(m)
        want = m.prefill(ids, static_depth=True)[0]
        with pytest.raises(RuntimeError, match="plain"):
            m.quantize_feed_forward_()
        assert torch.equal(m.prefill(ids, static_depth=True)[0], want)
        m.quantize_feed_forward_(False)


def test_weights_held_in_inference_mode_are_renewed():
    """Held first under torch.inference_mode(), then anew outside it and inside it again."""
    x = torch.randn(1, 5, 128, device="cuda").to(BF)
    m = moe()
    for i, mode in enumerate((torch.inference_mode, torch.no_grad, torch.inference_mode)):
        with torch.no_grad():
            m.base_w_down.weight.mul_(0.5)
        with mode():
            m.quantize_base_()
        fresh = moe()
        fresh.load_state_dict(m.state_dict())
        with torch.no_grad():
            assert torch.equal(m(x), fresh.quantize_base_()(x)), i


@torch.no_grad()
def test_a_graph_sees_weights_held_again():
    """Off and on again: a graph captured before replays with the weights that are held now, a call of the model too."""
    m = model()
    ids, nxt = (torch.randint(0, 128, s, device="cuda") for s in ((4, 12), (4, 1)))
    m.quantize_feed_forward_()
    held, state = (m.prefill(ids, static_depth=True)[1] for _ in range(2))
    graph = va().DecodeGraph(m, held, 4, static_depth=True)
    m.quantize_feed_forward_(False)
    for layer in m.layers:
        layer.mcmoe.base_w_down.weight.mul_(0.5)
        layer.mcmoe.base_situ_glu.w_up.weight.neg_()
    m.quantize_feed_forward_()
    assert torch.equal(graph.step(nxt), m.decode_step(nxt, state, static_depth=True, static_control=True))


@torch.no_grad()
def test_changed_weights_are_held_anew():
    """An in-place change, a state_dict, other data, another type, a copy of the module: the next call quantizes what it finds."""
    x = torch.randn(1, 5, 128, device="cuda").to(BF)

    def check(m, x):
        fresh = va().ManifoldContinuousMoE(128, rank=8, num_components=8).cuda().to(x.dtype)
        fresh.load_state_dict(m.state_dict())
        got = m(x)
        assert torch.equal(got, fresh.quantize_base_()(x))
        return got

    m = moe().quantize_base_()
    seen = [check(m, x)]
    m.base_w_down.weight.mul_(0.5)
    seen.append(check(m, x))
    m.load_state_dict({k: -v for k, v in m.state_dict().items()})
    seen.append(check(m, x))
    m.base_situ_glu.w_gate.weight.data = m.base_situ_glu.w_gate.weight.data * 1.5
    seen.append(check(m, x))
    m.base_situ_glu.w_up.weight = nn.Parameter(m.base_situ_glu.w_up.weight * 2)
    seen.append(check(m, x))
    for a, b in zip(seen, seen[1:]):
        assert not torch.equal(a, b)
    twin = copy.deepcopy(m)
    twin.base_w_down.weight.zero_()
    check(twin, x)
    assert torch.equal(m(x), seen[-1])
    m.half()
    check(m, x.half())


@torch.no_grad()
def test_changed_weights_are_not_held_by_a_capture():
    """A capture runs nothing: weights that changed since they were held are refused there, and nothing is captured half."""
    x = torch.randn(1, 5, 128, device="cuda").to(BF)
    m = moe().quantize_base_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    m.base_w_down.weight.mul_(0.5)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="quantize_base_"):
        with torch.cuda.graph(graph):
            m(x)
    want = m(x)  # holds them
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(m(x), want)


@torch.no_grad()
def test_weights_held_anew_on_another_stream():
    """A call on a busy side stream finds changed weights; one on the current stream right after it, which need not wait for the other,
    reads what was held, not what was there before."""
    x = torch.randn(1, 5, 128, device="cuda").to(BF)
    m, fresh = moe().quantize_base_(), moe()
    m(x)
    m.base_w_down.weight.mul_(0.5)
    fresh.load_state_dict(m.state_dict())
    want = fresh.quantize_base_()(x)
    a = torch.randn(8192, 8192, device="cuda").to(BF)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(40):
            a = (a @ a).clamp(-1, 1)
        there = m(x)
    here = m(x).clone()
    torch.cuda.synchronize()
    assert torch.equal(here, want) and torch.equal(there, want)


@torch.no_grad()
def test_weights_are_not_held_by_a_capture():
    """Nor by asking for it there: what is held, and how the path runs, stay as they were."""
    x = torch.randn(1, 5, 128, device="cuda").to(BF)
    for m in (moe(), moe().quantize_base_()):
        want = m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(graph):
                m.quantize_base_()
        assert torch.equal(m(x), want)
