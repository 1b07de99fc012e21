"""The layer's feed-forward on the fused products and in 8 bits, where a program has changed the modules, the weights or the mode
around it."""

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
