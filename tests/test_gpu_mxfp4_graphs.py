"""The MXFP4 layer above 16 tokens and the experts' product captured into graphs, and results written over the token rows."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
from test_gpu_few import DEV, _config, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,act,capacity", [(40, api.ACT_SWIGLU, 0.0), (200, api.ACT_GELU, 0.75), (16, api.ACT_SWIGLU, 0.0)])
def test_mxfp4_layer_replayed(S, act, capacity):
    """Two layers captured, replayed in turn with eager calls and other tokens between: every replay is the eager answer to the bit."""
    cfg = _config(S, 320, 448, 12, 3, act, capacity=capacity)
    x, w, _ = _inputs(cfg, "mxfp4", True, seed=S)
    layer, other = moe.MoELayer(cfg), moe.MoELayer(cfg)
    xs = [x, -x, x.roll(1, 0)]
    want = [layer.forward_mxfp4(v, w) for v in xs]
    held = [x.clone(), x.clone()]
    graphs, out = [], []
    for v, l in zip(held, (layer, other)):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(l.forward_mxfp4(v, w))
        graphs.append(g)
    for turn in range(4):
        for i in range(2):
            held[i].copy_(xs[(turn + i) % 3])
            out[i].zero_()
            graphs[i].replay()
        eager = layer.forward_mxfp4(xs[turn % 3], w)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[turn % 3])
        for i in range(2):
            assert torch.equal(out[i], want[(turn + i) % 3])


@pytest.mark.parametrize("rows4", [False, True])
def test_experts_product_replayed_with_other_counts(rows4):
    """The counts are read on the device: a replay follows what they hold by then."""
    E, N, K, A = 6, 192, 320, 300
    g = torch.Generator(device=DEV).manual_seed(5)
    layer = moe.MoELayer(_config(A, K, N, E, 1, api.ACT_RELU))
    a = torch.randn(A, K, generator=g, device=DEV).bfloat16()
    a, sa = moe.quantize_mxfp4(a) if rows4 else (a, None)
    w, s = moe.quantize_mxfp4(torch.randn(E, N, K, generator=g, device=DEV) * 0.05)
    tables = []
    for counts in ((50, 0, 100, 1, 17, 132), (0, 0, 0, 300, 0, 0), (0,) * 6, (1, 2, 3, 4, 5, 6)):
        count = torch.tensor(counts, dtype=torch.int32, device=DEV)
        tables.append((count, (torch.cumsum(count, 0) - count).int()))

    def fresh():
        return torch.full((A, N), 7.0, dtype=torch.bfloat16, device=DEV)

    want = [layer.expert_gemm_mxfp4(a, w, s, None, c, o, a_scales=sa, out=fresh()) for c, o in tables]
    count, offset, out = tables[0][0].clone(), tables[0][1].clone(), fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.expert_gemm_mxfp4(a, w, s, None, count, offset, a_scales=sa, out=out)
    for i in (1, 0, 2, 3, 1):
        count.copy_(tables[i][0]), offset.copy_(tables[i][1]), out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


@pytest.mark.parametrize("weights", ["mxfp4", "own"])
@pytest.mark.parametrize("S,H,E", [(1, 512, 8), (16, 1024, 64), (9, 4096, 4)])
def test_few_tokens_answered_in_place(S, H, E, weights):
    cfg = _config(S, H, 256, E, 2, api.ACT_SWIGLU)
    x, w, _ = _inputs(cfg, weights, True, seed=S)
    layer = moe.MoELayer(cfg)
    want = layer.forward_few(x, w)
    for _ in range(3):
        y = x.clone()
        assert layer.forward_few(y, w, out=y) is y and torch.equal(y, want)
