"""The layer for a few tokens on more MXFP4 weights than the memory-side cache holds (256 MB), where its loads are others: against 64 bits."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
from test_gpu_few import DEV, _close, _config, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,gate,S,H,I,E,k", [
    (api.ACT_SWIGLU, api.GATE_SIGMOID, 16, 2048, 1408, 128, 8), (api.ACT_GELU, api.GATE_SOFTMAX, 16, 2048, 1408, 128, 8),
    (api.ACT_RELU, api.GATE_SOFTMAX, 11, 1088, 6208, 96, 8), (api.ACT_SWIGLU, api.GATE_SOFTMAX, 2, 4096, 6464, 16, 4)])
def test_few_tokens_on_weights_that_no_cache_holds(act, gate, S, H, I, E, k):
    """With the tokens spread over the experts, and with two experts that all tokens choose: more than eight rows each, where half of the
    wavefronts work."""
    mats = 3 if act == api.ACT_SWIGLU else 2
    assert min(E, S * k) * H * I // 2 * mats > 256 << 20
    cfg = _config(S, H, I, E, k, act, gate=gate)
    x, w, exact = _inputs(cfg, "mxfp4", True, seed=S + E)
    layer = moe.MoELayer(cfg)
    for crowded in (False, True):
        if crowded:
            w["gate_bias"] = torch.zeros(E, device=DEV)
            w["gate_bias"][[1, E - 2]] = 90.0
        routing = layer.new_routing()
        got = layer.forward_few(x, w, routing=routing)
        assert int(routing["expert_count"].max()) == S if crowded else int(routing["expert_count"].sum()) == S * k
        idx, wts = layer.gate(x, w["gate_w"], w.get("gate_bias"))
        assert torch.equal(routing["topk_idx"], idx) and torch.equal(routing["topk_w"], wts)
        _close(got, x, cfg, w, exact, idx.cpu(), wts.cpu(), routing["slot"].cpu())
        assert torch.equal(layer.forward_few(x, w), got)
