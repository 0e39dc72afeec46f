"""What the layer on rows in e4m3 refuses for its sizes before its first launch: on the CPU, with stages that fail when they are reached."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api


class _Launched(Exception):
    pass


def _call(monkeypatch, S, k, E, H, I, norm=False):
    def launched(*a, **kw):
        raise _Launched
    for stage in ("quantize_rows128", "rms_norm_rows128"):
        monkeypatch.setattr(api, stage, launched)
    monkeypatch.setattr(api, "_on_current_device", lambda name, t: None)
    monkeypatch.setattr(api, "_on_16_bytes", lambda name, t, n=16: None)
    layer = api.MoELayer.__new__(api.MoELayer)
    layer.cfg = moe.MoEConfig(expert_top_k=k, hidden_act=api.ACT_GELU, hidden_size=H, intermediate_size=I, micro_batch=1, num_experts=E, sequence_len=S,
                              torch_dtype=api.DTYPE_FP8)
    layer.S, layer.k, layer.E, layer.H = S, k, E, H
    layer._h = None
    empty = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device="meta")     # noqa: E731
    w = {"gate_w": empty(torch.bfloat16, E, H)}
    for name, (N, K) in (("up", (I, H)), ("down", (H, I))):
        w["w_" + name], w["s_" + name] = empty(torch.uint8, E, N, K), empty(torch.float32, E, N // 128, K // 128)
    layer.forward_block128(empty(torch.bfloat16, S, H), w, empty(torch.bfloat16, H) if norm else None)


# S, k, E, H, I: the tokens' rows hold 3 GiB; the activation's values; a matrix of 3 GiB; combine's launch
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("sizes", [(196608, 1, 1, 16384, 128), (1 << 20, 2, 2, 128, 16384), (4, 1, 1, 16384, 196608), (1 << 24, 1, 1, 128, 128)])
def test_sizes_that_a_stage_refuses_launch_nothing(monkeypatch, sizes, norm):
    with pytest.raises(api.MoEError) as e:
        _call(monkeypatch, *sizes, norm=norm)
    assert e.value.status == api._UNSUPPORTED


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("sizes", [(196607, 1, 1, 16384, 128), ((1 << 20) - 128, 2, 2, 128, 16384), (4, 1, 1, 16384, 196480), (1, 1, 1, 128, 128), (2000, 8, 256, 7168, 2048)])
def test_sizes_below_are_launched(monkeypatch, sizes, norm):
    with pytest.raises(_Launched):
        _call(monkeypatch, *sizes, norm=norm)
