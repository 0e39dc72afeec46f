"""What the MXFP4 layer looks at before its first launch, alike for a few tokens and for many: on the CPU, with entry points that fail
when they are reached."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api

SIDES = pytest.mark.parametrize("S", [11, 40])
E, H, I = 4, 64, 96


class _Launched(Exception):
    pass


def _layer(monkeypatch, S, act=api.ACT_SWIGLU, dtype=api.DTYPE_BF16):
    """A layer without a handle; _Launched says that a call got as far as an entry point of the library."""
    layer = api.MoELayer.__new__(api.MoELayer)
    layer.cfg = moe.MoEConfig(expert_top_k=2, hidden_act=act, hidden_size=H, intermediate_size=I, micro_batch=1, num_experts=E, sequence_len=S, torch_dtype=dtype)
    layer.S, layer.k, layer.E, layer.H, layer.act_dtype = S, 2, E, H, api._torch_act_dtype(dtype)
    layer._h = layer.workspace = None
    layer.workspace_bytes = 0

    def launched(*a):
        raise _Launched
    layer.L = type("L", (), dict.fromkeys([n for n in api.EXPORTS if n != "moe_destroy"], staticmethod(launched)))
    monkeypatch.setattr(api, "_stream", lambda: None)
    monkeypatch.setattr(api, "_on_current_device", lambda name, t: None)
    return layer


def _set(act=api.ACT_SWIGLU, dtype=torch.bfloat16):
    w = {"gate_w": torch.zeros(E, H, dtype=dtype), "gate_bias": torch.zeros(E)}
    for m in ("up", "down", "gate")[:3 if act == api.ACT_SWIGLU else 2]:
        N, K = (H, I) if m == "down" else (I, H)
        w["w_" + m], w["s_" + m] = torch.zeros(E, N, K // 2, dtype=torch.uint8), torch.zeros(E, N, K // 32, dtype=torch.uint8)
        w["b_" + m] = torch.zeros(E, N, dtype=dtype)
    return w


def _x(S, dtype=torch.bfloat16):
    return torch.zeros(S, H, dtype=dtype)


@SIDES
@pytest.mark.parametrize("act", [api.ACT_RELU, api.ACT_GELU, api.ACT_SWIGLU])
def test_a_whole_set_reaches_the_launches(monkeypatch, S, act):
    layer, w = _layer(monkeypatch, S, act), _set(act)
    for gone in ((), ("gate_bias", "b_up"), ("b_down",)):
        for as_none in (False, True):
            given = {n: None if n in gone else t for n, t in w.items() if as_none or n not in gone}
            with pytest.raises(_Launched):
                layer.forward_mxfp4(_x(S), given)


@SIDES
def test_tensors_that_are_not_the_layers_are_refused(monkeypatch, S):
    """A gate's tensors where the activation has none, prepared operands, unknown names; and missing ones."""
    layer, w, gated = _layer(monkeypatch, S, api.ACT_GELU), _set(api.ACT_GELU), _set()
    for name in ("w_gate", "s_gate", "b_gate"):
        with pytest.raises(ValueError, match=name):
            layer.forward_mxfp4(_x(S), {**w, name: gated[name]})
    for name in ("prepared", "extra"):
        with pytest.raises(ValueError, match=name):
            layer.forward_mxfp4(_x(S), {**w, name: torch.zeros(16, dtype=torch.uint8)})
    layer = _layer(monkeypatch, S)
    for name in ("gate_w", "w_up", "w_gate", "w_down", "s_gate", "s_down"):
        with pytest.raises(ValueError, match=name):
            layer.forward_mxfp4(_x(S), {n: t for n, t in gated.items() if n != name})


def _odd(t):
    """The same values one element further on than 16 bytes."""
    flat = torch.zeros(t.numel() + 16, dtype=t.dtype)
    skip = next(i for i in range(1, 17) if flat[i:].data_ptr() % 16)
    return flat[skip:skip + t.numel()].view(t.shape)


@SIDES
def test_operands_that_do_not_lie_on_16_bytes_are_refused_by_name(monkeypatch, S):
    layer, w = _layer(monkeypatch, S), _set()
    for name in ("gate_w", "w_up", "w_gate", "w_down"):
        with pytest.raises(moe.MoEError, match=name) as e:
            layer.forward_mxfp4(_x(S), {**w, name: _odd(w[name])})
        assert e.value.status == 4
    with pytest.raises(moe.MoEError, match="x does"):
        layer.forward_mxfp4(_odd(_x(S)), w)
    with pytest.raises(_Launched):                   # scales are read byte by byte
        layer.forward_mxfp4(_x(S), {**w, "s_up": _odd(w["s_up"])})
    if S <= api.FEW_TOKENS:
        with pytest.raises(moe.MoEError, match="out does"):
            layer.forward_few(_x(S), w, out=_odd(_x(S)))


@SIDES
@pytest.mark.parametrize("dtype,act_dtype", [(api.DTYPE_FP16, torch.float16), (api.DTYPE_F32, torch.float32), (api.DTYPE_FP8, torch.bfloat16)])
def test_layers_of_another_type_are_refused(monkeypatch, S, dtype, act_dtype):
    with pytest.raises(moe.MoEError) as e:
        _layer(monkeypatch, S, dtype=dtype).forward_mxfp4(_x(S, act_dtype), _set(dtype=act_dtype))
    assert e.value.status == 2


@SIDES
@pytest.mark.parametrize("dtype", [api.DTYPE_BF16, api.DTYPE_FP8])
def test_layers_of_wider_weights_refuse_a_set_in_4_bits(monkeypatch, S, dtype):
    """An e4m3 layer has scales too, and codes of twice the size: it would read past these."""
    layer, w = _layer(monkeypatch, S, dtype=dtype), _set()
    layer.L.moe_prepared_bytes = staticmethod(lambda h, n: setattr(n._obj, "value", 256) or 0)
    for call in (lambda: layer.forward(_x(S), w), lambda: layer.forward(_x(S), w, static_workspace=True),
                 lambda: layer.prepare_weights(w, out=torch.zeros(256, dtype=torch.uint8))):
        with pytest.raises(TypeError, match="forward_mxfp4"):
            call()


def test_products_and_few_tokens_name_what_does_not_lie_right(monkeypatch):
    """... and a bias of the layer for a few tokens that does not lie on 8 bytes; above them any bias will do."""
    for S in (11, 40):
        layer, w = _layer(monkeypatch, S), _set()
        for name in ("b_up", "b_gate", "b_down"):
            shifted = torch.zeros(w[name].numel() + 1, dtype=torch.bfloat16)[1:].view(w[name].shape)
            assert shifted.data_ptr() % 8
            with pytest.raises(moe.MoEError if S <= api.FEW_TOKENS else _Launched, match=name if S <= api.FEW_TOKENS else None):
                layer.forward_mxfp4(_x(S), {**w, name: shifted})
    layer, w = _layer(monkeypatch, 11), _set()
    rows, out, table = torch.zeros(22, H, dtype=torch.bfloat16), torch.zeros(22, I, dtype=torch.bfloat16), torch.zeros(E, dtype=torch.int32)

    def product(a=rows, w=w["w_up"], out=out):
        return layer.expert_gemm_mxfp4(a, w, _set()["s_up"], None, table, table, out=out)

    with pytest.raises(_Launched):
        product()
    for name, kw in (("w", dict(w=_odd(w["w_up"]))), ("a_rows", dict(a=_odd(rows))), ("out", dict(out=_odd(out)))):
        with pytest.raises(moe.MoEError, match=name + " does") as e:
            product(**kw)
        assert e.value.status == 4
    one, scales = w["w_up"][0], w["s_up"][0]
    for name, a, m in (("A", _odd(rows), one), ("w", rows, _odd(one))):
        with pytest.raises(moe.MoEError, match=name + " does"):
            moe.gemm_mxfp4(a, m, scales)
