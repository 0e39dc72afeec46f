"""What the MXFP4 entry points and the layer for a few tokens refuse, on the host: nothing here needs a GPU."""
import ctypes as C

import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api, weights as W
import mxfp4_plain as plain

OK, BAD, UNSUPPORTED = 0, 4, 2
P = C.c_void_p(1 << 20)                 # some address, aligned; none of these calls gets as far as reading it
ODD = C.c_void_p((1 << 20) + 8)


def test_quantise_arguments():
    L = moe.load_library()
    q = lambda x=P, dt=api.DTYPE_BF16, rows=4, K=64, c=P, s=P: L.moe_quant_mxfp4(x, dt, rows, K, c, s, None)     # noqa: E731
    d = lambda c=P, s=P, rows=4, K=64, dt=api.DTYPE_BF16, o=P: L.moe_dequant_mxfp4(c, s, rows, K, dt, o, None)   # noqa: E731
    for call in (q, d):
        for kw in (dict(rows=-1), dict(K=0), dict(K=16), dict(K=48), dict(K=-32), dict(c=None), dict(s=None), dict(rows=1 << 40, K=1 << 20),
                   dict(rows=1 << 62, K=64)):
            assert call(**kw) == BAD, kw
        for dt in (api.DTYPE_TF32, api.DTYPE_FP8, api.DTYPE_MXFP4, -1):
            assert call(dt=dt) == UNSUPPORTED
        assert call(rows=0) == OK
    assert q(x=None) == BAD and q(x=ODD) == BAD and d(o=None) == BAD and d(o=ODD) == BAD
    assert q(c=C.c_void_p(2)) == BAD


def test_product_arguments():
    L = moe.load_library()

    def g(a=P, sa=None, dt=api.DTYPE_BF16, w=P, s=P, bias=None, out=P, M=4, N=64, K=64, act=api.ACT_NONE):
        return L.moe_gemm_mxfp4(a, sa, dt, w, s, bias, out, M, N, K, act, None)

    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(K=40), dict(a=None), dict(w=None), dict(s=None), dict(out=None), dict(act=api.ACT_SWIGLU),
               dict(act=7), dict(sa=P), dict(dt=api.DTYPE_MXFP4), dict(a=ODD), dict(w=ODD), dict(out=ODD), dict(bias=C.c_void_p(3))):
        assert g(**kw) == BAD, kw
    for kw in (dict(dt=api.DTYPE_F32), dict(dt=api.DTYPE_FP16), dict(N=1 << 23, K=1024), dict(K=1 << 21, N=1), dict(M=1 << 32),
               dict(M=(1 << 31) - 1, N=1 << 20), dict(N=1 << 40)):
        assert g(**kw) == UNSUPPORTED, kw
    assert g(M=0) == OK and g(M=0, a=None, out=None) == OK


def test_python_refuses_what_it_can_see():
    """Types, shapes and places are looked at before anything is called: on the CPU every one of these ends in Python."""
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="current GPU"):
        moe.quantize_mxfp4(x)
    with pytest.raises(ValueError, match="multiple of 32"):
        moe.quantize_mxfp4(torch.zeros(4, 48))
    with pytest.raises(ValueError, match="multiple of 32"):
        moe.quantize_mxfp4(torch.zeros(()))
    with pytest.raises(TypeError):
        moe.quantize_mxfp4(x.double())
    codes, scales = plain.quantize(x)
    with pytest.raises(TypeError):
        moe.dequantize_mxfp4(codes, scales, dtype=torch.int8)
    with pytest.raises(TypeError):
        moe.dequantize_mxfp4(codes.int(), scales)
    with pytest.raises(ValueError, match="multiple of 32"):
        moe.dequantize_mxfp4(codes[:, :5], scales)
    with pytest.raises(ValueError, match="current GPU"):
        moe.dequantize_mxfp4(codes, scales)
    with pytest.raises(ValueError, match="matrices"):
        moe.gemm_mxfp4(x.bfloat16()[0], codes, scales)
    with pytest.raises(ValueError):
        moe.gemm_mxfp4(x.bfloat16(), codes, scales[:, :1])
    with pytest.raises(TypeError):
        moe.gemm_mxfp4(x.bfloat16(), codes.int(), scales)
    with pytest.raises(ValueError, match="unknown form"):
        W.quantize_packed({}, form="mxfp6")


def test_plain_form_of_the_format():
    """The restatement that the GPU tests hold the kernels to: known values, ties to even, saturation, small and bad blocks."""
    v = torch.zeros(1, 32)
    v[0, :10] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0, 7.9])
    codes, scales = plain.quantize(v)
    assert scales.tolist() == [[127]]
    assert plain.values(codes, scales)[0, :10].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -6.0, 6.0]
    codes, scales = plain.quantize(v * 2.0 ** -7)
    assert scales.tolist() == [[120]] and plain.values(codes, scales)[0, 9] == 6.0 * 2.0 ** -7
    assert plain.quantize(torch.zeros(1, 32))[1].tolist() == [[127]]
    assert plain.quantize(torch.full((1, 32), 2.0 ** -140))[1].tolist() == [[0]]
    v[0, 3] = float("inf")
    codes, scales = plain.quantize(v)
    assert scales.tolist() == [[255]] and torch.isnan(plain.values(codes, scales)).all() and not codes.any()


def test_packed_set_of_four_bits_describes_a_bf16_layer():
    E, H, I = 4, 128, 192
    packed = {"gate_w": torch.zeros(E, H, dtype=torch.bfloat16), "w_up": torch.zeros(E, I, H // 2, dtype=torch.uint8),
              "s_up": torch.zeros(E, I, H // 32, dtype=torch.uint8)}
    cfg = W.mixtral_config(packed, tokens=9)
    assert (cfg.hidden_size, cfg.intermediate_size, cfg.num_experts, cfg.torch_dtype, cfg.tokens) == (H, I, E, api.DTYPE_BF16, 9)
