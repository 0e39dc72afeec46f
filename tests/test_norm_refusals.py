"""What the norm and the activation in e4m3 refuse, on the host: nothing here needs a GPU."""
import ctypes as C

import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api

OK, BAD, UNSUPPORTED, WORKSPACE = 0, 4, 2, 3
P = C.c_void_p(1 << 20)                 # some address, aligned; none of these calls gets as far as reading it
OFF8, OFF2, OFF1 = (C.c_void_p((1 << 20) + n) for n in (8, 2, 1))
BF16, F32, F16 = api.DTYPE_BF16, api.DTYPE_F32, api.DTYPE_FP16
NAN = float("nan")


def test_norm_arguments():
    L = moe.load_library()

    def f(x=P, res=None, w=P, rows=4, H=256, eps=1e-6, dt=BF16, wdt=BF16, total=None, out=P, q=None, s=None):
        return L.moe_rms_norm(x, res, w, rows, H, eps, dt, wdt, total, out, q, s, None)

    for kw in (dict(x=None), dict(w=None), dict(rows=-1), dict(H=0), dict(H=-8), dict(eps=-1e-6), dict(eps=NAN), dict(eps=float("inf")), dict(res=P), dict(total=P),
               dict(out=None), dict(q=P), dict(s=P), dict(q=P, s=P, H=192), dict(x=OFF1), dict(out=OFF1), dict(w=OFF1), dict(dt=F32, wdt=F32, x=OFF2),
               dict(q=P, s=P, x=OFF8), dict(q=P, s=P, out=OFF8), dict(q=P, s=P, w=OFF8), dict(q=P, s=P, res=OFF8, total=P), dict(q=P, s=P, res=P, total=OFF8),
               dict(q=C.c_void_p((1 << 20) + 4), s=P), dict(q=P, s=OFF2), dict(wdt=F32, w=OFF2)):
        assert f(**kw) == BAD, kw
    for kw in (dict(dt=api.DTYPE_TF32), dict(dt=api.DTYPE_FP8, wdt=api.DTYPE_FP8), dict(wdt=F16), dict(dt=F32, wdt=BF16), dict(H=16385), dict(rows=1 << 22),
               dict(rows=1 << 40)):
        assert f(**kw) == UNSUPPORTED, kw
    assert f(rows=0) == OK and f(rows=0, x=None) == OK and f(rows=0, q=P, s=P, out=None, wdt=F32) == OK


def test_gradient_arguments():
    L = moe.load_library()
    n = C.c_size_t(7)
    assert L.moe_rms_norm_scratch_bytes(100, 64, C.byref(n)) == OK and n.value >= 64 * 4
    need = n.value
    for a in ((-1, 64), (4, 0)):
        assert L.moe_rms_norm_scratch_bytes(*a, C.byref(n)) == BAD
    assert L.moe_rms_norm_scratch_bytes(4, 64, None) == BAD and L.moe_rms_norm_scratch_bytes(1 << 22, 64, C.byref(n)) == UNSUPPORTED
    assert L.moe_rms_norm_scratch_bytes(4, 16385, C.byref(n)) == UNSUPPORTED

    def f(dout=P, h=P, w=P, ds=None, rows=100, H=64, eps=1e-6, dt=BF16, wdt=F32, dx=P, dw=P, sc=P, n=need):
        return L.moe_rms_norm_backward(dout, h, w, ds, rows, H, eps, dt, wdt, dx, dw, sc, n, None)

    for kw in (dict(dout=None), dict(h=None), dict(w=None), dict(dx=None), dict(dw=None), dict(rows=-1), dict(H=0), dict(eps=-1.0), dict(dout=OFF1), dict(h=OFF1),
               dict(ds=OFF1), dict(dx=OFF1), dict(dw=OFF2), dict(w=OFF2)):
        assert f(**kw) == BAD, kw
    for kw in (dict(sc=None), dict(n=need - 1), dict(sc=OFF2)):
        assert f(**kw) == WORKSPACE, kw
    for kw in (dict(dt=api.DTYPE_FP8), dict(wdt=F16), dict(H=1 << 15), dict(rows=1 << 22)):
        assert f(**kw) == UNSUPPORTED, kw


def test_activation_arguments():
    L = moe.load_library()

    def f(u=P, g=P, rows=4, I=256, act=api.ACT_SWIGLU, c=None, o=None, E=0, q=P, s=P):
        return L.moe_act_rows128(u, g, rows, I, act, c, o, E, q, s, None)

    for kw in (dict(u=None), dict(g=None), dict(q=None), dict(s=None), dict(rows=-1), dict(I=0), dict(I=64), dict(I=192), dict(act=api.ACT_NONE), dict(act=9),
               dict(act=api.ACT_GELU), dict(c=P, E=2), dict(o=P, E=2), dict(c=P, o=P, E=0), dict(u=OFF8), dict(g=OFF8), dict(q=OFF2), dict(s=OFF2)):
        assert f(**kw) == BAD, kw
    assert f(rows=1 << 40) == UNSUPPORTED and f(rows=1 << 24, I=4096) == UNSUPPORTED
    assert f(rows=0) == OK and f(rows=0, u=None, q=None, s=None) == OK


def test_python_refuses_what_it_can_see():
    """Types, shapes and places are looked at before anything is called: on the CPU every one of these ends in Python."""
    x, w = torch.zeros(4, 256), torch.ones(256)
    for call in (moe.rms_norm, moe.rms_norm_rows128):
        with pytest.raises(ValueError, match="current GPU"):
            call(x, w)
        with pytest.raises(TypeError):
            call(x.double(), w)
        with pytest.raises(TypeError):
            call(x.half(), w.bfloat16())
        with pytest.raises(ValueError, match="shape"):
            call(x, w[:128])
        with pytest.raises(ValueError):
            call(torch.zeros(4, 0), torch.ones(0))
        with pytest.raises(ValueError):
            call(torch.zeros(()), w)
    with pytest.raises(ValueError, match="current GPU"):
        moe.rms_norm_backward(x, x, w)
    with pytest.raises(ValueError, match="multiple of 128"):
        moe.act_rows128(torch.zeros(4, 192, dtype=torch.bfloat16), None, api.ACT_RELU)
    with pytest.raises(ValueError, match="multiple of 128"):
        moe.act_rows128(torch.zeros(256, dtype=torch.bfloat16), None, api.ACT_RELU)
    with pytest.raises(TypeError):
        moe.act_rows128(x, None, api.ACT_RELU)
    with pytest.raises(ValueError, match="current GPU"):
        moe.act_rows128(x.bfloat16(), None, api.ACT_RELU)


def test_product_arguments():
    L = moe.load_library()

    def g(a=P, sa=P, w=P, s=P, bias=None, out=P, M=4, N=64, K=256, act=api.ACT_NONE):
        return L.moe_gemm_block128(a, sa, w, s, bias, out, M, N, K, act, None)

    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(K=64), dict(K=192), dict(a=None), dict(sa=None), dict(w=None), dict(s=None), dict(out=None), dict(act=api.ACT_SWIGLU),
               dict(act=7), dict(a=OFF8), dict(w=OFF8), dict(out=OFF8), dict(sa=OFF2), dict(s=OFF2), dict(bias=OFF1)):
        assert g(**kw) == BAD, kw
    for kw in (dict(N=1 << 22, K=1024), dict(K=1 << 21, N=1), dict(M=1 << 32), dict(M=(1 << 31) - 1, N=1 << 20), dict(N=1 << 40), dict(K=1 << 40)):
        assert g(**kw) == UNSUPPORTED, kw
    assert g(M=0) == OK and g(M=0, a=None, sa=None, out=None) == OK
    n = [C.c_int32(0) for _ in range(3)]
    plan = lambda M, N, K, E: L.moe_gemm_block128_plan(M, N, K, E, *[C.byref(v) for v in n])     # noqa: E731
    assert plan(4, 64, 256, 0) == OK and plan(4, 64, 256, 8) == OK
    assert plan(0, 64, 256, 0) == BAD and plan(4, 64, 200, 0) == BAD and plan(4, 64, 256, -1) == BAD and plan(4, 64, 256, 1000) == BAD
    assert plan(4, 1 << 22, 1024, 0) == UNSUPPORTED and L.moe_gemm_block128_plan(4, 64, 256, 0, None, None, None) == BAD
    assert L.moe_expert_gemm_block128(None, P, P, None, P, P, None, P, P, 128, 128, api.ACT_NONE, P, None) == BAD


def test_python_refuses_products_that_it_can_see():
    a, s = torch.zeros(4, 256, dtype=torch.uint8), torch.ones(4, 2)
    w, ws = torch.zeros(130, 256, dtype=torch.uint8), torch.ones(2, 2)
    with pytest.raises(ValueError, match="matrices"):
        moe.gemm_block128(a[0], s, w, ws)
    for bad in ((a, s[:, :1], w, ws), (a, s, w, ws[:1]), (torch.zeros(256, 4, dtype=torch.uint8).t(), s, w, ws), (a, s, w, ws, torch.zeros(128, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            moe.gemm_block128(*bad)
    with pytest.raises(TypeError):
        moe.gemm_block128(a, s, w.float(), ws)
    with pytest.raises(ValueError, match="contiguous"):
        moe.gemm_block128(a, s, torch.zeros(256, 130, dtype=torch.uint8).t(), ws)
    with pytest.raises(ValueError, match="current GPU"):
        moe.gemm_block128(a, s, w, ws)
