"""Rows whose places pass 31 and 32 bits, and operands that begin anywhere that their elements can: the norm, its gradient, the activation in e4m3 and
the products of e4m3 rows.  All rows but a few are zeros; those lie at both ends and around each power of two."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import rows8_plain as plain
from test_gpu_block128 import _check, _layer, _operands, _tables
from test_gpu_norm import SLACK, _close

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _far(rows, width, size=2):
    """Rows at both ends and around the places of 2^31 and 2^32 elements and bytes."""
    at = {0, 1, rows - 2, rows - 1}
    for place in (1 << 31, 1 << 32):
        for r in (place // width, place // size // width):
            at |= {r - 1, r, r + 1}
    return torch.tensor(sorted(r for r in at if 0 <= r < rows), device=DEV)


def _sparse(rows, width, at, seed, dtype=BF16, std=1.0):
    x = torch.zeros(rows, width, dtype=dtype, device=DEV)
    x[at] = (torch.randn(len(at), width, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * std).to(dtype)
    return x


def test_norm_of_far_rows():
    R, H, eps = 1_050_000, 4096, 1e-6
    at = _far(R, H)
    x, res = _sparse(R, H, at, 1), _sparse(R, H, at, 2)
    w = (1 + 0.2 * torch.randn(H, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)).to(BF16)
    q, s, out, h = moe.rms_norm_rows128(x, w, eps, residual=res, want_rows=True)
    y, total, _ = plain.norm(x[at], w, eps, res[at])
    assert torch.equal(h[at].double(), total)
    _close(out[at], y, BF16)
    plain.check_rows8(q[at], s[at], y, SLACK)
    assert not out[at[0] + 2:at[0] + 500].any() and not q[at[-1] - 500:at[-1] - 1].any()
    del q, s, out, res
    dout, ds = _sparse(R, H, at, 4), _sparse(R, H, at, 5)
    dx, dw = moe.rms_norm_backward(dout, h, w, eps, dsum=ds)
    h_at, dout_at, ds_at = h[at], dout[at], ds[at]
    small = moe.rms_norm_backward(dout_at, h_at, w, eps, dsum=ds_at)
    assert torch.equal(dx[at], small[0])                       # a row's gradient depends on nothing but the row
    _, want, _, size = plain.norm_backward(dout_at, h_at, w, eps, ds_at)
    _close(dw, want, BF16, size)
    assert not dx[at[0] + 2:at[0] + 500].any()


def test_activation_of_far_rows():
    R, I = 300_100, 14336
    at = _far(R, I)
    u, g = _sparse(R, I, at, 1), _sparse(R, I, at, 2)
    q, s = moe.act_rows128(u, g, api.ACT_SWIGLU)
    small = moe.act_rows128(u[at], g[at], api.ACT_SWIGLU)
    assert torch.equal(q[at], small[0]) and torch.equal(s[at], small[1])
    assert not q[at[0] + 2:at[0] + 500].any() and (s[at[0] + 2:at[0] + 500] == 1).all()


@pytest.mark.parametrize("experts", [0, 2])
def test_products_of_far_rows(experts):
    M, N, K = 2_200_000, 2048, 2048
    at = _far(M, N)
    few = _operands(len(at), N, K, experts, seed=9)
    q = torch.zeros(M, K, dtype=torch.uint8, device=DEV)
    s = torch.ones(M, K // 128, device=DEV)
    q[at], s[at] = few[0], few[1]
    if not experts:
        out = moe.gemm_block128(q, s, few[2], few[3], bias=few[4])
        _check(out[at], few[:4], few[4], api.ACT_NONE)
        return
    last = 3                                                   # the last rows are another expert's
    out = _layer(M, 1, experts, N, K).expert_gemm_block128(q, s, few[2], few[3], few[4], *_tables((M - last, last)))
    for e, r in enumerate((slice(0, len(at) - 2), slice(len(at) - 2, len(at)))):
        _check(out[at[r]], (few[0][r], few[1][r], few[2][e], few[3][e]), few[4][e], api.ACT_NONE)


@pytest.mark.parametrize("M,N,K", [(1, 1000, 4096), (3, 1000, 4096), (20, 333, 640), (100, 2752, 384), (513, 2049, 640), (2100, 4100, 384)])
def test_products_of_scales_and_biases_at_any_address(M, N, K):
    q, s, w, ws, b = _operands(M, N, K, seed=3)

    def moved(t):
        big = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
        big[1:] = t.flatten()
        return big[1:].view(t.shape)

    want = moe.gemm_block128(q, s, w, ws, bias=b)
    got = moe.gemm_block128(q.view(torch.float8_e4m3fn), moved(s), w.view(torch.float8_e4m3fn), moved(ws), bias=moved(b))
    assert torch.equal(got, want)
    with pytest.raises(Exception):
        moe.gemm_block128(moved(q), s, w, ws)
