"""Rows whose squares' sum, or whose squares themselves, are more than fp32 holds: the norm, its gradient and its form in e4m3 of bf16 and fp32 rows.

Tolerances are those of rows of ordinary size (a power of two in front of a value changes no rounding of it), and for a root above 2^126 that its
reciprocal, below fp32's normal numbers, is off by 2^-150 of 2^-128: 4 U."""
import pytest
import torch

import cuplayground_amd as moe
import rows8_plain as plain
from rows8_plain import U
from test_gpu_norm import SLACK, _close

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
# Values' sizes: the mean of the squares is a number and their sum is none (of four values on); no square is one; all values next to the largest
SIZES = [1e19, 3e37, "largest"]


def _rows(rows, H, dtype, size, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randn(rows, H, generator=g, device=DEV)
    return (torch.where(v > 0, 3.2e38, -3.1e38) if size == "largest" else v * size).to(dtype)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype,H", [(t, H) for t in (BF16, F32) for H in (64, 129, 520, 1000, 2048, 4096, 7168, 8200, 16384)])
def test_norm_and_gradient_of_far_rows(dtype, H, size):
    for rows, residual, w32 in ((5, False, True), (150, True, False)):
        residual = residual and size != "largest"                  # (their sum would be infinite)
        x, res = _rows(rows, H, dtype, size, H), _rows(rows, H, dtype, size, H + 1)
        g = torch.Generator(device=DEV).manual_seed(H + 2)
        w = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(F32 if w32 else dtype)
        dout = torch.randn(rows, H, generator=g, device=DEV).to(dtype)
        y, h, _ = plain.norm(x, w, 1e-6, res if residual else None)
        assert torch.isfinite(h).all() and not torch.isfinite((h.float() ** 2).sum(1)).any()
        got = moe.rms_norm(x, w, 1e-6, residual=res if residual else None)
        if residual:
            got, total = got
            assert torch.equal(total.double(), h)
        _close(got, y, dtype, slack=SLACK + 4 * U)
        ds = (torch.randn(rows, H, generator=g, device=DEV) * 1e-19).to(dtype) if residual else None
        dx, dw = moe.rms_norm_backward(dout, total if residual else x, w, 1e-6, dsum=ds)
        wx, ww, sx, sw = plain.norm_backward(dout, h, w, 1e-6, ds)
        # (r of at most 22 bits times a number of fp32: below its normal numbers the product is rounded to steps of 2^-149)
        off = (dx.double() - wx).abs()
        assert (off <= wx.abs() * plain.half_step(dtype) + plain.smallest_half(dtype) + 2.0 ** -149 + sx * (3 * SLACK + 4 * U) * 1.01).all(), off.max()
        _close(dw, ww, w.dtype, sw, SLACK + (rows / 256 + 74) * U)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype,H", [(t, H) for t in (BF16, F32) for H in (128, 640, 4096, 16384)])
def test_far_rows_to_8_bits(dtype, H, size):
    x = _rows(9, H, dtype, size, H)
    w = (1 + 0.2 * torch.randn(H, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)).to(dtype)
    q, s, out, _ = moe.rms_norm_rows128(x, w, 1e-6, want_rows=True)
    y = plain.norm(x, w, 1e-6)[0]
    plain.check_rows8(q, s, y, SLACK + 4 * U)
    assert torch.equal(out, moe.rms_norm(x, w, 1e-6))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H", [64, 1024, 4104, 16384])
def test_far_rows_among_others(dtype, H):
    """A row's result and gradient depend on nothing but the row, whatever lies beside it: ordinary ones, far ones, zeros, infinities and NaN."""
    x = _rows(12, H, dtype, 1.0, 1)
    x[1::4] = _rows(3, H, dtype, 1e19, 2)
    x[2] = 0
    x[3, H // 2], x[6, 1], x[7, 2] = float("inf"), float("nan"), float("-inf")
    w = torch.ones(H, device=DEV, dtype=dtype)
    dout = _rows(12, H, dtype, 1.0, 3)
    y, dx = moe.rms_norm(x, w), moe.rms_norm_backward(dout, x, w)[0]
    for r in range(12):
        assert torch.equal(y[r:r + 1].nan_to_num(7.0), moe.rms_norm(x[r:r + 1].clone(), w).nan_to_num(7.0))
        assert torch.equal(dx[r:r + 1].nan_to_num(7.0), moe.rms_norm_backward(dout[r:r + 1].clone(), x[r:r + 1].clone(), w)[0].nan_to_num(7.0))
    bad = [3, 6, 7]
    assert torch.isnan(y[bad]).any(1).all() and torch.isnan(dx[bad]).all()
    good = [r for r in range(12) if r not in bad]
    assert torch.isfinite(y[good]).all() and torch.isfinite(dx[good]).all() and y[1::4].abs().max() > 0.5
    assert not y[3, :H // 2].any()                                 # (an infinity's row: r is 0)


@pytest.mark.parametrize("H,v", [(256, 2.0e19), (1, 1.73e19), (256, 1.1e19)])
def test_eps_of_far_rows(H, v):
    """An eps as large as the mean: either may be a number of fp32 where their sum is none."""
    x, w = torch.full((3, H), v, device=DEV), torch.ones(H, device=DEV)
    _close(moe.rms_norm(x, w, 3e38), plain.norm(x, w, 3e38)[0], F32)
    dout = torch.ones(3, H, device=DEV)
    wx, ww, sx, sw = plain.norm_backward(dout, x, w, 3e38)
    dx, dw = moe.rms_norm_backward(dout, x, w, 3e38)
    _close(dx, wx, F32, sx, 3 * SLACK)
    _close(dw, ww, F32, sw, SLACK)
