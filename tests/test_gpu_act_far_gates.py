"""SwiGLU to e4m3 at gates where the sigmoid leaves fp32's normal numbers, and its error at ordinary ones, which grows with a negative gate.

Tolerance, U = 2^-24: the exponential's argument, |g| log2 e + 2, is rounded once and its constant is off by 0.45 U: (1.45 |g| + 1.4) U of e^-g, which for
a positive gate is e^-g / (1 + e^-g) of that, below 1 U + 0.7 U.  Then exp2 and the reciprocal, 2 U each, the sum and three products: 8 U."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import rows8_plain as plain
from rows8_plain import U

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _check(u, g):
    q, s = moe.act_rows128(u, g, api.ACT_SWIGLU)
    y = plain.activate(u.double(), api.ACT_SWIGLU, g.double())
    slack = torch.where(g < 0, 1.45 * g.double().abs() + 1.4, 2.0) * U + 8 * U
    want = plain.rows8_scales(y)
    assert ((s.double() - want).abs() <= want * (slack.unflatten(-1, (-1, 128)).amax(-1) + 2 * U)).all()
    v, d = (y / want.repeat_interleave(128, -1)).abs(), 2 * slack.unflatten(-1, (-1, 128)).amax(-1).repeat_interleave(128, -1) + 8 * U
    code = q.view(torch.float8_e4m3fn).double()
    assert ((code.abs() >= plain.e4m3(v * (1 - d))) & (code.abs() <= plain.e4m3(v * (1 + d))) & (code * y >= 0)).all()
    return q, s


@pytest.mark.parametrize("size", [1.0, -3.0, 1000.0, 1e30])
@pytest.mark.parametrize("gate", [-60.0, -80.0, -87.0, -87.5, -88.0, -88.5])
def test_far_gates(gate, size):
    """A piece of nothing but such gates, whose scale is as small as their results."""
    u = (torch.linspace(0.5, 1.0, 256, device=DEV) * size).to(BF16).view(1, 256)
    q, s = _check(u, torch.full((1, 256), gate, device=DEV, dtype=BF16))
    assert (q.view(torch.float8_e4m3fn).float() != 0).all() or (gate < -87 and abs(size) <= 3)      # (below half a step of the least scale)


def test_gates_behind_the_exponentials_end():
    """Below -88.72 the result is 0, whatever lies beside it."""
    u, g = torch.ones(2, 128, device=DEV, dtype=BF16), torch.zeros(2, 128, device=DEV, dtype=BF16)
    g[0, :7] = torch.tensor([-3.0e38, -1e20, -1000.0, -200.0, -128.0, -100.0, -90.0]).to(BF16).to(DEV)
    g[1] = g[0, torch.arange(128, device=DEV) % 7]
    q, s = moe.act_rows128(u, g, api.ACT_SWIGLU)
    assert (plain.widen_rows(q, s)[0, :7] == 0).all() and (plain.widen_rows(q, s)[1] == 0).all() and (s == 1).all()


@pytest.mark.parametrize("std", [0.01, 1.0, 6.0, 30.0])
def test_ordinary_gates(std):
    gen = torch.Generator(device=DEV).manual_seed(int(std * 100))
    u = torch.randn(200, 1408, generator=gen, device=DEV).to(BF16)
    _check(u, (torch.randn(200, 1408, generator=gen, device=DEV) * std).clamp(min=-88).to(BF16))


def test_small_and_large_gates():
    """bf16's least numbers and its largest ones keep their bits: the quarters are exact."""
    g = torch.tensor([2.0 ** -133, -2.0 ** -133, 2.0 ** -126, -1.5 * 2.0 ** -125, 1e-30, 3e38, 1e38, 500.0], device=DEV).to(BF16).repeat(16).view(1, 128)
    u = torch.tensor([2.0 ** 120], device=DEV).to(BF16).expand(1, 128).contiguous()
    small = g.abs() < 1
    _check(torch.where(small, u, 0), g)
    _check(torch.where(small, 0, torch.ones_like(u)), g)
