"""MXFP4 in 64 bits, from its definition: borders half way between neighbouring values, ties to the even code."""
import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x):
    """(codes [.., K/2], scales [.., K/32]) of x on its device."""
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b)
    amax = b.abs().amax(-1)
    exponent = torch.frexp(amax).exponent - 1               # amax = m * 2^exponent, 1 <= m < 2
    s = torch.where(amax > 0, (exponent - 2).clamp(min=-127), torch.zeros_like(exponent))
    a = b.abs() / torch.pow(2.0, s.double()).unsqueeze(-1)
    code = torch.zeros_like(a, dtype=torch.int64)
    for c in range(1, 8):                                   # above the border to code c, or on it and c even
        border = (GRID[c - 1] + GRID[c]) / 2
        code += (a > border) | ((a == border) & (c % 2 == 0))
    code = torch.where(torch.signbit(b), code + 8, code)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).flatten(-2).unflatten(-1, (-1, 2))
    scales = torch.where(bad, torch.full_like(s, 255), s + 127)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scales.to(torch.uint8)


def values(codes, scales):
    """fp64 values; NaN where the scale is."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=codes.device)
    v = torch.stack((grid[(codes & 15).long()], grid[(codes >> 4).long()]), -1).flatten(-2).unflatten(-1, (-1, 32))
    s = torch.where(scales == 255, torch.nan, torch.pow(2.0, scales.double() - 127))
    return (v * s.unsqueeze(-1)).flatten(-2)


def activate(u, act):
    """act: MOE_ACT_* without the gated one."""
    return torch.relu(u) if act == 0 else torch.nn.functional.gelu(u) if act == 1 else u


def product_close(got, a, w, bias=None, act=3):
    """got (bf16) against act(a . w^T + bias) in 64 bits.  Of a value: half a unit of bf16 in the last place, 2^-8 of it, and K additions in
    fp32 that are each off by at most 2^-23 of a partial sum, which is at most the sum of the products' magnitudes; an activation (slope at
    most 1.13) carries that on, and GELU's own arithmetic is within 1e-6.  Of all values together: the roundings to bf16 are 2^-8 / sqrt 3 or
    less in the mean square, the sums' errors add up like steps of a random walk: 2^-8 has room for both."""
    K = a.shape[1]
    y = a @ w.t()
    size = a.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias, size + bias.abs()
    want = activate(y, act)
    off = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 1.13 * (K + 2) * 2.0 ** -23 * size + 1e-6
    assert (off <= tol).all(), float((off - tol).max())
    if want.norm() > 0 and want.numel() >= 64:
        assert off.norm() <= 2.0 ** -8 * want.norm() + 1e-6 * want.numel() ** 0.5, float(off.norm() / want.norm())
