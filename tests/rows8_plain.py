"""The formats of the 8-bit operands and the norm, restated in 64 bits: what the tests hold the kernels to."""
import math

import torch

U = 2.0 ** -24                      # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest_half(dtype):
    """Half a step next to zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def norm(x, weight, eps, residual=None):
    """(y, h, r) in 64 bits; h as the rows' type holds it."""
    h = x.double() if residual is None else (x.double() + residual.double()).to(x.dtype).double()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * r * weight.double(), h, r


def norm_backward(dout, h, weight, eps, dsum=None):
    """(dx, dweight, and for either the sum of what its terms are as magnitudes)."""
    h, w, dy = h.double(), weight.double(), dout.double()
    H = h.shape[-1]
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n, dn = h * r, dy * w
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    size = r * (dn.abs() + n.abs() * (dn * n).abs().mean(-1, keepdim=True))
    if dsum is not None:
        dx, size = dx + dsum.double(), size + dsum.double().abs()
    return dx, (dy * n).reshape(-1, H).sum(0), size, (dy * n).abs().reshape(-1, H).sum(0)


def rows8_scales(y):
    amax = y.unflatten(-1, (-1, 128)).abs().amax(-1)
    return torch.where(amax > 0, (amax / 448).clamp(min=2.0 ** -126), torch.ones_like(amax))


def check_rows8(q, scales, y, slack):
    """Codes and scales stand for y (64 bits, itself known to `slack`, relative): half a step of e4m3 -- 2^-4 of the value, or 2^-10 of the scale
    next to zero -- and what y and the scale are off by."""
    want = rows8_scales(y)
    assert ((scales.double() - want).abs() <= want * (slack + 2 * U)).all()
    s = scales.double().repeat_interleave(128, -1)
    got = q.view(torch.float8_e4m3fn).double() * s
    off = (got - y).abs()
    assert (off <= torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) + y.abs() * (slack + 4 * U)).all(), (off / y.abs().clamp(min=1e-300)).max()
    # ... and every code is the nearest of some value that the slack allows: rounding keeps order, so it lies between those of the ends.  (How many differ
    # from the nearest of y itself says little: quotients of products of 8-bit numbers lie exactly half way between two codes now and then.)
    v, d = (y / want.repeat_interleave(128, -1)).abs(), 2 * slack + 8 * U
    code = q.view(torch.float8_e4m3fn).double()
    assert ((code.abs() >= e4m3(v * (1 - d))) & (code.abs() <= e4m3(v * (1 + d))) & (code * y >= 0)).all()


def e4m3(v):
    """The nearest number of e4m3, halves to even, at most 448."""
    step = torch.exp2((torch.frexp(v).exponent.double() - 4).clamp(min=-9))
    return (torch.round(v / step) * step).clamp(-448, 448)


def widen_rows(q, s):
    return q.view(torch.float8_e4m3fn).double() * s.double().repeat_interleave(128, -1)


def widen_blocks(q, s):
    return q.view(torch.float8_e4m3fn).double() * s.double().repeat_interleave(128, -1).repeat_interleave(128, -2)[..., :q.shape[-2], :]


def blocks8(w):
    """w [.., N, K] (fp32) -> uint8 codes and scales [.., ceil(N/128), K/128], a last block of fewer rows with a scale of its own."""
    N, K = w.shape[-2:]
    full = torch.nn.functional.pad(w, (0, 0, 0, -N % 128))
    b = full.unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128))
    amax = b.abs().amax((-1, -3))
    s = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    q = (b / s.unsqueeze(-1).unsqueeze(-3)).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-4, -3).flatten(-2)
    return q[..., :N, :].contiguous(), s


def rows8(x):
    b = x.float().unflatten(-1, (-1, 128))
    amax = b.abs().amax(-1)
    s = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    return (b / s.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2), s


def activate(u, act, g=None):
    from cuplayground_amd import api
    if act == api.ACT_SWIGLU:
        return g / (1 + torch.exp(-g)) * u
    if act == api.ACT_GELU:
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return u.clamp(min=0) if act == api.ACT_RELU else u
