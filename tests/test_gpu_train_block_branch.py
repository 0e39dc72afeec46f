"""The experts' branch of a trainable block by itself: what the block adds to its stream, and what its gradient adds to the stream's, each against its own
size.  (With weights of ordinary size the branch is a fiftieth of the stream, and a comparison of the sums hardly sees it.)"""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api, training
from test_gpu_block128_layer import _config

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype,tol", [(api.DTYPE_F32, 2e-4), (api.DTYPE_BF16, 4e-2)])
@pytest.mark.parametrize("residual", [False, True])
def test_branch_of_a_block(dtype, tol, residual):
    """fp32: sums of 512 terms and the experts' products; bf16: some ten roundings of half a step, 2^-8 each at most, on the way of the branch; and the
    sum's own rounding, half a step of the sum."""
    S, H, I = 200, 256, 384
    cfg = _config(S, H, I, 4, 2, api.ACT_SWIGLU, dtype=dtype)
    block = training.MoE355TrainBlock(cfg, init_std=0.08, seed=3)
    g = torch.Generator(device=DEV).manual_seed(7)
    dt = block.norm_w.dtype
    x = torch.randn(S, H, generator=g, device=DEV).to(dt).requires_grad_()
    res = torch.randn(S, H, generator=g, device=DEV).to(dt).requires_grad_() if residual else None
    d = torch.randn(S, H, generator=g, device=DEV).to(dt)
    out = block(x, res)[0] if residual else block(x)
    dx, *others = torch.autograd.grad(out, [x] + ([res] if residual else []), d)

    with torch.no_grad():
        h = x if res is None else moe.rms_norm(x, block.norm_w, residual=res)[1]
        idx = block.moe.route(moe.rms_norm(h, block.norm_w))[0].long().cpu()
    p = {n: t.detach().double().cpu() for n, t in block.named_parameters()}
    h64 = h.detach().double().cpu().requires_grad_()
    n = h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-6) * p["norm_w"]
    score = torch.softmax(n @ p["moe.gate_w"].t(), 1).gather(1, idx)
    score = score / score.sum(1, keepdim=True)
    y = torch.zeros_like(h64)
    for e in range(4):
        t, j = (idx == e).nonzero(as_tuple=True)
        hid = torch.nn.functional.silu(n[t] @ p["moe.w_gate"][e].t()) * (n[t] @ p["moe.w_up"][e].t())
        y = y.index_add(0, t, score[t, j].unsqueeze(1) * (hid @ p["moe.w_down"][e].t()))
    dy = torch.autograd.grad(y, h64, d.double().cpu())[0]
    y = y.detach()
    stream, dstream = (0.0, 0.0) if residual else (x.detach().double().cpu(), d.double().cpu())
    half = torch.finfo(dt).eps / 2
    for got, base, want in ((out.detach(), stream, y), (dx, dstream, dy)):
        got = got.double().cpu()
        assert want.norm() > 0.3 * S ** 0.5 * H ** 0.5               # the branch is as large as the stream
        assert ((got - base) - want).norm() <= tol * want.norm() + half * got.norm(), float(((got - base) - want).norm() / want.norm())
    for o in others:
        assert torch.equal(o, dx)
