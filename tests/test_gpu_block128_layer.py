"""The e4m3 layer on rows in e4m3 behind its norm, and the trainable block: runs of the operators together, as they are used."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api, training
import rows8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _config(S, H, I, E, k, act, capacity=0.0, dtype=api.DTYPE_FP8, gate_fn=api.GATE_SOFTMAX):
    return moe.MoEConfig(capacity_factor=capacity or 1.0, drop_tokens=int(capacity > 0), expert_top_k=k, hidden_act=act, hidden_size=H, intermediate_size=I,
                         micro_batch=1, num_experts=E, sequence_len=S, torch_dtype=dtype, gate_fn=gate_fn, norm_topk_prob=1)


def _inputs(cfg, seed=0, bias=True):
    S, H, I, E = cfg.tokens, cfg.hidden_size, cfg.intermediate_size, cfg.num_experts
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *shape, std=1.0: (torch.randn(*shape, generator=g, device=DEV) * std).to(BF16)     # noqa: E731
    w = {"gate_w": n(E, H, std=0.05)}
    for name in ("up", "gate", "down") if cfg.hidden_act == api.ACT_SWIGLU else ("up", "down"):
        N, K = (H, I) if name == "down" else (I, H)
        w["w_" + name], w["s_" + name] = moe.quantize_block128(n(E, N, K, std=0.05))
        if bias:
            w["b_" + name] = n(E, N, std=0.1)
    if bias:
        w["gate_bias"] = torch.randn(E, generator=g, device=DEV) * 0.1
    return n(S, H), n(S, H), (1 + 0.1 * n(H).float()).to(BF16), w


def _chain(layer, rows, q, s, w):
    """The layer from its public pieces: the packed rows as copies instead of indices."""
    cfg = layer.cfg
    idx, gate = layer.gate(rows, w["gate_w"], w.get("gate_bias"))
    r = layer.route(idx)
    c, o = r["expert_count"], r["expert_offset"]
    kept = int(c.sum())
    token = r["token_indices"].long().clamp(0, layer.S - 1)
    aq, as_ = q[token].contiguous(), s[token].contiguous()
    u = layer.expert_gemm_block128(aq, as_, w["w_up"], w["s_up"], w.get("b_up"), c, o)
    g = layer.expert_gemm_block128(aq, as_, w["w_gate"], w["s_gate"], w.get("b_gate"), c, o) if cfg.hidden_act == api.ACT_SWIGLU else None
    hq, hs = moe.act_rows128(u[:kept].contiguous(), None if g is None else g[:kept].contiguous(), cfg.hidden_act)
    full_q, full_s = torch.zeros(u.shape[0], u.shape[1], dtype=torch.uint8, device=DEV), torch.zeros(u.shape[0], u.shape[1] // 128, device=DEV)
    full_q[:kept], full_s[:kept] = hq, hs
    y = layer.expert_gemm_block128(full_q, full_s, w["w_down"], w["s_down"], w.get("b_down"), c, o)
    return moe.combine(y, r["pair_row"], gate)


SHAPES = [(1, 256, 128, 4, 2, api.ACT_SWIGLU, 0.0), (5, 512, 384, 8, 3, api.ACT_GELU, 0.0), (16, 1024, 512, 64, 6, api.ACT_SWIGLU, 0.0), (130, 384, 640, 8, 2, api.ACT_RELU, 0.75),
          (700, 768, 1408, 12, 4, api.ACT_SWIGLU, 1.0), (2100, 512, 768, 4, 2, api.ACT_SWIGLU, 0.0)]


@pytest.mark.parametrize("S,H,I,E,k,act,capacity", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_layer_behind_its_norm(S, H, I, E, k, act, capacity, bias):
    cfg = _config(S, H, I, E, k, act, capacity, gate_fn=api.GATE_SIGMOID if S == 16 else api.GATE_SOFTMAX)
    x, res, nw, w = _inputs(cfg, seed=S, bias=bias)
    layer = moe.MoELayer(cfg)
    out, h = layer.forward_block128(x, w, nw, 1e-6, residual=res)
    q, s, rows, total = moe.rms_norm_rows128(x, nw, 1e-6, residual=res, want_rows=True)
    assert torch.equal(h, total) and torch.equal(out, _chain(layer, rows, q, s, w))
    assert torch.equal(layer.forward_block128(x, w, nw), _chain(layer, *[(a[2], a[0], a[1]) for a in [moe.rms_norm_rows128(x, nw, want_rows=True)]][0], w))
    q, s = moe.quantize_rows128(x)
    assert torch.equal(layer.forward_block128(x, w), _chain(layer, x, q, s, w))


@pytest.mark.parametrize("act", [api.ACT_SWIGLU, api.ACT_GELU])
def test_layer_against_64_bits(act):
    """Two roundings to e4m3 on the way of a value, of which none is off by more than 2^-4 of it: on the whole 2 to 3 % each (a step is 2^-4 to 2^-3 of
    what it rounds, evenly filled: 0.29 steps).  SwiGLU multiplies two such projections.  0.043 and 0.037 of the answer; the bound is the largest
    roundings everywhere, sqrt(3) 2^-4."""
    cfg = _config(300, 512, 768, 8, 2, act)
    x, _, nw, w = _inputs(cfg, seed=1, bias=False)
    layer = moe.MoELayer(cfg)
    got = layer.forward_block128(x, w, nw).double()
    rows = moe.rms_norm(x, nw)
    idx, gate = layer.gate(rows, w["gate_w"])
    full = {n: plain.widen_blocks(w["w_" + n], w["s_" + n]) for n in ("up", "gate", "down") if "w_" + n in w}
    v = plain.norm(x, nw, 1e-6)[0]
    want = torch.zeros_like(v)
    for e in range(8):
        t, j = (idx == e).nonzero(as_tuple=True)
        u = v[t] @ full["up"][e].t()
        hh = plain.activate(u, act, v[t] @ full["gate"][e].t() if act == api.ACT_SWIGLU else None)
        want.index_add_(0, t, gate[t, j].double().unsqueeze(1) * (hh @ full["down"][e].t()))
    assert 0.01 < (got - want).norm() / want.norm() < 3 ** 0.5 * 2 ** -4
    # a layer on bf16 rows is as near to 64 bits as its tests say, so this one is as near to it
    assert (got - layer.forward(rows, w).double()).norm() / want.norm() < 3 ** 0.5 * 2 ** -4 + 0.01


def test_layers_replayed():
    """Two layers captured and replayed in turn, on other tokens and with eager calls between: every replay is the eager answer to the bit."""
    cfg = _config(60, 512, 384, 8, 2, api.ACT_SWIGLU)
    x, res, nw, w = _inputs(cfg, seed=5)
    layer, other = moe.MoELayer(cfg), moe.MoELayer(cfg)
    xs = [x, -x, x.roll(1, 0)]
    want = [layer.forward_block128(v, w, nw, residual=res) for v in xs]
    held, graphs, outs = [x.clone(), x.clone()], [], []
    for v, l in zip(held, (layer, other)):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(l.forward_block128(v, w, nw, residual=res))
        graphs.append(g)
    for turn in range(4):
        for i in range(2):
            held[i].copy_(xs[(turn + i) % 3])
            for o in outs[i]:
                o.zero_()
            graphs[i].replay()
        eager = layer.forward_block128(xs[turn % 3], w, nw, residual=res)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 3]))
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[(turn + i) % 3]))


def test_two_streams_at_once():
    cfg = _config(90, 512, 384, 8, 2, api.ACT_SWIGLU)
    x, res, nw, w = _inputs(cfg, seed=6)
    layers = [moe.MoELayer(cfg) for _ in range(2)]           # (a workspace is one call's at a time)
    want = [layers[0].forward_block128(v, w, nw, residual=res) for v in (x, -x)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, v in enumerate((x, -x)):
            with torch.cuda.stream(streams[i]):
                got[i] = layers[i].forward_block128(v, w, nw, residual=res)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---- training ----

@pytest.mark.parametrize("dtype,tol", [(api.DTYPE_F32, 2e-4), (api.DTYPE_BF16, 4e-2)])
@pytest.mark.parametrize("residual", [False, True])
def test_trainable_block(dtype, tol, residual):
    """Gradients of a block in its stream against torch's own on the same routing.  fp32: sums of 512 terms and the experts' products; bf16: some ten
    roundings of half a step on the way of a gradient, 2^-8 each at most, and terms that cancel."""
    cfg = _config(200, 256, 384, 4, 2, api.ACT_SWIGLU, dtype=dtype)
    block = training.MoE355TrainBlock(cfg, seed=3)
    g = torch.Generator(device=DEV).manual_seed(7)
    dt = block.norm_w.dtype
    x = torch.randn(200, 256, generator=g, device=DEV).to(dt).requires_grad_()
    res = torch.randn(200, 256, generator=g, device=DEV).to(dt).requires_grad_() if residual else None
    with torch.no_grad():
        block.norm_w += 0.1 * torch.randn(256, generator=g, device=DEV).to(dt)
    d0, d1 = (torch.randn(200, 256, generator=g, device=DEV).to(dt) for _ in range(2))
    leaves = [x] + ([res] if residual else []) + list(block.parameters())
    out = block(x, res) if residual else (block(x),)
    got = torch.autograd.grad([*out], leaves, [d0, d1][:len(out)])

    # the same in 64 bits on the CPU, on the block's own choice of experts
    with torch.no_grad():
        rows = moe.rms_norm(x if res is None else moe.rms_norm(x, block.norm_w, residual=res)[1], block.norm_w)
        idx = block.moe.route(rows)[0].long().cpu()
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in block.named_parameters()}
    x64, r64 = x.detach().double().cpu().requires_grad_(), None if res is None else res.detach().double().cpu().requires_grad_()
    h = x64 if r64 is None else x64 + r64
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * p["norm_w"]
    score = torch.softmax(n @ p["moe.gate_w"].t(), 1).gather(1, idx)
    score = score / score.sum(1, keepdim=True)
    y = torch.zeros_like(h)
    for e in range(4):
        t, j = (idx == e).nonzero(as_tuple=True)
        hid = torch.nn.functional.silu(n[t] @ p["moe.w_gate"][e].t()) * (n[t] @ p["moe.w_up"][e].t())
        y = y.index_add(0, t, score[t, j].unsqueeze(1) * (hid @ p["moe.w_down"][e].t()))
    out64 = (y, h) if residual else (h + y,)
    for a, b in zip(out, out64):
        assert (a.detach().double().cpu() - b.detach()).norm() <= tol * b.detach().norm()
    l64 = [x64] + ([r64] if residual else []) + [p[n] for n, _ in block.named_parameters()]
    want = torch.autograd.grad(out64, l64, [d0.double().cpu(), d1.double().cpu()][:len(out64)])
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).norm() <= tol * b.norm(), (a.shape, float((a.double().cpu() - b).norm() / b.norm()))


def test_norm_node_gives_what_is_asked():
    g = torch.Generator(device=DEV).manual_seed(2)
    x, res, d0, d1 = (torch.randn(3, 5, 64, generator=g, device=DEV).to(BF16) for _ in range(4))
    w = torch.ones(64, device=DEV, dtype=torch.float32)
    want_dx, want_dw = moe.rms_norm_backward(d0, moe.rms_norm(x, w, residual=res)[1], w, dsum=d1)
    a, b, c = x.clone().requires_grad_(), res.clone().requires_grad_(), w.clone().requires_grad_()
    y, h = training.rms_norm(a, c, residual=b)
    torch.autograd.backward([y, h], [d0, d1])
    assert torch.equal(a.grad, want_dx) and torch.equal(b.grad, want_dx) and torch.equal(c.grad, want_dw) and a.grad.data_ptr() != b.grad.data_ptr()
    y, h = training.rms_norm(a, w, residual=res)                       # the stream alone goes on
    assert torch.equal(torch.autograd.grad(h, a, d1)[0], d1)
    y = training.rms_norm(a, c)
    dx, dw = torch.autograd.grad(y, [a, c], d0)
    want = moe.rms_norm_backward(d0, x, w)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    y = training.rms_norm(a.transpose(0, 1), c)                        # not in one piece: copies, gradients in the caller's shape
    dx = torch.autograd.grad(y, a, d0.transpose(0, 1))[0]
    assert torch.equal(dx, want[0])
    y = training.rms_norm(a, c)
    with pytest.raises(RuntimeError):                                  # no second derivatives
        (gx,) = torch.autograd.grad(y, a, d0, create_graph=True)
        gx.sum().backward()


def test_training_step_replayed():
    """A whole step of the block captured (its earlier graphs gone), replayed on other tokens: every replay is the eager step."""
    cfg = _config(128, 256, 384, 4, 2, api.ACT_SWIGLU, dtype=api.DTYPE_BF16)
    block = training.MoE355TrainBlock(cfg, seed=4)
    g = torch.Generator(device=DEV).manual_seed(1)
    xs = [torch.randn(128, 256, generator=g, device=DEV).to(BF16) for _ in range(3)]
    d = torch.randn(128, 256, generator=g, device=DEV).to(BF16)
    params = list(block.parameters())

    def step(x):
        x = x.detach().requires_grad_()
        out = block(x)
        grads = torch.autograd.grad(out, [x, *params], d)
        return [out.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(x) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    held = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(held)
    for i in (1, 2, 0, 1):
        held.copy_(xs[i])
        graph.replay()
        eager = step(xs[i])
        torch.cuda.synchronize()
        for a, b, c in zip(got, want[i], eager):
            assert torch.equal(a, b) and torch.equal(c, b)
