"""The layer for a few tokens: against 64 bits, and its routing against the general path's to the bit."""
import math

import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import mxfp4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROUTING = ("topk_idx", "topk_w", "slot", "expert_count", "expert_offset")


def _config(S, H, I, E, k, act, dtype=api.DTYPE_BF16, gate=api.GATE_SOFTMAX, norm=1, capacity=0.0):
    return moe.MoEConfig(capacity_factor=capacity or 1.0, drop_tokens=int(capacity > 0), expert_top_k=k, hidden_act=act, hidden_size=H, intermediate_size=I,
                         micro_batch=1, num_experts=E, sequence_len=S, torch_dtype=dtype, gate_fn=gate, norm_topk_prob=norm)


def _inputs(cfg, weights, bias, seed, gate_bias=False):
    """(x, the layer's tensors, its expert matrices in 64 bits)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = torch.float16 if cfg.torch_dtype == api.DTYPE_FP16 else torch.bfloat16
    S, H, I, E = cfg.tokens, cfg.hidden_size, cfg.intermediate_size, cfg.num_experts

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * std

    w, exact = {"gate_w": normal(E, H, std=0.05).to(dt)}, {}
    if gate_bias:
        w["gate_bias"] = normal(E)
    for m in ("up", "down") + (("gate",) if cfg.hidden_act == api.ACT_SWIGLU else ()):
        N, K = (H, I) if m == "down" else (I, H)
        full = normal(E, N, K, std=K ** -0.5)
        if weights == "mxfp4":
            w["w_" + m], w["s_" + m] = moe.quantize_mxfp4(full)
            exact[m] = plain.values(w["w_" + m], w["s_" + m])
        else:
            w["w_" + m] = full.to(dt)
            exact[m] = w["w_" + m].double()
        if bias:
            w["b_" + m] = normal(E, N, std=0.3).to(dt)
    return normal(S, H).to(dt), w, exact


def _close(got, x, cfg, w, exact, idx, wts, slot):
    """The layer in 64 bits with the routing that the call reported.  Of a value: the rounding of the output and that of the intermediate
    (half a unit in the last place of each, eps / 2), the latter weighted as the down projection weights it; what the fp32 sums and gate
    weights add is smaller by their 2^-24 and H + I + k terms.  Of all values together: two roundings of eps / 2 each at most."""
    F = torch.nn.functional
    half = torch.finfo(x.dtype).eps / 2
    xd = x.double()
    want, room = torch.zeros_like(xd), torch.zeros_like(xd)
    for t in range(cfg.tokens):
        for r in range(cfg.expert_top_k):
            if slot[t, r] < 0:
                continue
            e, p = int(idx[t, r]), wts[t, r].double()

            def project(v, m):
                y = exact[m][e] @ v
                return y + w["b_" + m][e].double() if "b_" + m in w else y

            u = project(xd[t], "up")
            h = F.silu(project(xd[t], "gate")) * u if cfg.hidden_act == api.ACT_SWIGLU else plain.activate(u, cfg.hidden_act)
            want[t] += p * project(h, "down")
            room[t] += p * (exact["down"][e].abs() @ (h.abs() + 1e-3))
    off = (got.double() - want).abs()
    sums = (cfg.hidden_size + cfg.intermediate_size) * 2.0 ** -23
    tol = half * want.abs() + (half + 4 * sums) * 1.02 * room + 1e-6
    assert (off <= tol).all(), float((off - tol).max())
    assert off.norm() <= 2 * half * want.norm() + 1e-5 * want.numel() ** 0.5, float(off.norm() / want.norm())


def _check(cfg, weights, bias, seed, gate_bias=False):
    x, w, exact = _inputs(cfg, weights, bias, seed, gate_bias)
    layer = moe.MoELayer(cfg)
    routing = layer.new_routing()
    got = layer.forward_few(x, w, routing=routing)
    # the general path routes the same tokens: its gate and its slots
    idx, wts = layer.gate(x, w["gate_w"], w.get("gate_bias"))
    r = layer.route(idx)
    want = dict(r, topk_idx=idx, topk_w=wts)
    for key in ROUTING:
        assert torch.equal(routing[key], want[key]), key
    kept = int(want["expert_count"].sum())
    assert torch.equal(routing["token_indices"][:kept], want["token_indices"][:kept]) and bool((routing["token_indices"][kept:] == -1).all())
    _close(got, x, cfg, w, exact, idx.cpu(), wts.cpu(), r["slot"].cpu())
    return layer, x, w, got


KINDS = [("mxfp4", api.DTYPE_BF16), ("own", api.DTYPE_BF16), ("own", api.DTYPE_FP16)]


@pytest.mark.parametrize("weights,dtype", KINDS)
@pytest.mark.parametrize("S,H,I,E,k,act,gate,norm,capacity,bias", [
    (1, 64, 64, 1, 1, api.ACT_RELU, api.GATE_SOFTMAX, 0, 0.0, False),
    (1, 512, 1024, 8, 2, api.ACT_SWIGLU, api.GATE_SOFTMAX, 1, 0.0, False),
    (1, 2048, 192, 4, 4, api.ACT_GELU, api.GATE_SIGMOID, 0, 0.0, True),
    (2, 448, 320, 300, 5, api.ACT_SWIGLU, api.GATE_SIGMOID, 1, 0.0, True),
    (5, 256, 832, 16, 3, api.ACT_GELU, api.GATE_SOFTMAX, 1, 1.0, True),
    (7, 1344, 448, 12, 3, api.ACT_RELU, api.GATE_SOFTMAX, 1, 0.0, True),
    (9, 1024, 512, 64, 8, api.ACT_SWIGLU, api.GATE_SOFTMAX, 0, 1.25, False),
    (16, 576, 576, 128, 16, api.ACT_SWIGLU, api.GATE_SIGMOID, 1, 0.0, False),
    (16, 512, 256, 2, 2, api.ACT_GELU, api.GATE_SOFTMAX, 1, 0.5, True),
    (16, 256, 2112, 512, 8, api.ACT_SWIGLU, api.GATE_SOFTMAX, 1, 1.0, True),
])
def test_few(S, H, I, E, k, act, gate, norm, capacity, bias, weights, dtype):
    _check(_config(S, H, I, E, k, act, dtype, gate, norm, capacity), weights, bias, seed=S + E + k, gate_bias=E % 3 == 0)


@pytest.mark.parametrize("weights", ["mxfp4", "own"])
def test_few_where_all_tokens_choose_the_same_experts(weights):
    """Sixteen rows in two experts, the others hit by none; and with room for three rows an expert, tokens that lose every pair."""
    for capacity in (0.0, 0.75):
        cfg = _config(16, 256, 320, 8, 2, api.ACT_SWIGLU, capacity=capacity)
        x, w, exact = _inputs(cfg, weights, True, seed=5)
        w["gate_bias"] = torch.tensor([0, 0, 60.0, 0, 0, 50.0, 0, 0], device=DEV)
        layer = moe.MoELayer(cfg)
        routing = layer.new_routing()
        got = layer.forward_few(x, w, routing=routing)
        assert torch.equal(routing["topk_idx"], torch.tensor([[2, 5]] * 16, dtype=torch.int32, device=DEV))
        room = 16 if not capacity else math.ceil(0.75 * 32 / 8)
        assert int(routing["expert_count"][2]) == room and int(routing["expert_count"].sum()) == 2 * room
        _close(got, x, cfg, w, exact, routing["topk_idx"].cpu(), routing["topk_w"].cpu(), routing["slot"].cpu())
        assert bool((got[room:] == 0).all())


@pytest.mark.parametrize("weights,dtype", KINDS)
def test_few_against_the_general_path(weights, dtype):
    """The same layer by moe_forward (on the widened weights): rounded once more, an expert's rows, so three roundings apart at most."""
    cfg = _config(16, 512, 768, 16, 4, api.ACT_SWIGLU, dtype)
    layer, x, w, got = _check(cfg, weights, False, seed=3)
    if weights == "mxfp4":
        w = {n: moe.dequantize_mxfp4(t, w["s_" + n[2:]]) if n[:2] == "w_" else t for n, t in w.items() if n[:2] != "s_"}
    want = layer.forward(x, w)
    half = torch.finfo(x.dtype).eps / 2
    assert (got.double() - want.double()).norm() <= 5 * half * want.double().norm()


def test_few_keeps_a_token_that_is_not_finite_to_itself():
    cfg = _config(6, 320, 192, 16, 2, api.ACT_SWIGLU)
    x, w, exact = _inputs(cfg, "mxfp4", False, seed=8)
    layer = moe.MoELayer(cfg)
    clean = layer.forward_few(x, w)
    x[2, 319], x[4, 0] = float("nan"), float("inf")
    got = layer.forward_few(x, w)
    others = [0, 1, 3, 5]
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[4]).all()
    assert torch.isfinite(got[others]).all()
    # the others' experts and sums are what they were; which experts are hit may shift the order of the down projection's sums
    assert (got[others].double() - clean[others].double()).norm() <= 2.0 ** -8 * clean[others].double().norm()


@pytest.mark.parametrize("weights", ["mxfp4", "own"])
def test_few_repeats_in_a_graph_and_on_another_stream(weights):
    cfg = _config(4, 512, 1408, 64, 6, api.ACT_SWIGLU)
    x, w, _ = _inputs(cfg, weights, False, seed=2)
    layer, other = moe.MoELayer(cfg), moe.MoELayer(cfg)
    xs = [x, -x, x.roll(1, 0)]
    want = [layer.forward_few(v, w) for v in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                             # two handles, two workspaces, at the same time
        there = [other.forward_few(v, w) for v in xs]
    here = [layer.forward_few(v, w) for v in xs]
    torch.cuda.synchronize()
    for a, b, c in zip(want, there, here):
        assert torch.equal(a, b) and torch.equal(a, c)
    held, out = x.clone(), torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward_few(held, w, out=out)
    for v, y in zip(xs * 2, want * 2):
        held.copy_(v)
        graph.replay()
        other.forward_few(xs[1], w)
        torch.cuda.synchronize()
        assert torch.equal(out, y)


def test_mxfp4_layer_from_a_checkpoint_to_its_answers(tmp_path):
    """Expert matrices packed, quantised, saved and loaded; a prompt by the stages, a decoding step by the few-token launches, and the
    torch operator over both."""
    from cuplayground_amd import torch_op, weights as W
    E, H, I, k = 8, 256, 384, 2
    g = torch.Generator().manual_seed(1)

    def mats(n, r, c):
        return [torch.randn(r, c, generator=g) * c ** -0.5 for _ in range(n)]

    packed = W.pack_experts(torch.randn(E, H, generator=g) * 0.1, mats(E, I, H), mats(E, H, I), mats(E, I, H), device=DEV)
    held = W.quantize_packed(packed, form="mxfp4")
    exact = {m: plain.values(held["w_" + m], held["s_" + m]) for m in ("up", "gate", "down")}
    for tokens in (3, 70):
        cfg = W.mixtral_config(held, tokens=tokens, top_k=k)
        assert (cfg.hidden_size, cfg.intermediate_size, cfg.torch_dtype) == (H, I, api.DTYPE_BF16)
        path = str(tmp_path / ("layer%d.safetensors" % tokens))
        W.save_packed(path, held, cfg)
        loaded, cfg = W.load_packed(path)
        x = torch.randn(tokens, H, generator=g).to(DEV).bfloat16()
        layer = moe.MoELayer(cfg)
        got = layer.forward_mxfp4(x, loaded)
        idx, wts = layer.gate(x, loaded["gate_w"])
        slot = layer.route(idx)["slot"]
        if tokens <= api.FEW_TOKENS:
            _close(got, x, cfg, loaded, exact, idx.cpu(), wts.cpu(), slot.cpu())
        # the general path on the widened weights: at most three roundings of each apart (the projections', the intermediate's, the rows')
        wide = {n: moe.dequantize_mxfp4(t, loaded["s_" + n[2:]]) if n[:2] == "w_" else t for n, t in loaded.items() if n[:2] != "s_"}
        want = layer.forward(x, wide)
        assert (got.double() - want.double()).norm() <= 6 * 2.0 ** -8 * want.double().norm()
        module = torch_op.MoE355.from_packed(cfg, loaded)
        assert torch.equal(module(x), got)


@pytest.mark.parametrize("weights", ["mxfp4", "own"])
@pytest.mark.parametrize("S,H,I,E,k", [(16, 2048, 64, 2, 2), (16, 4096, 128, 3, 2), (13, 4096, 64, 2, 1), (16, 8192, 192, 5, 2), (16, 192, 4160, 4, 3), (8, 2048, 832, 64, 8)])
def test_few_with_many_rows_an_expert(S, H, I, E, k, weights):
    """Experts of nine rows and more, where wavefronts share a contraction, and where half of them work; workgroups that share columns."""
    cfg = _config(S, H, I, E, k, api.ACT_SWIGLU)
    x, w, exact = _inputs(cfg, weights, True, seed=S + H + I)
    layer = moe.MoELayer(cfg)
    routing = layer.new_routing()
    got = layer.forward_few(x, w, routing=routing)
    torch.cuda.synchronize()
    _close(got, x, cfg, w, exact, routing["topk_idx"].cpu(), routing["topk_w"].cpu(), routing["slot"].cpu())


@pytest.mark.parametrize("E,k", [(8, 3), (64, 6), (200, 8), (512, 16)])
def test_selection_among_equal_and_infinite_logits(E, k):
    """The order of selection: the larger logit, the lower index among equal ones (0 and -0 are), a NaN like -inf; k distinct experts always."""
    cfg = _config(3, 64, 64, E, k, api.ACT_RELU, gate=api.GATE_SIGMOID)
    _, w, _ = _inputs(cfg, "own", False, seed=E)
    layer = moe.MoELayer(cfg)
    x = torch.zeros(3, 64, device=DEV, dtype=torch.bfloat16)
    inf, nan = math.inf, math.nan
    rows = [[0.0] * E, [-inf] * E, [nan] * E, [nan, -inf] * (E // 2), [(-1) ** e * 0.0 for e in range(E)], [float(e % 5) for e in range(E)],
            [inf if e % 7 == 3 else nan if e % 3 == 0 else -float(e) for e in range(E)], [-inf if e < E - 2 else -3.0 for e in range(E)],
            [-3.0e38 if e % 2 else 1e-45 for e in range(E)]]
    for row in rows:
        keys = [-inf if math.isnan(v) else v for v in row]
        want = sorted(range(E), key=lambda e: (-keys[e], e))[:k]
        w["gate_bias"] = torch.tensor(row, device=DEV)                  # the products of a row of zeros are zeros: these are the logits
        idx, wts = layer.gate(x, w["gate_w"], w["gate_bias"])
        routing = layer.new_routing()
        layer.forward_few(x, w, routing=routing)
        assert idx.tolist() == [want] * 3 and routing["topk_idx"].tolist() == [want] * 3, row[:8]
        assert torch.equal(torch.isnan(wts), torch.isnan(routing["topk_w"]))
        assert torch.equal(wts.nan_to_num(7.0), routing["topk_w"].nan_to_num(7.0))


def test_layer_refusals():
    """Operands of another kind are refused before anything is launched, for a few tokens and for many."""
    for S in (4, 40):
        cfg = _config(S, 64, 64, 4, 2, api.ACT_SWIGLU)
        x, w, _ = _inputs(cfg, "mxfp4", True, seed=S)
        layer = moe.MoELayer(cfg)
        layer.forward_mxfp4(x, w)
        own = _inputs(cfg, "own", True, seed=S)[1]
        with pytest.raises(TypeError):
            layer.forward_mxfp4(x, own)
        with pytest.raises(TypeError):
            layer.forward_mxfp4(x.float(), w)
        for bad in ({"w_up": own["w_up"]}, {"gate_bias": torch.zeros(4, device=DEV, dtype=torch.bfloat16)}, {"b_down": own["b_down"].float()}):
            with pytest.raises(TypeError):
                layer.forward_mxfp4(x, {**w, **bad})
        for bad in ({"extra": x}, {"s_gate": w["s_gate"][:, :32]}, {"w_down": w["w_down"].cpu()}, {"b_up": own["b_up"][:2]}):
            with pytest.raises(ValueError):
                layer.forward_mxfp4(x, {**w, **bad})
        for name in ("gate_w", "w_gate", "s_down", "s_gate", "w_down"):
            with pytest.raises((ValueError, moe.MoEError)):
                layer.forward_mxfp4(x, {n: t for n, t in w.items() if n != name})
    with pytest.raises(moe.MoEError):
        layer.forward_few(x, w)                       # 40 tokens
    few = moe.MoELayer(_config(4, 64, 64, 4, 2, api.ACT_SWIGLU))
    odd = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, 64)
    with pytest.raises(moe.MoEError):
        few.forward_few(x[:4].contiguous(), {**w, "b_down": odd})          # a bias that is not 8-byte aligned
    count = torch.full((4,), 20, dtype=torch.int32, device=DEV)
    offset = (torch.cumsum(count, 0) - count).int()
    rows = torch.zeros(80, 64, dtype=torch.bfloat16, device=DEV)
    for bad in ((rows, w["w_up"][0], w["s_up"]), (rows[:79], w["w_up"], w["s_up"]), (rows, w["w_up"], w["s_up"][:, :, :1])):
        with pytest.raises(ValueError):
            layer.expert_gemm_mxfp4(*bad, None, count, offset)
    with pytest.raises(moe.MoEError):
        layer.expert_gemm_mxfp4(rows, w["w_up"], w["s_up"], None, count, offset, act=api.ACT_SWIGLU)


def test_few_beyond_4_gib_of_weights():
    """The last of 150 experts of 29 MB a matrix; the others' weights are zeros under scales of 2^-127."""
    E, H, I = 150, 4096, 14336
    cfg = _config(2, H, I, E, 1, api.ACT_RELU)
    one, w1, exact = _inputs(_config(2, H, I, 1, 1, api.ACT_RELU), "mxfp4", False, seed=3)
    w = {"gate_w": torch.zeros(E, H, dtype=torch.bfloat16, device=DEV), "gate_bias": torch.arange(E, dtype=torch.float32, device=DEV)}
    for n in ("w_up", "s_up", "w_down", "s_down"):
        w[n] = torch.zeros(E, *w1[n].shape[1:], dtype=torch.uint8, device=DEV)
        w[n][-1] = w1[n][0]
    layer = moe.MoELayer(cfg)
    routing = layer.new_routing()
    got = layer.forward_few(one, w, routing=routing)
    assert routing["topk_idx"].tolist() == [[E - 1]] * 2
    _close(got, one, cfg, w, {m: {E - 1: exact[m][0]} for m in exact}, routing["topk_idx"].cpu(), routing["topk_w"].cpu(), routing["slot"].cpu())


@pytest.mark.parametrize("act,gate,norm,capacity", [(api.ACT_GELU, api.GATE_SIGMOID, 1, 1.0), (api.ACT_SWIGLU, api.GATE_SOFTMAX, 0, 0.75), (api.ACT_RELU, api.GATE_SOFTMAX, 1, 0.0)])
@pytest.mark.parametrize("S", [11, 17, 130])
def test_mxfp4_layer_with_drops_and_biases(S, act, gate, norm, capacity):
    """forward_mxfp4 on both sides of the few tokens, against the layer in 64 bits with the routing of the general path: its bf16 rows, and the
    stages' roundings of projections and experts' rows, are at most five of half a unit each, weighted as the sums weight them."""
    F = torch.nn.functional
    cfg = _config(S, 320, 448, 12, 3, act, gate=gate, norm=norm, capacity=capacity)
    x, w, exact = _inputs(cfg, "mxfp4", True, seed=S + act, gate_bias=True)
    layer = moe.MoELayer(cfg)
    got = layer.forward_mxfp4(x, w)
    idx, wts = layer.gate(x, w["gate_w"], w["gate_bias"])
    slot = layer.route(idx)["slot"]
    if capacity:
        assert int((slot < 0).sum()) > 0
    want = torch.zeros(S, 320, dtype=torch.float64, device=DEV)
    for t in range(S):
        for r in range(3):
            if slot[t, r] >= 0:
                e = int(idx[t, r])
                u = exact["up"][e] @ x[t].double() + w["b_up"][e].double()
                h = F.silu(exact["gate"][e] @ x[t].double() + w["b_gate"][e].double()) * u if act == api.ACT_SWIGLU else plain.activate(u, act)
                want[t] += wts[t, r].double() * (exact["down"][e] @ h + w["b_down"][e].double())
    assert (got.double() - want).norm() <= 5 * 2.0 ** -8 * want.norm()
    lost = (slot < 0).all(1)
    assert not got[lost].any()
