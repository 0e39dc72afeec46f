"""Expert weights held in 4 bits (MXFP4: e2m1 values, one power-of-two scale for 32 of them), and the layer for a few tokens.

Four operators, as a serving program meets them: a matrix is quantised once and can be widened again; a product takes its
weights from the codes, and its rows in bf16 or in 4 bits too; the same product runs over the packed rows of every expert; and
a whole layer answers a batch of a few tokens, on 16-bit weights or on 4-bit ones.  `run` makes these calls of the package
(own = True) or computes the same from elementary operations in 32 bits.  The dimensions are those of the repository's
workloads, at batches from one token to a long prompt, and some that fit no tile.
"""
import math

import torch

own = False

_FLOAT = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_ACT = {"relu": 0, "gelu": 1, "swiglu": 2, "none": 3}


def _quant(name, rows, K, dtype):
    return dict(op="quant", rows=rows, K=K, dtype=dtype, **name)


def _product(name, M, N, K, rows4=False, bias=False, act="none"):
    """rows4: the left operand is held in 4 bits too."""
    return dict(op="product", M=M, N=N, K=K, rows4=rows4, bias=bias, act=act, **name)


def _experts(name, S, k, E, N, K, rows4=False, bias=False, act="none", zipf=False):
    """S tokens, k experts each: S * k packed rows of K values through matrices of N x K."""
    return dict(op="experts", S=S, k=k, E=E, N=N, K=K, rows4=rows4, bias=bias, act=act, zipf=zipf, **name)


def _few(name, S, H, I, E, k, weights, act="swiglu", gate="softmax", norm=True, bias=False, capacity=0.0):
    """weights: "bf16" or "fp16", the layer's own type, or "mxfp4" with bf16 tokens.  capacity: the factor of a layer that drops tokens."""
    return dict(op="few", S=S, H=H, I=I, E=E, k=k, weights=weights, act=act, gate=gate, norm=norm, bias=bias, capacity=capacity, **name)


def listed():
    def named(f, name, *a, **kw):
        return f({"name": name}, *a, **kw)

    return [
        # the rows of one decoding step, quantised in front of a product of two 4-bit operands: a call of a few microseconds
        named(_quant, "quant_step", 64, 7168, "bf16"),
        # one projection of all experts of a large layer, when a checkpoint is brought into 4 bits
        named(_quant, "quant_weights", 8 * 14336, 4096, "bf16"),
        # one token through one matrix
        named(_product, "product_one", 1, 4096, 14336),
        # a batch of decoding sequences, with the bias and the activation
        named(_product, "product_batch", 48, 14336, 4096, bias=True, act="gelu"),
        # a whole prompt, bf16 rows
        named(_product, "product_prompt", 8192, 14336, 4096),
        # both operands in 4 bits: an odd number of rows and dimensions that fit no tile, and the prompt
        named(_product, "both4_ragged", 1777, 2752, 1344, rows4=True, bias=True),
        named(_product, "both4_prompt", 8192, 14336, 4096, rows4=True),
        # a chunk of a prompt on many small experts, about 90 rows in each
        named(_experts, "experts_chunk", 1000, 6, 64, 1408, 2048),
        # a prompt on a few large ones
        named(_experts, "experts_prompt", 8192, 2, 8, 4096, 14336),
        # a single token through a whole layer: two of eight experts' weights, once
        named(_few, "few_one", 1, 4096, 14336, 8, 2, "mxfp4"),
        # a decoding step of 16 sequences on 256 small experts: about a hundred of them are hit
        named(_few, "few_batch", 16, 7168, 2048, 256, 8, "mxfp4", gate="sigmoid"),
        # four sequences on 64 small experts with bf16 weights
        named(_few, "few_bf16", 4, 2048, 1408, 64, 6, "bf16"),
    ]


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""

    def spread(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return n if rng.random() < 0.7 else max(lo, n // 64 * 64)

    def dims(lo, hi, step=64):
        return step * rng.randint(lo // step, hi // step)

    op = rng.choice(("quant", "product", "product", "experts", "few", "few"))
    if op == "quant":
        return _quant({}, spread(1, 65536), dims(256, 7168, 32), rng.choice(("f32", "bf16", "fp16")))
    if op == "product":
        return _product({}, spread(1, 6000), rng.choice((dims(256, 14336), rng.randint(250, 8000))), dims(512, 7168, 32),
                        rows4=rng.random() < 0.4, bias=rng.random() < 0.5, act=rng.choice(("none", "relu", "gelu")))
    if op == "experts":
        E = rng.choice((4, 8, 12, 16, 64))
        wide = E <= 8
        return _experts({}, spread(8, 6000), rng.randint(1, min(E, 6)), E, dims(512, 4096 if wide else 2048), dims(512, 8192 if wide else 2048),
                        rows4=rng.random() < 0.3, bias=rng.random() < 0.3, act=rng.choice(("none", "relu", "gelu")), zipf=rng.random() < 0.4)
    E = rng.choice((4, 8, 16, 64, 128, 256))
    wide = E <= 8
    return _few({}, rng.randint(1, 16), dims(512, 4096), dims(512, 14336 if wide else 2048), E, rng.randint(1, min(E, 8)),
                rng.choice(("mxfp4", "mxfp4", "bf16", "fp16")), act=rng.choice(("relu", "gelu", "swiglu", "swiglu")),
                gate=rng.choice(("softmax", "sigmoid")), norm=rng.random() < 0.7, bias=rng.random() < 0.4,
                capacity=rng.choice((0.0, 0.0, 1.25)))


def _mats(c):
    return ("up", "gate", "down") if c["act"] == "swiglu" else ("up", "down")


# ---- the format, in elementary operations ----

def _scale_bytes(blocks):
    """blocks [..., 32] fp32: the biased exponent of each block's scale, 2^(floor(log2 amax) - 2), and 1 for a block of zeros."""
    amax = blocks.abs().amax(-1)
    e = torch.frexp(amax).exponent.to(torch.int32) - 3          # amax = m * 2^exponent with 0.5 <= m < 1
    return torch.where(amax > 0, (e + 127).clamp(0, 254), torch.full_like(e, 127))


def _power(e):
    """2^e as fp32, e from -127 to 127 (2^-127 is no normal number: a half of 2^-126)."""
    whole = ((e + 127).clamp(min=1) << 23).view(torch.float32)
    return torch.where(e < -126, whole * 0.5, whole)


def _round_e2m1(v):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), with v's sign; as (value, code)."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a.dtype)
    r = (torch.round(a / step) * step).clamp(max=6.0)           # torch.round: halves to even
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r * 0.5 + 4)).to(torch.int32)
    return torch.copysign(r, v), torch.where(torch.signbit(v), code + 8, code)


def _values(x):
    """The values that x [..., K] has in MXFP4, fp32, and what holds them: codes [..., K/2], scales [..., K/32] (bytes)."""
    b = x.float().unflatten(-1, (-1, 32))
    s = _scale_bytes(b)
    up, down = _power((127 - s).clamp(max=127)), _power(s - 127)
    v, code = _round_e2m1(b * up.unsqueeze(-1))
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return (v * down.unsqueeze(-1)).flatten(-2), (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), s.to(torch.uint8)


def _widen(codes, scales):
    """fp32 values of codes [..., K/2] (the low half first) and scales [..., K/32]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    m = (c & 7).float()
    v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, 2 * m - 8))
    v = torch.where(c > 7, -v, v).unflatten(-1, (-1, 32))
    return (v * _power(scales.to(torch.int32) - 127).unsqueeze(-1)).flatten(-2)


def _activate(u, act, g=None):
    if act == "swiglu":
        return g / (1 + torch.exp(-g)) * u
    if act == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return torch.clamp(u, min=0) if act == "relu" else u


# ---- inputs ----

def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def _held4(g, *shape, std):
    """A matrix that was quantised: codes and scales, a slice of the first dimension at a time."""
    parts = [_values(_normal(g, *shape[1:], std=std))[1:] for _ in range(shape[0])]
    return torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])


def _config(c, api):
    few = c["op"] == "few"
    return api.MoEConfig(capacity_factor=(c["capacity"] if few else 0.0) or 1.0, drop_tokens=int(few and c["capacity"] > 0), expert_top_k=c["k"],
                         hidden_act=_ACT[c["act"]] if few else 0, hidden_size=c["H"] if few else c["K"],
                         intermediate_size=c["I"] if few else c["N"], micro_batch=1, num_experts=c["E"], sequence_len=c["S"],
                         torch_dtype=api.DTYPE_FP16 if few and c["weights"] == "fp16" else api.DTYPE_BF16,
                         gate_fn=api.GATE_SIGMOID if few and c["gate"] == "sigmoid" else api.GATE_SOFTMAX,
                         norm_topk_prob=int(few and c["norm"]))


def prepare(case, seed):
    """Rows N(0, 1), every 64th value of a row eight times that (as activations have them); weights N(0, 0.02)."""
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(n, K, dtype=torch.bfloat16):
        x = torch.randn(n, K, generator=g, device="cuda")
        x[:, ::64] *= 8
        return x.to(dtype)

    if c["op"] == "quant":
        return {"case": c, "x": rows(c["rows"], c["K"], _FLOAT[c["dtype"]])}
    st = {"case": c}
    if c["op"] in ("product", "experts"):
        n = c["M"] if c["op"] == "product" else c["S"] * c["k"]
        E = 1 if c["op"] == "product" else c["E"]
        a = rows(n, c["K"])
        st["a"], st["a_scales"] = _values(a)[1:] if c["rows4"] else (a, None)
        st["w"], st["s"] = _held4(g, E, c["N"], c["K"], std=0.02)
        st["bias"] = _normal(g, E, c["N"], std=0.02, dtype=torch.bfloat16) if c["bias"] else None
        if c["op"] == "product":
            st["w"], st["s"] = st["w"][0], st["s"][0]
            st["bias"] = None if st["bias"] is None else st["bias"][0]
            return st
        score = torch.rand(c["S"], E, generator=g, device="cuda").log()         # k distinct experts for every token
        p = (torch.randperm(E, generator=g, device="cuda") + 1.0) ** (-1.1 if c["zipf"] else 0.0)
        chosen = (score / p).topk(c["k"], dim=1).indices.flatten()
        st["count"] = torch.bincount(chosen, minlength=E).to(torch.int32)
        st["offset"] = (torch.cumsum(st["count"], 0) - st["count"]).to(torch.int32)
        st["most"] = int(st["count"].max())
    else:
        dt = _FLOAT["fp16" if c["weights"] == "fp16" else "bf16"]
        st["x"] = rows(c["S"], c["H"], dt)
        w = {"gate_w": _normal(g, c["E"], c["H"], std=0.02, dtype=dt)}
        for m in _mats(c):
            N, K = (c["H"], c["I"]) if m == "down" else (c["I"], c["H"])
            if c["weights"] == "mxfp4":
                w["w_" + m], w["s_" + m] = _held4(g, c["E"], N, K, std=0.02)
            else:
                w["w_" + m] = torch.stack([_normal(g, N, K, std=0.02, dtype=dt) for _ in range(c["E"])])
            if c["bias"]:
                w["b_" + m] = _normal(g, c["E"], N, std=0.02, dtype=dt)
        st["weights"] = w
    if own:
        from cuplayground_amd import api
        st["layer"] = api.MoELayer(_config(c, api))         # the handle and the workspace that a program keeps
    return st


# ---- one pass ----

def _own(st):
    from cuplayground_amd import api
    c = st["case"]
    if c["op"] == "quant":
        return api.dequantize_mxfp4(*api.quantize_mxfp4(st["x"]), dtype=st["x"].dtype)
    if c["op"] == "product":
        return api.gemm_mxfp4(st["a"], st["w"], st["s"], bias=st["bias"], act=_ACT[c["act"]], a_scales=st["a_scales"])
    if c["op"] == "experts":
        return st["layer"].expert_gemm_mxfp4(st["a"], st["w"], st["s"], st["bias"], st["count"], st["offset"], act=_ACT[c["act"]], a_scales=st["a_scales"])
    return st["layer"].forward_few(st["x"], st["weights"])


def _few_plain(st):
    c, w, x = st["case"], st["weights"], st["x"].float()
    S, E, k = c["S"], c["E"], c["k"]
    logits = st["x"].double() @ w["gate_w"].double().t()           # which experts are chosen hangs on small differences
    top, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    idx = idx[:, :k]
    p = torch.softmax(logits, 1).gather(1, idx) if c["gate"] == "softmax" else torch.sigmoid(top[:, :k])
    p = (p / p.sum(1, keepdim=True) if c["norm"] else p).float()
    flat = idx.flatten()
    if c["capacity"]:
        one = (flat.unsqueeze(1) == torch.arange(E, device=flat.device)).to(torch.int32)
        place = ((one.cumsum(0) - one) * one).sum(1)                # earlier pairs of the same expert
        p = p * (place < math.ceil(c["capacity"] * S * k / E)).view(S, k)

    def project(rows, m):
        e = w["w_" + m].index_select(0, flat)
        e = _widen(e, w["s_" + m].index_select(0, flat)) if c["weights"] == "mxfp4" else e.float()
        y = torch.bmm(e, rows.unsqueeze(2)).squeeze(2)
        return y + w["b_" + m].index_select(0, flat).float() if c["bias"] else y

    rows = x.repeat_interleave(k, 0)
    h = _activate(project(rows, "up"), c["act"], project(rows, "gate") if c["act"] == "swiglu" else None)
    y = project(h, "down").view(S, k, -1)
    return (y * p.unsqueeze(2)).sum(1).to(st["x"].dtype)


def _plain(st):
    c = st["case"]
    if c["op"] == "quant":
        return _values(st["x"])[0].to(st["x"].dtype)
    if c["op"] == "few":
        return _few_plain(st)
    a = _widen(st["a"], st["a_scales"]) if c["rows4"] else st["a"].float()
    w = _widen(st["w"], st["s"])
    if c["op"] == "product":
        y = a @ w.t()
        return _activate(y if st["bias"] is None else y + st["bias"].float(), c["act"]).to(torch.bfloat16)
    E, most = c["E"], st["most"]                                    # every expert's rows, padded to the longest
    row = torch.arange(a.shape[0], device=a.device, dtype=torch.int32)
    ends = torch.cumsum(st["count"], 0).to(torch.int32)
    e = torch.searchsorted(ends, row, right=True)
    place = (e * most + row - st["offset"][e]).long()
    padded = torch.zeros(E * most, a.shape[1], device=a.device)
    padded[place] = a
    y = torch.bmm(padded.view(E, most, -1), w.transpose(1, 2).contiguous()).view(E * most, -1)[place]
    return _activate(y if st["bias"] is None else y + st["bias"].float()[e], c["act"]).to(torch.bfloat16)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """The operands and results once each: 17/32 of a byte for a value in 4 bits.  Quantised values are written and read again."""
    c = case
    if c["op"] == "quant":
        n, es = c["rows"] * c["K"], 4 if c["dtype"] == "f32" else 2
        return {"bytes": n * (2.0 * es + 2 * 17 / 32), "flops": 4.0 * n}
    four = 17.0 / 32.0
    if c["op"] == "few":
        hit = c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** c["S"])
        n = len(_mats(c)) * c["H"] * c["I"]
        return {"bytes": hit * n * (four if c["weights"] == "mxfp4" else 2.0) + 2.0 * c["E"] * c["H"] + 4.0 * c["S"] * c["H"],
                "flops": 2.0 * c["S"] * c["k"] * n + 2.0 * c["S"] * c["E"] * c["H"]}
    one = c["op"] == "product"
    n = c["M"] if one else c["S"] * c["k"]
    hit = 1.0 if one else c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** c["S"])
    return {"bytes": hit * c["N"] * c["K"] * four + n * c["K"] * (four if c["rows4"] else 2.0) + 2.0 * n * c["N"], "flops": 2.0 * n * c["N"] * c["K"]}


# ---- the definition in 64 bits, written apart from the above ----

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _widen64(codes, scales):
    grid = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=codes.device)
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    out[..., 0::2] = grid[(codes & 15).int()]
    out[..., 1::2] = grid[(codes >> 4).int()]
    return out * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def _quant64(x):
    """A piece of the rows: nearest by the borders half way between neighbours; a tie goes to the even code."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0 ** -125))) - 2), torch.ones_like(amax))
    a = (b / scale).abs()
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    middle = (grid[:-1] + grid[1:]) / 2
    lower = torch.bucketize(a, middle)                              # borders strictly below a
    tie = (lower < 7) & (a == middle[lower.clamp(max=6)]) & (lower % 2 == 1)
    return (grid[(lower + tie.long()).clamp(max=7)] * scale * torch.sign(b)).flatten(-2)


def exact(case, seed):
    global own
    c, keep = case, own
    own = False
    st = prepare(case, seed)
    own = keep
    if c["op"] == "quant":
        return torch.cat([_quant64(x) for x in st["x"].split(8192)]).to(st["x"].dtype)
    F = torch.nn.functional
    act = {"relu": F.relu, "gelu": F.gelu, "none": lambda v: v}
    if c["op"] != "few":
        a = _widen64(st["a"], st["a_scales"]) if c["rows4"] else st["a"].double()
        if c["op"] == "product":
            bias = 0.0 if st["bias"] is None else st["bias"].double()
            return act[c["act"]](a @ _widen64(st["w"], st["s"]).t() + bias)
        out = torch.zeros(a.shape[0], c["N"], dtype=torch.float64, device=a.device)
        for e, (n, o) in enumerate(zip(st["count"].tolist(), st["offset"].tolist())):
            if n:
                y = a[o:o + n] @ _widen64(st["w"][e], st["s"][e]).t()
                out[o:o + n] = act[c["act"]](y if st["bias"] is None else y + st["bias"][e].double())
        return out
    w, x = st["weights"], st["x"].double()
    logits = x @ w["gate_w"].double().t()
    idx = logits.topk(c["k"], dim=1).indices
    score = torch.softmax(logits, 1) if c["gate"] == "softmax" else torch.sigmoid(logits)
    room = math.ceil(c["capacity"] * c["S"] * c["k"] / c["E"]) if c["capacity"] else c["S"] * c["k"]
    out, took = torch.zeros_like(x), {}
    for t, chosen in enumerate(idx.tolist()):
        total = float(sum(score[t, e] for e in chosen)) if c["norm"] else 1.0
        for e in chosen:
            took.setdefault(e, []).append((t, float(score[t, e]) / total))
    for e, pairs in took.items():
        pairs = pairs[:room]                                        # token by token: the first ones are kept
        rows = x[[t for t, _ in pairs]]

        def project(v, m):
            full = _widen64(w["w_" + m][e], w["s_" + m][e]) if c["weights"] == "mxfp4" else w["w_" + m][e].double()
            y = v @ full.t()
            return y + w["b_" + m][e].double() if c["bias"] else y

        h = project(rows, "up")
        h = F.silu(project(rows, "gate")) * h if c["act"] == "swiglu" else act[c["act"]](h)
        y = project(h, "down")
        for (t, p), row in zip(pairs, y):
            out[t] += p * row
    return out
