"""MXFP4 on the GPU: quantisation and its inverse to the bit, products against 64 bits."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import mxfp4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _same_quantised(x):
    codes, scales = moe.quantize_mxfp4(x)
    want_codes, want_scales = plain.quantize(x.cpu())
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu(), want_codes)
    return codes, scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 7, 160), (64, 7168), (257, 2080), (0, 64)])
def test_quantise_is_the_definition(shape, dtype):
    g = _gen(shape[-1])
    x = torch.randn(*shape, generator=g, device=DEV) * torch.exp2(torch.randint(-12, 13, (*shape[:-1], shape[-1]), generator=g, device=DEV).float() / 3)
    codes, scales = _same_quantised(x.to(dtype))
    assert codes.shape == (*shape[:-1], shape[-1] // 2) and scales.shape == (*shape[:-1], shape[-1] // 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantise_borders_and_ends_of_the_range(dtype):
    top = torch.finfo(dtype)
    rows = []
    for e in (-140, -130, -127, -126, -125, -24, -14, -3, 0, 7, 13, 125):
        s = 2.0 ** e
        # every border, every value, their neighbours, under a largest magnitude that keeps the scale at s
        v = [0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.5, 1.0, 1.5, 2.0, 3.0]
        v = v + [-x for x in v]
        rows.append(torch.tensor(v, dtype=torch.float64) * s)
        rows.append(torch.tensor(v, dtype=torch.float64) * s * (1 + 2.0 ** -7))
        rows.append(torch.tensor(v, dtype=torch.float64) * s * (1 - 2.0 ** -8))
    rows.append(torch.zeros(32, dtype=torch.float64))
    rows.append(-torch.zeros(32, dtype=torch.float64))
    x = torch.stack(rows).clamp(-top.max, top.max).to(dtype)
    extra = torch.zeros(6, 32, dtype=dtype)
    extra[0, 5], extra[1, 31], extra[2, 0] = float("inf"), float("-inf"), float("nan")
    extra[3, 7], extra[4, 1] = top.max, top.smallest_normal
    extra[5, 2] = top.tiny * top.eps                         # the smallest subnormal
    _same_quantised(torch.cat([x, extra]).to(DEV))


def test_quantise_takes_views():
    x = torch.randn(64, 256, generator=_gen(3), device=DEV)
    _same_quantised(x[:, 64:192])                            # rows further apart than they are long
    _same_quantised(x.t().contiguous().t()[:, :96])          # the other order
    flat = torch.randn(33 * 32 + 1, generator=_gen(4), device=DEV).bfloat16()
    _same_quantised(flat[1:].view(33, 32))                   # not on 16 bytes
    _same_quantised(x[:1].expand(5, 256))                    # one row, five times


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequantise_every_code_under_every_scale(dtype):
    """Every byte of codes with every scale but the three whose largest values overflow bf16 before fp32's rounding would say so."""
    codes = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(1, 256, 16).expand(256, 256, 16).contiguous()
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 256, 1).contiguous()
    got = moe.dequantize_mxfp4(codes.to(DEV), scales.to(DEV), dtype=dtype).cpu()
    want = plain.values(codes, scales).float().to(dtype)     # the values are exact in fp32 as far as it reaches
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float(), nan=0.0), torch.nan_to_num(want.float(), nan=0.0))


def test_dequantise_inverts_and_defaults_to_bf16():
    x = torch.randn(7, 96, generator=_gen(5), device=DEV).bfloat16()
    codes, scales = moe.quantize_mxfp4(x)
    y = moe.dequantize_mxfp4(codes, scales)
    assert y.dtype == torch.bfloat16
    again = moe.quantize_mxfp4(y)                            # what is held is held again (6 stays the largest of its block or 4 does)
    assert torch.equal(moe.dequantize_mxfp4(*again), y)
    assert moe.dequantize_mxfp4(codes[:0], scales[:0]).shape == (0, 96)
    odd = torch.cat([codes.flatten()[:1], codes.flatten()])[1:].view(7, 48)
    assert torch.equal(moe.dequantize_mxfp4(odd, scales), y)


def _held(g, *shape, std=0.05):
    codes, scales = moe.quantize_mxfp4(torch.randn(*shape, generator=g, device=DEV) * std)
    return codes, scales, plain.values(codes, scales)


def _rows(g, M, K, rows4):
    a = torch.randn(M, K, generator=g, device=DEV)
    a[:, ::37] *= 8
    a = a.bfloat16()
    if not rows4:
        return a, None, a.double()
    codes, scales = moe.quantize_mxfp4(a)
    return codes, scales, plain.values(codes, scales)


@pytest.mark.parametrize("rows4", [False, True])
@pytest.mark.parametrize("N,K", [(16, 32), (1, 64), (100, 96), (33, 1344), (72, 160), (512, 512), (260, 2080), (1030, 7168 + 32)])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 129, 300])
def test_product(M, N, K, rows4):
    g = _gen(M * 7 + N + K)
    a, sa, av = _rows(g, M, K, rows4)
    w, s, wv = _held(g, N, K)
    act = (3, 0, 1)[(M + N) % 3]
    bias = torch.randn(N, generator=g, device=DEV).bfloat16() if (M + K) % 2 else None
    got = moe.gemm_mxfp4(a, w, s, bias=bias, act=act, a_scales=sa)
    assert got.shape == (M, N) and got.dtype == torch.bfloat16
    plain.product_close(got, av, wv, None if bias is None else bias.double(), act)


@pytest.mark.parametrize("rows4", [False, True])
@pytest.mark.parametrize("M,N,K", [(3000, 4096, 544), (4096, 4100, 256), (1, 20000, 640), (40, 9000, 4096), (257, 14336, 128)])
def test_product_large(M, N, K, rows4):
    g = _gen(M + N)
    a, sa, av = _rows(g, M, K, rows4)
    w, s, wv = _held(g, N, K)
    plain.product_close(moe.gemm_mxfp4(a, w, s, a_scales=sa), av, wv)


@pytest.mark.parametrize("rows4", [False, True])
@pytest.mark.parametrize("M,N,K", [
    (34, 8587, 32), (94, 8045, 448), (409, 6995, 160), (726, 6321, 352), (328, 8325, 544), (1358, 8901, 672), (227, 8262, 576), (584, 6660, 1056),
    (1154, 6865, 800), (1, 33001, 1056), (13, 33010, 1056), (2, 323, 4128), (14, 186, 3936), (491, 222, 4032), (1, 3, 4032), (982, 150, 1312),
    (1358, 8904, 672), (1154, 6872, 800), (1, 33001, 8192), (3, 65540, 4096)])
def test_product_at_odd_sizes_of_every_kernel(M, N, K, rows4):
    """The sizes reach every tile and cut of the streamer, and end inside their rows, columns and slabs."""
    g = _gen(M + N + K)
    a, sa, av = _rows(g, M, K, rows4)
    w, s, wv = _held(g, N, K)
    bias = torch.randn(N, generator=g, device=DEV).bfloat16()
    plain.product_close(moe.gemm_mxfp4(a, w, s, bias, act=api.ACT_GELU, a_scales=sa), av, wv, bias.double(), 1)


@pytest.mark.parametrize("rows4", [False, True])
@pytest.mark.parametrize("M", [5, 40, 200])
def test_product_keeps_what_is_not_finite_where_it_is(M, rows4):
    """A row that holds a NaN or an infinity, a column whose scale is NaN: no other row or column sees them, at the end of a cut-off row
    (K is no multiple of any step) as elsewhere."""
    N, K = 70, 352
    g = _gen(M)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    x[1, K - 1], x[M - 1, 3] = float("nan"), float("inf")
    a, sa = moe.quantize_mxfp4(x) if rows4 else (x, None)
    w, s, wv = _held(g, N, K)
    s[9, K // 32 - 1] = 255
    wv = plain.values(w, s)
    got = moe.gemm_mxfp4(a, w, s, a_scales=sa)
    fine_rows = [r for r in range(M) if r not in (1, M - 1)]
    fine_cols = [c for c in range(N) if c != 9]
    av = plain.values(a, sa) if rows4 else x.double()
    plain.product_close(got[fine_rows][:, fine_cols], av[fine_rows], wv[fine_cols])
    assert torch.isnan(got[:, 9]).all() and torch.isnan(got[1]).all()
    assert not torch.isfinite(got[M - 1]).any()
    if not rows4:                                            # an infinity times finite weights: an infinity, or a NaN where the weight is zero
        want = torch.where(wv[:, 3] == 0, torch.nan, torch.sign(wv[:, 3]) * torch.inf)
        cols = torch.tensor(fine_cols, device=DEV)
        assert torch.equal(torch.isnan(got[M - 1, cols]), torch.isnan(want[cols]))


def test_product_of_no_rows_and_of_a_strided_left_operand():
    g = _gen(9)
    w, s, wv = _held(g, 64, 128)
    assert moe.gemm_mxfp4(torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), w, s).shape == (0, 64)
    wide = torch.randn(20, 256, generator=g, device=DEV).bfloat16()
    plain.product_close(moe.gemm_mxfp4(wide[:, 128:], w, s), wide[:, 128:].double(), wv)


def _layer(S, k, E, N, K, **kw):
    return moe.MoELayer(moe.MoEConfig(expert_top_k=k, hidden_size=K, intermediate_size=N, micro_batch=1, num_experts=E, sequence_len=S,
                                      torch_dtype=api.DTYPE_BF16, norm_topk_prob=0, **kw))


@pytest.mark.parametrize("rows4", [False, True])
@pytest.mark.parametrize("counts,N,K", [
    ((3, 0, 1, 12), 64, 128), ((16, 17, 0, 31), 192, 320), ((0, 0, 64, 0), 128, 64), ((128, 1, 127, 0, 129, 300), 192, 192),
    ((700, 20, 0, 300, 4), 256, 448), ((90,) * 16, 320, 256), ((600, 511, 257, 0), 3200, 128), ((2, 1) * 40, 64, 576)])
def test_expert_product(counts, N, K, rows4):
    """Rows of every expert through its matrix; the last rows belong to no expert and stay as they were."""
    E, left = len(counts), 2
    A = sum(counts) + left
    g = _gen(A + N)
    layer = _layer(A, 1, E, N, K)
    a, sa, av = _rows(g, A, K, rows4)
    w, s, wv = _held(g, E, N, K)
    bias = torch.randn(E, N, generator=g, device=DEV).bfloat16()
    count = torch.tensor(counts, dtype=torch.int32, device=DEV)
    offset = (torch.cumsum(count, 0) - count).to(torch.int32)
    out = torch.full((A, N), 7.0, dtype=torch.bfloat16, device=DEV)
    got = layer.expert_gemm_mxfp4(a, w, s, bias, count, offset, act=api.ACT_GELU, a_scales=sa, out=out)
    assert got is out and bool((out[A - left:] == 7.0).all())
    at = 0
    for e, n in enumerate(counts):
        if n:
            plain.product_close(out[at:at + n], av[at:at + n], wv[e], bias[e].double(), 1)
        at += n


@pytest.mark.parametrize("rows4", [False, True])
@pytest.mark.parametrize("A,E,N,K", [(1, 3, 1088, 64), (3, 3, 64, 64), (34, 30, 2240, 960), (726, 30, 448, 320), (422, 8, 1536, 256), (733, 30, 2176, 64),
                                     (2132, 8, 1920, 384), (2253, 30, 832, 704), (1470, 30, 1920, 1088), (1987, 8, 1600, 640), (2428, 8, 2496, 1024)])
def test_expert_product_of_every_kernel(A, E, N, K, rows4):
    """As above, with as many rows an expert as chance gives it; behind a gap in front of the last expert's."""
    g = _gen(A + N + K)
    layer = _layer(A, 1, E, N, K)
    a, sa, av = _rows(g, A, K, rows4)
    w, s, wv = _held(g, E, N, K)
    of = torch.randint(0, E + 1, (A,), generator=g, device=DEV)              # E: nobody's, the gap
    count = torch.bincount(of, minlength=E + 1).to(torch.int32)
    gap, count = int(count[E]), count[:E].contiguous()
    offset = (torch.cumsum(count, 0) - count).to(torch.int32)
    offset[E - 1] += gap
    out = torch.full((A, N), 7.0, dtype=torch.bfloat16, device=DEV)
    layer.expert_gemm_mxfp4(a, w, s, None, count, offset, act=api.ACT_NONE, a_scales=sa, out=out)
    left = torch.ones(A, dtype=torch.bool, device=DEV)
    for e, (at, n) in enumerate(zip(offset.tolist(), count.tolist())):
        if n:
            plain.product_close(out[at:at + n], av[at:at + n], wv[e])
        left[at:at + n] = False
    assert bool((out[left] == 7.0).all())


def test_products_are_the_same_every_time_on_any_stream_and_in_a_graph():
    g = _gen(11)
    w, s, _ = _held(g, 1000, 1024)
    xs = [torch.randn(m, 1024, generator=g, device=DEV).bfloat16() for m in (1, 40, 700)]
    x4 = moe.quantize_mxfp4(xs[2])
    want = [moe.gemm_mxfp4(x, w, s) for x in xs] + [moe.gemm_mxfp4(x4[0], w, s, a_scales=x4[1])]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = [moe.gemm_mxfp4(x, w, s) for x in xs]
    here = [moe.gemm_mxfp4(x, w, s) for x in xs]             # at the same time, on two streams
    torch.cuda.synchronize()
    for a, b, c in zip(want, there, here):
        assert torch.equal(a, b) and torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = moe.quantize_mxfp4(xs[2])
        out = [moe.gemm_mxfp4(x, w, s) for x in xs] + [moe.gemm_mxfp4(q[0], w, s, a_scales=q[1])]
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        moe.gemm_mxfp4(xs[1], w, s)
        torch.cuda.synchronize()
        for a, b in zip(want, out):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows4", [False, True])
def test_products_whose_offsets_pass_32_bits(rows4):
    """More than 4 GiB of rows, of results, and of experts' weights: the last of each."""
    g = _gen(7)
    for M, N, K in ((560000, 32, 16384) if rows4 else (280000, 32, 8192), (160000, 14336, 64)):
        w, s, wv = _held(g, N, K)
        a, sa, av = _rows(g, 300, K, rows4)
        big = torch.zeros(M, a.shape[1], dtype=a.dtype, device=DEV)
        big[-300:] = a
        if rows4:
            bs = torch.full((M, K // 32), 127, dtype=torch.uint8, device=DEV)
            bs[-300:] = sa
        out = moe.gemm_mxfp4(big, w, s, a_scales=bs if rows4 else None)
        plain.product_close(out[-300:], av, wv)
        assert not out[:-300].any()
        del out, big
    E, H, I, n = 150, 4096, 14336, 40
    layer = _layer(n, 1, E, I, H)
    w1, s1, wv = _held(g, I, H)
    w = torch.zeros(E, I, H // 2, dtype=torch.uint8, device=DEV)
    s = torch.zeros(E, I, H // 32, dtype=torch.uint8, device=DEV)
    w[-1], s[-1] = w1, s1
    count = torch.zeros(E, dtype=torch.int32, device=DEV)
    for rows in (3, n):
        count[-1] = rows
        a, sa, av = _rows(g, n, H, rows4)
        out = layer.expert_gemm_mxfp4(a, w, s, None, count, torch.zeros_like(count), a_scales=sa)
        plain.product_close(out[:rows], av[:rows], wv)
