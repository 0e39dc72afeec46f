"""Every kernel of the MXFP4 products at sizes that end inside its rows, columns and slabs.  Which kernel a size takes is asked of the
library and asserted, so that another choice shows as a missing kernel here instead of as one that no test runs."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import mxfp4_plain as plain

DEV = "cuda"

# (rows, columns, parts) of moe_gemm_mxfp4_plan.  The weight streamer has 16 rows and 16 or 32 columns (1, 2, 4 or 8 wavefronts a contraction).
STREAMER = {(16, 16, 1), (16, 16, 2), (16, 16, 4), (16, 16, 8), (16, 32, 1)}
TILES16 = {(16, 64, 2), (32, 64, 2), (48, 64, 2), (64, 64, 2), (64, 128, 1), (96, 128, 1), (128, 128, 1), (256, 256, 1)}
TILES4 = {(32, 64, 4), (32, 64, 2), (64, 64, 2), (64, 128, 1), (128, 128, 1), (128, 256, 1), (256, 256, 1)}

# M, N, K, the kernel; one matrix
DENSE16 = [(1, 16775, 1952, (16, 16, 1)), (1, 14336, 4096, (16, 16, 2)), (4, 15473, 13088, (16, 16, 2)), (1, 17, 2336, (16, 16, 4)), (1, 17, 3904, (16, 16, 8)),
           (10, 67602, 3008, (16, 32, 1)), (13, 6001, 2336, (16, 64, 2)), (70, 2001, 3040, (16, 64, 2)), (77, 4099, 1120, (32, 64, 2)), (130, 4001, 2080, (48, 64, 2)),
           (64, 9001, 608, (64, 64, 2)), (95, 14001, 608, (64, 128, 1)), (1956, 14745, 160, (96, 128, 1)), (327, 8854, 544, (128, 128, 1)),
           (2050, 14001, 416, (256, 256, 1)), (2905, 14752, 544, (256, 256, 1))]
DENSE4 = [(15, 17, 32, (64, 128, 1)), (1, 28612, 7264, (16, 16, 1)), (15, 15454, 13664, (16, 16, 2)), (11, 4999, 3552, (16, 16, 4)), (14, 1003, 4032, (16, 16, 8)),
          (10, 67602, 3008, (16, 32, 1)), (21, 3077, 5440, (32, 64, 4)), (77, 4099, 1120, (32, 64, 2)), (130, 4001, 2080, (64, 64, 2)), (99, 7003, 352, (64, 128, 1)),
          (327, 8854, 544, (128, 128, 1)), (1000, 6003, 608, (128, 256, 1)), (1999, 8003, 416, (256, 256, 1)), (1999, 8008, 416, (256, 256, 1))]
# M, N, K, experts, the kernel
EXPERTS16 = [(31, 576, 1856, 30, (16, 16, 1)), (10, 1216, 4032, 8, (16, 16, 2)), (94, 128, 5824, 70, (16, 16, 2)), (9, 128, 2880, 3, (16, 16, 4)),
             (9, 64, 3904, 3, (16, 16, 8)), (275, 960, 960, 70, (16, 32, 1)), (11, 4096, 10048, 8, (16, 32, 2)), (55, 128, 7232, 3, (16, 64, 2)),
             (350, 2112, 576, 8, (32, 64, 2)), (250, 1408, 1088, 8, (48, 64, 2)), (300, 2048, 576, 8, (64, 64, 2)),
             (800, 1408, 1088, 8, (64, 128, 1)), (6462, 960, 192, 3, (96, 128, 1)), (900, 3200, 576, 3, (128, 128, 1)),
             (12345, 1984, 576, 4, (256, 256, 1))]
EXPERTS4 = [(46, 1088, 6208, 30, (16, 16, 1)), (27, 1984, 12736, 8, (16, 16, 2)), (9, 128, 2880, 3, (16, 16, 4)), (9, 64, 3904, 3, (16, 16, 8)),
            (68, 3520, 1920, 30, (16, 32, 1)), (32, 4096, 10048, 8, (16, 32, 2)), (62, 64, 6080, 3, (32, 64, 4)), (275, 960, 960, 70, (32, 64, 2)),
            (300, 2048, 576, 8, (64, 64, 2)), (400, 1984, 576, 8, (64, 128, 1)), (900, 3200, 576, 3, (128, 128, 1)),
            (4481, 1344, 192, 5, (128, 256, 1)), (12345, 1984, 576, 4, (256, 256, 1))]
# More weights than the memory-side cache holds: the streamer's other loads.
COLD = 256 << 20
COLD_DENSE = [(3, 65540, 8224, (16, 32, 1)), (3, 32700, 16480, (16, 16, 1))]
COLD_EXPERTS = [(30, 2048, 9216, 30, (16, 32, 1)), (8, 4096, 33024, 4, (16, 16, 2))]


def _plan(*a, **kw):
    return tuple(moe.gemm_mxfp4_plan(*a, **kw).values())


def test_the_sizes_below_take_every_kernel():
    for sizes, rows4, tiles in ((DENSE16, False, TILES16), (DENSE4, True, TILES4)):
        for M, N, K, kernel in sizes + COLD_DENSE:
            assert _plan(M, N, K, rows4=rows4) == kernel, (M, N, K)
        assert {s[-1] for s in sizes} == STREAMER | tiles
    for sizes, rows4, tiles in ((EXPERTS16, False, TILES16), (EXPERTS4, True, TILES4)):
        for M, N, K, E, kernel in sizes + COLD_EXPERTS:
            assert _plan(M, N, K, E, rows4=rows4) == kernel, (M, N, K, E)
        assert {s[-1] for s in sizes} == STREAMER | tiles | {(16, 32, 2)}
    assert all(N * K // 2 > COLD for _, N, K, _ in COLD_DENSE) and all(E * N * K // 2 > COLD for _, N, K, E, _ in COLD_EXPERTS)
    for sizes in (DENSE16, DENSE4):          # with and without whole 16 bytes at the end of a result's row, both ways that results are stored
        assert {s[1] % 8 == 0 for s in sizes if s[-1] == (256, 256, 1)} == {False, True}


def test_the_plan_of_a_product():
    assert _plan(1, 1, 32) == _plan(5, 7, 32) == _plan(1, 1024, 64, rows4=True) == (1, 1, 1)      # fewer than eight scales
    for a, status in (((0, 64, 64), 4), ((4, 0, 64), 4), ((4, 64, 48), 4), ((4, 64, 64, -1), 4), ((4, 64, 64, 513), 4), ((1 << 31, 64, 64), 2),
                      ((4, 1 << 40, 64), 2), ((4, 1 << 23, 1024), 2), ((4, 64, (1 << 20) + 32), 2), (((1 << 31) - 1, 1 << 20, 64), 2)):
        with pytest.raises(moe.MoEError) as e:
            moe.gemm_mxfp4_plan(*a)
        assert e.value.status == status, a


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(g, M, K, rows4):
    a = torch.randn(M, K, generator=g, device=DEV)
    a[:, ::37] *= 8
    a = a.bfloat16()
    if not rows4:
        return a, None, a.double()
    codes, scales = moe.quantize_mxfp4(a)
    return codes, scales, plain.values(codes, scales)


def _weights(g, *shape):
    return moe.quantize_mxfp4(torch.randn(*shape, generator=g, device=DEV) * 0.05)


def _dense(M, N, K, rows4):
    g = _gen(M + N + K)
    a, sa, av = _rows(g, M, K, rows4)
    w, s = _weights(g, N, K)
    bias = torch.randn(N, generator=g, device=DEV).bfloat16()
    got = moe.gemm_mxfp4(a, w, s, bias, act=api.ACT_GELU, a_scales=sa)
    plain.product_close(got, av, plain.values(w, s), bias.double(), 1)


def _counts(g, M, E):
    """Uneven, some of them none, with a row or more for nobody at the end; of many rows, whole blocks of 256, and remainders of one row,
    of 128 and on both sides of them."""
    if M > 10000:
        count = torch.tensor([256 * 16 + 1, 256 * 9 + 128, 256 * 11 + 129, 0], dtype=torch.int32)
        count[3] = M - int(count.sum()) - 3
        return count.to(DEV)
    p = torch.rand(E + 1, generator=g, device=DEV) ** 2
    p[E] = p[:E].mean() / 8
    if E > 2:
        p[int(torch.randint(0, E, (1,), generator=g, device=DEV))] = 0
    of = torch.multinomial(p, M - 1, replacement=True, generator=g)
    return torch.bincount(of, minlength=E + 1)[:E].to(torch.int32)


def _experts(M, N, K, E, rows4):
    g = _gen(M + N + K)
    count = _counts(g, M, E)
    offset = (torch.cumsum(count, 0) - count).to(torch.int32)
    a, sa, av = _rows(g, M, K, rows4)
    w, s = _weights(g, E, N, K)
    bias = torch.randn(E, N, generator=g, device=DEV).bfloat16()
    H, I = sorted((N, K))          # of a layer that has such a product
    layer = moe.MoELayer(moe.MoEConfig(expert_top_k=1, hidden_size=H, intermediate_size=I, micro_batch=1, num_experts=E, sequence_len=M, torch_dtype=api.DTYPE_BF16))
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=DEV)
    layer.expert_gemm_mxfp4(a, w, s, bias, count, offset, act=api.ACT_GELU, a_scales=sa, out=out)
    ends = 0
    for e, (at, n) in enumerate(zip(offset.tolist(), count.tolist())):
        if n:
            plain.product_close(out[at:at + n], av[at:at + n], plain.values(w[e], s[e]), bias[e].double(), 1)
        ends = at + n
    assert ends < M and bool((out[ends:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,rows4", [(*s[:3], False) for s in DENSE16] + [(*s[:3], True) for s in DENSE4])
def test_every_kernel_on_one_matrix(M, N, K, rows4):
    _dense(M, N, K, rows4)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,E,rows4", [(*s[:4], False) for s in EXPERTS16] + [(*s[:4], True) for s in EXPERTS4])
def test_every_kernel_on_experts(M, N, K, E, rows4):
    _experts(M, N, K, E, rows4)


@pytest.mark.gpu
@pytest.mark.parametrize("rows4", [False, True])
def test_streamers_of_weights_that_no_cache_holds(rows4):
    for M, N, K, _ in COLD_DENSE:
        _dense(M, N, K, rows4)
    for M, N, K, E, _ in COLD_EXPERTS:
        _experts(M, N, K, E, rows4)
