"""Every kernel of the block-scaled e4m3 products at sizes that end inside its rows and columns.  Which kernel a size takes is asked of the library and
asserted, so that another choice shows as a missing kernel here instead of as one that no test runs."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
from test_gpu_block128 import _check, _layer, _operands, _tables

DEV = "cuda"
BF16 = torch.bfloat16

# (rows, columns, parts) of moe_gemm_block128_plan.  The weight streamer has 16 rows and 16 or 32 columns.
STREAMER = {(16, 16, 8), (16, 32, 2), (16, 32, 4)}
TILES = {(16, 64, 4), (32, 64, 2), (64, 64, 2), (64, 128, 1), (128, 128, 1), (128, 256, 1), (256, 256, 1)}

# M, N, K, the kernel; one matrix
DENSE = [(9, 29, 4096, (16, 16, 8)), (1, 18, 5760, (16, 16, 8)), (10, 16, 7552, (16, 16, 8)), (1, 4096, 14336, (16, 16, 8)), (3, 17314, 2048, (16, 32, 4)),
         (1, 20, 1280, (16, 64, 4)), (1, 16, 1280, (16, 64, 4)), (20, 8555, 640, (32, 64, 2)), (2249, 80, 640, (32, 64, 2)), (43, 8474, 768, (64, 64, 2)),
         (35, 9352, 768, (64, 64, 2)), (1, 16715, 384, (64, 128, 1)), (1, 16840, 384, (64, 128, 1)), (76, 18605, 1792, (128, 128, 1)), (2399, 784, 1664, (128, 128, 1)),
         (215, 16973, 384, (128, 256, 1)), (717, 5744, 384, (128, 256, 1)), (651, 17620, 384, (256, 256, 1)), (2052, 5976, 384, (256, 256, 1))]
# M, N, K, experts, the kernel
EXPERTS = [(1, 128, 4096, 3, (16, 16, 8)), (11, 4352, 1024, 8, (16, 32, 2)), (71, 256, 2048, 70, (16, 32, 4)), (1, 128, 1152, 3, (16, 64, 4)), (1492, 128, 640, 70, (32, 64, 2)),
           (579, 512, 768, 30, (64, 64, 2)), (3, 5760, 384, 3, (64, 128, 1)), (3345, 384, 1664, 70, (128, 128, 1)), (1388, 1792, 384, 30, (128, 256, 1)),
           (1177, 7552, 384, 8, (256, 256, 1))]
# More weights than the memory-side cache holds, one block of rows to a matrix: the other way that weights are fetched.
COLD = 256 << 20
COLD_DENSE = [(2, 33280, 8192, (16, 32, 2)), (3, 16384, 16640, (16, 64, 4)), (33, 49024, 5760, (64, 128, 1)), (125, 27136, 10112, (128, 128, 1)), (114, 48640, 6144, (128, 256, 1)),
              (205, 62976, 4992, (256, 256, 1))]
COLD_EXPERTS = [(23, 11136, 8192, 3, (16, 32, 2)), (65, 6144, 14592, 3, (64, 128, 1)), (172, 9856, 9088, 3, (128, 128, 1))]


def _plan(*a):
    return tuple(moe.gemm_block128_plan(*a).values())


def test_the_sizes_below_take_every_kernel():
    for M, N, K, kernel in DENSE + COLD_DENSE:
        assert _plan(M, N, K) == kernel, (M, N, K)
    for M, N, K, E, kernel in EXPERTS + COLD_EXPERTS:
        assert _plan(M, N, K, E) == kernel, (M, N, K, E)
    assert {s[-1] for s in DENSE} == TILES | {(16, 16, 8), (16, 32, 4)} and {s[-1] for s in EXPERTS} == TILES | STREAMER
    assert all(N * K > COLD and M <= k[0] for M, N, K, k in COLD_DENSE) and all(min(E, M) * N * K > COLD and M <= min(E, M) * k[0] for M, N, K, E, k in COLD_EXPERTS)
    for kernel in TILES:                     # with and without whole 16 bytes at the end of a result's row, both ways that results are stored
        assert {s[1] % 8 == 0 for s in DENSE if s[-1] == kernel} == {False, True}


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,kernel", DENSE + COLD_DENSE)
def test_one_matrix(M, N, K, kernel):
    q, s, w, ws, b = _operands(M, N, K, seed=M + N)
    for bias, act in ((None, api.ACT_NONE), (b, api.ACT_GELU)):
        _check(moe.gemm_block128(q, s, w, ws, bias=bias, act=act), (q, s, w, ws), bias, act)


def _spread(M, E, how):
    """Rows of the experts: evenly, all on one, or drawn; some rows are nobody's."""
    if how == "one":
        return tuple(M if e == E // 2 else 0 for e in range(E))
    if how == "even":
        return tuple(M // E + (e < M % E) for e in range(E))
    g = torch.Generator().manual_seed(M)
    c = torch.bincount(torch.multinomial(torch.rand(E, generator=g) ** 3 + 1e-3, max(1, M - M // 9), replacement=True, generator=g), minlength=E)
    return tuple(c.tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["even", "one", "drawn"])
@pytest.mark.parametrize("M,N,K,E,kernel", EXPERTS + COLD_EXPERTS)
def test_experts(M, N, K, E, kernel, how):
    counts = _spread(M, E, how)
    q, s, w, ws, b = _operands(M, N, K, E, seed=M)
    layer = _layer(M, 1, E, N, K)
    out = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
    layer.expert_gemm_block128(q, s, w, ws, b, *_tables(counts), out=out)
    o = 0
    for e, n in enumerate(counts):
        if n:
            _check(out[o:o + n], (q[o:o + n], s[o:o + n], w[e], ws[e]), b[e], api.ACT_NONE)
        o += n
    assert (out[o:] == 7).all()
