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


# The last round of the largest tiles (256 compute units, 32 of a share) in smaller ones: blocks of 256 rows in halves; what is left of up to 128 rows in
# pieces of 64 x 128, where no block is beside it, or as a tile of its own.  M, N, K.
LAST = [(2100, 8187, 384), (2148, 8136, 384), (2052, 8192, 512), (2148, 17617, 384), (2100, 5977, 384), (2204, 8190, 384), (2344, 8192, 384), (2177, 5976, 384),
        (20564, 1000, 384), (2304, 8187, 512)]
# rows of 70 experts (all rows are 40000), with remainders in both parts of the table, one behind another, and of one row: pieces; halves and tiles; tiles
SOME = {3: 612, 4: 576, 5: 577, 20: 1, 21: 0, 22: 128, 23: 129, 63: 640, 64: 520, 66: 0, 67: 612, 69: 64}
PIECES = tuple(SOME.get(e, 512 if e < 65 else 256) for e in range(70))
HALVES = tuple(SOME.get(e, 512 if e < 69 else 300) for e in range(70))
TILES_LEFT = tuple(257 + e % 128 if e % 3 else 700 for e in range(70))


def _last(counts, N):
    """(halves, pieces, tiles of what is left) of these row counts."""
    ncol = (N + 255) // 256
    share = -(-sum((n + 127) // 256 for n in counts) * ncol // 8)
    left = [n % 256 for n in counts if 0 < n % 256 <= 128]
    high = sum(1 if n <= 64 else 2 for n in left)
    if share % 32 == 0 and 2 * high * ncol <= 256:
        return 0, 2 * high * ncol, 0
    rest, tiles = share % 32, len(left) * ncol
    return (rest if 2 * rest + -(-tiles // 8) <= 32 else 0), 0, tiles


def test_the_sizes_below_end_in_every_way():
    assert all(_plan(M, N, K) == (256, 256, 1) for M, N, K in LAST) and _plan(40000, 512, 384, 70) == (256, 256, 1)
    assert {tuple(v > 0 for v in _last((M,), N)) for M, N, K in LAST} >= {(False, True, False), (False, False, True), (True, False, True), (True, False, False)}
    assert [tuple(v > 0 for v in _last(c, 512)) for c in (PIECES, HALVES, TILES_LEFT)] == [(False, True, False), (True, False, True), (False, False, True)]
    assert max(sum(c) for c in (PIECES, HALVES, TILES_LEFT)) <= 40000


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", LAST)
def test_the_last_round(M, N, K):
    q, s, w, ws, b = _operands(M, N, K, seed=M + N)
    for bias, act in ((None, api.ACT_NONE), (b, api.ACT_GELU)):
        _check(moe.gemm_block128(q, s, w, ws, bias=bias, act=act), (q, s, w, ws), bias, act)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [PIECES, HALVES, TILES_LEFT])
@pytest.mark.parametrize("gather", [False, True])
def test_the_last_round_of_experts(counts, gather):
    M, N, K, E = 40000, 512, 384, 70
    q, s, w, ws, b = _operands(M, N, K, E, seed=sum(counts))
    layer = _layer(M, 1, E, N, K)
    out = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
    rows = torch.randperm(M, generator=torch.Generator().manual_seed(5)).to(DEV) if gather else torch.arange(M, device=DEV)
    layer.expert_gemm_block128(q, s, w, ws, b, *_tables(counts), out=out, token_indices=rows.int() if gather else None)
    o = 0
    for e, n in enumerate(counts):
        if n:
            r = rows[o:o + n]
            _check(out[o:o + n], (q[r], s[r], w[e], ws[e]), b[e], api.ACT_NONE)
        o += n
    assert (out[o:] == 7).all()
