"""The kernels of the block-scaled e4m3 products that test_block128_kernels.py has no size for: every streamer with weights read past the caches and
kept there, the tiles that read them past, rows fetched by index through every kernel, and tokens' rows of more than 2 GiB.  As there, which kernel
a size takes is asked of the library and asserted."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import rows8_plain as plain
from rows8_plain import U
from test_block128_kernels import _plan, _spread
from test_gpu_block128 import _check, _cut, _operands, _tables

DEV = "cuda"
BF16 = torch.bfloat16
STREAMERS = [(16, 16, 8), (16, 32, 1), (16, 32, 2), (16, 32, 4)]
TILES = [(16, 64, 4), (32, 64, 2), (64, 64, 2), (64, 128, 1), (128, 128, 1), (128, 256, 1), (256, 256, 1)]

# M, N, K, the kernel: up to eight rows, and more, in a streamer
DENSE = [(11, 18, 4096, (16, 16, 8)), (4, 32909, 1024, (16, 32, 2)), (13, 32987, 1024, (16, 32, 2))]
# ... with more than 256 MiB of weights for one block of rows
COLD_DENSE = [(5, 3625, 74112, (16, 16, 8)), (12, 3712, 76288, (16, 16, 8)), (6, 33037, 8960, (16, 32, 2)), (3, 10666, 25216, (16, 64, 4)), (21, 10885, 24704, (32, 64, 2)),
              (36, 16098, 16768, (64, 64, 2)), (8, 26568, 10112, (64, 128, 1))]
# M, N, K, experts, the kernel: rows packed and rows fetched by index
EXPERTS = [(1, 128, 4096, 1, (16, 16, 8)), (57, 1152, 512, 70, (16, 32, 1)), (3, 21888, 512, 3, (16, 32, 1)), (11, 4352, 1024, 8, (16, 32, 2)), (3, 5504, 2048, 3, (16, 32, 4)),
           (40, 128, 1152, 3, (16, 64, 4)), (1492, 128, 640, 70, (32, 64, 2)), (579, 512, 768, 30, (64, 64, 2)), (816, 640, 128, 1, (64, 128, 1)),
           (3345, 384, 1664, 70, (128, 128, 1)), (1388, 1792, 384, 30, (128, 256, 1)), (1177, 7552, 384, 8, (256, 256, 1))]
# ... with more than 128 MiB, about one block of rows to an expert
COLD_EXPERTS = [(2, 1792, 37504, 2, (16, 16, 8)), (1, 34048, 3968, 1, (16, 32, 2)), (4, 2304, 19456, 3, (16, 64, 4)), (29, 6912, 9728, 2, (32, 64, 2)),
                (30, 14976, 9088, 1, (64, 64, 2)), (5, 30848, 2176, 2, (64, 128, 1)), (123, 18176, 7424, 1, (128, 128, 1)), (70, 42240, 3200, 1, (128, 256, 1)),
                (230, 38912, 3456, 1, (256, 256, 1))]


def _layer(S, E, N, K):
    """Of either projection: a layer's rows have at most 16384 values, its experts' as many as they like."""
    return moe.MoELayer(moe.MoEConfig(expert_top_k=1, hidden_act=0, hidden_size=min(N, K), intermediate_size=max(N, K), micro_batch=1, num_experts=E, sequence_len=S,
                                      torch_dtype=api.DTYPE_FP8))


def test_the_sizes_below_take_every_kernel():
    for M, N, K, kernel in DENSE + COLD_DENSE:
        assert _plan(M, N, K) == kernel, (M, N, K, _plan(M, N, K))
    for M, N, K, E, kernel in EXPERTS + COLD_EXPERTS:
        assert _plan(M, N, K, E) == kernel, (M, N, K, E, _plan(M, N, K, E))
    assert {s[-1] for s in EXPERTS} == set(STREAMERS + TILES)
    # (fewer parts than that have streamers with little to read)
    assert {s[-1] for s in COLD_EXPERTS} == set(TILES) | {(16, 16, 8), (16, 32, 2)}
    assert all(N * K > 256 << 20 and M <= k[0] for M, N, K, k in COLD_DENSE)
    assert all(min(E, M) * N * K > 128 << 20 and M <= min(E, M) * k[0] for M, N, K, E, k in COLD_EXPERTS)
    assert {M > 8 for M, N, K, k in DENSE if k[1] == 32} == {M > 8 for M, N, K, k in COLD_DENSE if k[:2] == (16, 16)} == {False, True}


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,kernel", DENSE + COLD_DENSE)
def test_one_matrix(M, N, K, kernel):
    q, s, w, ws, b = _operands(M, N, K, seed=M + N)
    for bias, act in ((None, api.ACT_NONE), (b, api.ACT_GELU)):
        _check(moe.gemm_block128(q, s, w, ws, bias=bias, act=act), (q, s, w, ws), bias, act)


@pytest.mark.gpu
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("how", ["even", "drawn"])
@pytest.mark.parametrize("M,N,K,E,kernel", EXPERTS + COLD_EXPERTS)
def test_experts(M, N, K, E, kernel, how, gather):
    """Indices in no order, some of them twice, one of no token: a row of zeros."""
    counts = _spread(M, E, how)
    q, s, w, ws, b = _operands(M, N, K, E, seed=M)
    token = torch.randint(0, M, (M,), generator=torch.Generator().manual_seed(M)).int().to(DEV) if gather else None
    a = plain.widen_rows(q, s)
    bad = sum(counts) // 2 if gather and sum(counts) > 1 else -1
    if bad >= 0:
        token[bad] = M
    out = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
    _layer(M, E, N, K).expert_gemm_block128(q, s, w, ws, b, *_tables(counts), out=out, token_indices=token)
    o = 0
    for e, n in enumerate(counts):
        if n:
            rows = torch.arange(o, o + n, device=DEV)
            known = rows[rows != bad]
            r = token[known].long() if gather else known
            if len(known):
                _check(out[known], (q[r], s[r], w[e], ws[e]), b[e], api.ACT_NONE)
            if o <= bad < o + n:
                assert torch.equal(out[bad], b[e])
        o += n
    assert (out[o:] == 7).all() and torch.equal(plain.widen_rows(q, s), a)


# tokens, K, N: rows of 2 to 3 GiB
@pytest.mark.gpu
@pytest.mark.parametrize("S,K,N", [(1_250_000, 2048, 256), (49_000, 65_536, 128), (1_572_863, 2048, 128)])
def test_far_tokens_fetched(S, K, N):
    assert 2 << 30 < S * K < 3 << 30
    E, counts = 2, (300, 41)
    kept = sum(counts)
    token = torch.randint(0, S, (S,), generator=torch.Generator().manual_seed(1)).int().to(DEV)
    edge = [r for place in (1 << 31, S * K) for r in (place // K - 2, place // K - 1, place // K, place // K + 1) if r < S]
    token[:len(edge)] = torch.tensor(edge, dtype=torch.int32)
    token[kept - 3:kept] = torch.tensor([S, S - 1, S + 1], dtype=torch.int32)      # just past the last row, it, and past it
    at = token[:kept].long()
    at = at[at < S].unique()
    few = _operands(len(at), N, K, E, seed=9)
    q, s = torch.zeros(S, K, dtype=torch.uint8, device=DEV), torch.ones(S, K // 128, device=DEV)
    q[at], s[at] = few[0], few[1]
    out = torch.full((S, N), 7.0, dtype=BF16, device=DEV)
    _layer(S, E, N, K).expert_gemm_block128(q, s, few[2], few[3], few[4], *_tables(counts), out=out, token_indices=token)
    o = 0
    for e, n in enumerate(counts):
        rows = torch.arange(o, o + n, device=DEV)
        known = rows[token[rows] < S]
        r = token[known].long()
        _check(out[known], (q[r], s[r], few[2][e], few[3][e]), few[4][e], api.ACT_NONE)
        o += n
    assert torch.equal(out[kept - 3], few[4][1]) and torch.equal(out[kept - 1], few[4][1]) and (out[kept:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 18, 5760), (20, 333, 640), (100, 2752, 384), (513, 2049, 640)])
def test_sums_that_cancel(M, N, K):
    """The second half of the contraction takes back the first: what is left of the instruction's eights is within what the header says."""
    q, s, w, ws, _ = _operands(M, N, K // 2 // 128 * 128, seed=M)
    q2, w2 = torch.cat([q, q ^ 0x80], 1), torch.cat([w, w], 1)
    s2, ws2 = torch.cat([s, s], 1).contiguous(), torch.cat([ws, ws], 1).contiguous()
    got = moe.gemm_block128(q2, s2, w2, ws2).double()
    size = plain.widen_rows(q2, s2).abs() @ plain.widen_blocks(w2, ws2).abs().t()
    assert (got.abs() <= (_cut(q2, s2, w2, ws2) + 2 * (2 + 17 * q2.shape[1] / 128) * U * size) * (1 + plain.half_step(BF16))).all()
