"""The norm of the residual stream, its gradient, its form in e4m3, and the activation in e4m3, against their formulas in 64 bits.

Tolerances: a result is rounded once, half a step of its type.  In front of that a row's sum of H squares is made in fp32 by at most 64 additions a
thread and 20 between threads, so r is off by at most 84 / 2 + 4 half steps of fp32, and y by 3 more: 64 U is above that."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api
import rows8_plain as plain
from rows8_plain import U

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SLACK = 64 * U
# one value to the widest row: every number of threads and pieces, rows that begin on no 16 bytes, last pieces of one column
WIDTHS = [1, 2, 7, 64, 72, 129, 510, 512, 520, 1000, 1024, 1031, 2048, 2056, 4096, 4097, 4104, 7168, 8200, 16383, 16384]


def _inputs(rows, H, dtype, seed=0, w32=False, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, res, dout, ds = (torch.randn(rows, H, generator=g, device=DEV).mul_(std).to(dtype) for _ in range(4))
    w = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(F32 if w32 else dtype)
    return x, res, w, dout, ds


def _close(got, want, dtype, size=None, slack=SLACK):
    tol = want.abs() * plain.half_step(dtype) + plain.smallest_half(dtype) + (want.abs() if size is None else size) * slack * 1.01
    off = (got.double() - want).abs()
    assert got.dtype == dtype and (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_and_gradient(H, dtype):
    for rows, residual, w32 in ((1, True, False), (5, False, True), (131, True, True), (4100 if H < 1100 else 300, True, False)):
        x, res, w, dout, ds = _inputs(rows, H, dtype, seed=H + rows, w32=w32)
        want, h, _ = plain.norm(x, w, 1e-6, res if residual else None)
        got = moe.rms_norm(x, w, 1e-6, residual=res if residual else None)
        if residual:
            got, total = got
            assert total.dtype == dtype and torch.equal(total.double(), h)
        _close(got, want, dtype)
        dsum = ds if residual else None
        dx, dw = moe.rms_norm_backward(dout, total if residual else x, w, 1e-6, dsum=dsum)
        wx, ww, sx, sw = plain.norm_backward(dout, h, w, 1e-6, dsum)
        _close(dx, wx, dtype, sx, 3 * SLACK)
        # a column's sum: at most rows / 256 + 1 additions a workgroup, 32 + 32 between them, and n is off by SLACK
        _close(dw, ww, w.dtype, sw, SLACK + (rows / 256 + 70) * U)
        assert torch.equal(dw, moe.rms_norm_backward(dout, total if residual else x, w, 1e-6, dsum=dsum)[1])


def test_gradient_against_differences():
    rows, H, step = 6, 96, 1e-3
    x, res, w, dout, ds = _inputs(rows, H, F32, seed=3, w32=True)

    def loss(x, res, w):
        y, h, _ = plain.norm(x.double(), w, 1e-5, res.double())
        return (y * dout.double()).sum() + (h * ds.double()).sum()

    total = moe.rms_norm(x, w, 1e-5, residual=res)[1]
    dx, dw = moe.rms_norm_backward(dout, total, w, 1e-5, dsum=ds)
    # central differences of a smooth function, 64 bits: step^2 times its third derivative (below 20 here) and 1e-16 / step of rounding; the kernel's fp32
    for got, at in ((dx, 0), (dw, 2)):
        args = [x.double(), res.double(), w.double()]
        for i in range(0, got.numel(), 37):
            up, down = [a.clone() for a in args], [a.clone() for a in args]
            up[at].view(-1)[i] += step
            down[at].view(-1)[i] -= step
            d = (loss(*up) - loss(*down)) / (2 * step)
            assert abs(float(d) - float(got.view(-1)[i])) <= 20 * step ** 2 + 1e-4


@pytest.mark.parametrize("H", [128, 256, 512, 640, 1024, 1152, 2048, 4096, 7168, 8320, 16384])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_to_8_bits(H, dtype):
    for rows, residual, both, w32 in ((1, True, True, False), (3, False, False, True), (77, True, False, False), (5000 if H <= 1024 else 200, False, True, True)):
        x, res, w, _, _ = _inputs(rows, H, dtype, seed=H + rows, w32=w32)
        q, s, out, h = moe.rms_norm_rows128(x, w, 1e-6, residual=res if residual else None, want_rows=both)
        y, hw, _ = plain.norm(x, w, 1e-6, res if residual else None)
        plain.check_rows8(q, s, y, SLACK)
        assert (out is not None) == both and (h is not None) == residual
        same = moe.rms_norm(x, w, 1e-6, residual=res if residual else None)
        if both:
            assert torch.equal(out, same[0] if residual else same)
        if residual:
            assert torch.equal(h.double(), hw)


def test_pieces_of_zeros_small_and_bad_values():
    H = 512
    x = torch.randn(6, H, device=DEV, dtype=F32)
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    w = torch.ones(H, device=DEV)
    w[256:384] = 2.0 ** -130                        # results that fp32 has no normal numbers for
    q, s, out, _ = moe.rms_norm_rows128(x, w, 1e-6, want_rows=True)
    assert not q[0].any() and (s[0] == 1).all() and not out[0].any()
    assert not q[1, 128:256].any() and s[1, 1] == 1
    assert torch.isnan(plain.widen_rows(q, s)[2, 5]) and torch.isnan(out[2, 5]) and not out[2, 6:].any()      # r = 0
    assert torch.isnan(out[3]).all() and torch.isnan(plain.widen_rows(q, s)[3]).all()
    assert (s[4:, 2] == 2.0 ** -126).all() and torch.isfinite(plain.widen_rows(q, s)[4:]).all()
    y = plain.norm(x[4:], w, 1e-6)[0]
    assert ((plain.widen_rows(q, s)[4:] - y).abs()[:, 256:384] <= y.abs()[:, 256:384] * 2.0 ** -4 + 2.0 ** -136).all()


def test_no_rows():
    w = torch.ones(256, device=DEV, dtype=BF16)
    x = torch.empty(0, 256, device=DEV, dtype=BF16)
    assert moe.rms_norm(x, w).shape == (0, 256)
    q, s, out, h = moe.rms_norm_rows128(x, w, residual=x)
    assert q.shape == (0, 256) and s.shape == (0, 2) and h.shape == (0, 256) and out is None
    dx, dw = moe.rms_norm_backward(x, x, w)
    assert dx.shape == (0, 256) and not dw.any()
    q, s = moe.act_rows128(x, None, api.ACT_RELU)
    assert q.shape == (0, 256) and s.shape == (0, 2)


@pytest.mark.parametrize("shift", [1, 4])
def test_rows_at_any_address(shift):
    """Views that begin on no 16 bytes: the same numbers as from copies."""
    rows, H = 9, 264
    for dtype in (BF16, F32):
        x, res, w, dout, ds = _inputs(rows, H, dtype, seed=1)

        def moved(t):
            room = torch.empty(t.numel() + shift, dtype=t.dtype, device=DEV)
            v = room[shift:].view(t.shape)
            v.copy_(t)
            return v

        want = moe.rms_norm(x, w, residual=res)
        got = moe.rms_norm(moved(x), moved(w), residual=moved(res))
        y, h, _ = plain.norm(x, w, 1e-6, res)
        _close(got[0], y, dtype)
        assert torch.equal(got[1], want[1])
        dx, dw = moe.rms_norm_backward(moved(dout), moved(want[1]), moved(w), dsum=moved(ds))
        wx, ww, sx, sw = plain.norm_backward(dout, h, w, 1e-6, ds)
        _close(dx, wx, dtype, sx, 3 * SLACK)
        _close(dw, ww, dtype, sw, 2 * SLACK)


@pytest.mark.parametrize("act", [api.ACT_SWIGLU, api.ACT_GELU, api.ACT_RELU])
@pytest.mark.parametrize("rows,I", [(1, 128), (3, 640), (1000, 1408), (37, 14336)])
def test_activation_to_8_bits(rows, I, act):
    g = torch.Generator(device=DEV).manual_seed(rows)
    u = (torch.randn(rows, I, generator=g, device=DEV) * 3).bfloat16()
    gate = (torch.randn(rows, I, generator=g, device=DEV) * 6).bfloat16() if act == api.ACT_SWIGLU else None
    q, s = moe.act_rows128(u, gate, act)
    y = plain.activate(u.double(), act, None if gate is None else gate.double())
    # SwiGLU: exp and a reciprocal of 2 U each, two products.  GELU in fp32: 1 + erf is off by 2 U, which is u 2 U of the result; a value that is
    # small against that (in the tail) is small against its piece's scale
    if act == api.ACT_GELU:
        y32 = plain.activate(u.float(), act).double()
        assert ((y32 - y).abs() <= 4 * U * u.double().abs()).all()
        want = plain.rows8_scales(y)
        step = want.repeat_interleave(128, -1)
        got = plain.widen_rows(q, s)
        assert ((s.double() - want).abs() <= 16 * U * want).all()
        assert ((got - y).abs() <= torch.maximum(y.abs() * 2.0 ** -4, step * 2.0 ** -10) + 16 * U * u.double().abs()).all()
    else:
        plain.check_rows8(q, s, y, 16 * U)


def test_activation_of_far_and_bad_values():
    v = torch.tensor([-3.0e38, -1000.0, -88.0, -87.0, -20.0, 0.0, 20.0, 88.0, 1000.0, 3.0e4], device=DEV).bfloat16()
    gate, u = torch.zeros(3, 128, device=DEV, dtype=BF16), torch.ones(3, 128, device=DEV, dtype=BF16)
    gate[0, :10] = v
    gate[1, 3] = float("nan")
    gate[2, 9] = float("inf")
    q, s = moe.act_rows128(u, gate, api.ACT_SWIGLU)
    got, want = plain.widen_rows(q, s), plain.activate(u.double(), api.ACT_SWIGLU, gate.double())
    assert ((got[0, 1:] - want[0, 1:]).abs() <= torch.maximum(want[0, 1:].abs() * 0.0626, s[0].double() * 2.0 ** -10)).all()
    assert got[0, 0].abs() <= 1                                     # -3e38 / 2^126, where the exact one is 0: nothing against its piece's 3e4
    assert torch.isnan(got[1, 3]) and not got[1, 4:].any() and torch.isnan(got[2]).all()


def test_activation_keeps_to_the_experts_rows():
    R, I = 50, 256
    g = torch.Generator(device=DEV).manual_seed(2)
    u, gate = (torch.randn(R, I, generator=g, device=DEV).bfloat16() for _ in range(2))
    count = torch.tensor([7, 0, 20], dtype=torch.int32, device=DEV)
    offset = torch.tensor([0, 7, 7], dtype=torch.int32, device=DEV)
    u[27:] = float("nan")
    whole_q, whole_s = moe.act_rows128(u, gate, api.ACT_SWIGLU)
    L, P = api.load_library(), api._ptr
    q = torch.full((R, I), 77, dtype=torch.uint8, device=DEV)
    s = torch.full((R, I // 128), 5.0, device=DEV)
    assert L.moe_act_rows128(P(u), P(gate), R, I, api.ACT_SWIGLU, P(count), P(offset), 3, P(q), P(s), api._stream()) == 0
    assert torch.equal(q[:27], whole_q[:27]) and torch.equal(s[:27], whole_s[:27]) and (q[27:] == 77).all() and (s[27:] == 5).all()
    q2, s2 = moe.act_rows128(u, gate, api.ACT_SWIGLU, count, offset)
    assert torch.equal(q2[:27], q[:27]) and torch.equal(s2[:27], s[:27])


def test_norm_in_graphs_and_on_other_streams():
    """Captured calls share nothing: two graphs replayed in turn, eager calls between them, on a stream of their own."""
    rows, H = 40, 1280
    ins = [_inputs(rows, H, BF16, seed=i) for i in range(3)]

    def step(x, res, w, dout, ds):
        y, h = moe.rms_norm(x, w, residual=res)
        dx, dw = moe.rms_norm_backward(dout, h, w, dsum=ds)
        return (y, h, dx, dw, *moe.rms_norm_rows128(x, w, residual=res, want_rows=True), *moe.act_rows128(x, res, api.ACT_SWIGLU))

    want = [step(*i) for i in ins]
    held = [tuple(t.clone() for t in ins[0]) for _ in range(2)]
    graphs, outs = [], []
    for hh in held:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*hh))
        graphs.append(g)
    other = torch.cuda.Stream()
    for turn in range(4):
        for i in range(2):
            for dst, src in zip(held[i], ins[(turn + i) % 3]):
                dst.copy_(src)
            graphs[i].replay()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            eager = step(*ins[turn % 3])
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], want[(turn + i) % 3]):
                assert torch.equal(a, b)
        for a, b in zip(eager, want[turn % 3]):
            assert torch.equal(a, b)


def test_sum_in_place():
    x, res, w, _, _ = _inputs(33, 768, BF16, seed=9)
    want = moe.rms_norm(x, w, residual=res)
    L, P = api.load_library(), api._ptr
    for which in range(2):
        a, b, out = x.clone(), res.clone(), torch.empty_like(x)
        assert L.moe_rms_norm(P(a), P(b), P(w), 33, 768, 1e-6, api.DTYPE_BF16, api.DTYPE_BF16, P((a, b)[which]), P(out), None, None, api._stream()) == 0
        assert torch.equal(out, want[0]) and torch.equal((a, b)[which], want[1]) and torch.equal((b, a)[which], (res, x)[which])
