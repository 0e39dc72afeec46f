"""The rows of partial sums that the norm's gradient leaves in its scratch memory: one of every workgroup that has rows, and no other."""
import pytest
import torch

from cuplayground_amd import api
import rows8_plain as plain
from test_gpu_norm import SLACK, _close, _inputs

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
MARK = 12345.0


# rows, H, the type, and how many workgroups have rows: of rows of up to 64 pieces (16 bytes each) a workgroup takes four
@pytest.mark.parametrize("rows,H,dtype,parts", [(1, 64, BF16, 1), (5, 512, BF16, 2), (256, 510, BF16, 64), (900, 256, F32, 225), (1023, 64, BF16, 256), (1500, 512, BF16, 375),
                                                 (9000, 64, F32, 1024), (5, 520, BF16, 5), (300, 520, BF16, 256), (2000, 1024, F32, 500), (300, 4096, F32, 256)])
def test_only_workgroups_with_rows_leave_sums(rows, H, dtype, parts):
    x, res, w, dout, ds = _inputs(rows, H, dtype, seed=rows)
    size = api._norm_scratch(rows, H)
    scratch = torch.full((size // 4 // H, H), MARK, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    L, P = api.load_library(), api._ptr
    kind = api.DTYPE_F32 if dtype == F32 else api.DTYPE_BF16
    assert L.moe_rms_norm_backward(P(dout), P(x), P(w), P(ds), rows, H, 1e-6, kind, kind, P(dx), P(dw), P(scratch), size, api._stream()) == 0
    assert scratch.shape[0] >= parts and (scratch[parts:] == MARK).all() and not (scratch[:parts] == MARK).all(1).any()
    wx, ww, sx, sw = plain.norm_backward(dout, x, w, 1e-6, ds)
    _close(dx, wx, dtype, sx, 3 * SLACK)
    # the sums of the rows that are there, in fp32 (a column's: 32 threads' parts / 32 additions each)
    assert ((scratch[:parts].double().sum(0) - ww).abs() <= sw * (SLACK + (rows / 64 + 70) * plain.U)).all()
    _close(dw, ww, w.dtype, sw, SLACK + (rows / 64 + 140) * plain.U)
