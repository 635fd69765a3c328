"""The 4-bit draft head at the edges of what its call allows: one row of a tensor with odd strides, and hidden sizes of several
blocks of drafted rows. Tolerance: test_gpu_mxfp4's."""

import pytest
import torch

from test_gpu_mxfp4 import _check, _weight

pytestmark = pytest.mark.gpu


def test_one_row_has_no_stride():
    """Slices of one row, whose stride is that of the tensor they come from and means nothing: as x, and as the result's buffer."""
    import mxfp4_head

    codes, exps = _weight(3001, 128, seed=7)
    base = torch.randn(3, 129, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    x = base.cuda()[:1, :128]
    got = mxfp4_head.draft_head_mxfp4(x, codes.cuda(), exps.cuda())
    torch.cuda.synchronize()
    _check(got, base[:1, :128], codes, exps)
    buf = torch.full((2, 3003), 7.0, dtype=torch.bfloat16, device="cuda")
    again = mxfp4_head.draft_head_mxfp4(x.contiguous(), codes.cuda(), exps.cuda(), out=buf[:1, :3001])
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), got.view(torch.int16))
    assert bool((buf[0, 3001:] == 7).all()) and bool((buf[1] == 7).all())


# The wide form (vocabularies above a 16-row tile per CU, or more than 32 rows) by its number of 16-row drafted tiles. A block of
# drafted rows in LDS is 1024 k up to 16 rows, 512 up to 64, 256 above, and a step 256: blocks of four steps, two and one.
# Several blocks each, the last one full or partly filled, hidden sizes of an odd number of 128-k halves, one tile a wave and
# more, more than one round of workgroups (the last of each).
WIDE = [
    (15, 20001, 2560), (7, 16500, 1152), (16, 33000, 4096), (1, 70001, 2176), (15, 150001, 1920), (9, 230001, 1280),  # <= 16
    (30, 20003, 2560), (17, 70003, 1152), (32, 150001, 896), (20, 230003, 640),                                       # <= 32
    (40, 20003, 2560), (48, 100003, 1152), (33, 163843, 640),                                                         # <= 48
    (60, 20001, 1152), (64, 90001, 2560), (50, 170001, 640),                                                          # <= 64
    (90, 20003, 2560), (65, 100001, 1152), (96, 140003, 640),                                                         # <= 96
    (128, 20001, 2560), (100, 60001, 1152), (120, 110003, 640),                                                       # <= 128
]


@pytest.mark.parametrize("rows,vocab,hidden", WIDE)
def test_blocks_of_drafted_rows(rows, vocab, hidden):
    import mxfp4_head

    print(f"case: mxfp4 head, blocks, rows={rows} vocab={vocab} hidden={hidden}", flush=True)
    codes, exps = (t.cuda() for t in _weight(vocab, hidden, seed=rows + vocab))
    x = torch.randn(rows, hidden, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    got = mxfp4_head.draft_head_mxfp4(x, codes, exps)
    xd = x.double()
    for lo in range(0, vocab, 16384):
        part = slice(lo, lo + 16384)
        w = mxfp4_head.dequantize(mxfp4_head.Mxfp4Weight(codes[part], exps[part])).double()
        ref, mass = xd @ w.t(), xd.abs() @ w.abs().t()
        bound = (2.0 ** -8 * ref.abs() + hidden * 2.0 ** -24 * mass) * (1 + 2.0 ** -8)
        assert bool(((got[:, part].double() - ref).abs() <= bound).all()), lo
