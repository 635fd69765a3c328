"""The 4-bit draft head at the edges of what its call allows: one row of a tensor with odd strides. Tolerance: test_gpu_mxfp4's."""

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
