"""The 4-bit draft head at the edges of what its call allows: one row of a tensor with odd strides, hidden sizes of several
blocks of drafted rows, exponent 0. Tolerance: test_gpu_mxfp4's."""

import pytest
import torch

from test_gpu_mxfp4 import _check, _weight

pytestmark = pytest.mark.gpu


def test_one_row_has_no_stride():
    """Slices of one row, whose stride is that of the tensor they come from and means nothing: as x, and as the
    result's buffer."""
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


def _ready_made():
    """A weight as ready-made files have it: groups of zeros under exponent 0 (2^-127), and one group of codes under it."""
    codes, exps = _weight(20001, 256, seed=11)
    codes[5:500:7, 16:32] = 0
    exps[5:500:7, 1] = 0
    codes[9, 32:48], exps[9, 2] = torch.arange(16, 32, dtype=torch.uint8), 0
    return codes, exps


def test_exponent_zero():
    """2^-127 under each code, met by a single one and by 2^100: exact, the subnormal values too; and a weight with
    such groups."""
    import mxfp4_head

    for vocab in (252, 20000):  # k-split and wide form
        codes = torch.arange(256, dtype=torch.uint8)[torch.arange(vocab * 64) % 256].view(vocab, 64).contiguous()
        exps = torch.zeros(vocab, 4, dtype=torch.uint8)
        pair = torch.stack([codes & 15, codes >> 4], dim=-1).view(vocab, 128).int()
        ref = torch.tensor(mxfp4_head.E2M1 + tuple(-v for v in mxfp4_head.E2M1), dtype=torch.float64)[pair].t() * 2.0 ** -127
        assert torch.equal(mxfp4_head.dequantize(mxfp4_head.Mxfp4Weight(codes, exps)).double().t(), ref)
        for size in (1.0, 2.0 ** 100):
            x = (torch.eye(128) * size).to(torch.bfloat16)
            got = mxfp4_head.draft_head_mxfp4(x.cuda(), codes.cuda(), exps.cuda())
            assert torch.equal(got.cpu().double(), ref * size)
    codes, exps = _ready_made()
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(12)).to(torch.bfloat16)
    _check(mxfp4_head.draft_head_mxfp4(x.cuda(), codes.cuda(), exps.cuda()), x, codes, exps)


def test_candidates_from_a_ready_made_weight():
    """DDTreeDraftTopK takes such a weight as it is."""
    import ddtree_sglang_ops
    import mxfp4_head

    codes, exps = (t.cuda() for t in _ready_made())
    head = ddtree_sglang_ops.DDTreeDraftTopK(weight=mxfp4_head.Mxfp4Weight(codes, exps), block_size=8, num_modes=2, budget=17,
                                             max_bs=1)
    x = torch.randn(16, 256, generator=torch.Generator().manual_seed(13)).to(torch.bfloat16).cuda()
    head(x)
    logits = mxfp4_head.draft_head_mxfp4(x.view(2, 8, 256)[:, 1:].reshape(14, 256), codes, exps)
    assert torch.equal(head.logits[:14].view(torch.int16), logits.view(torch.int16))
    for e in (253, 255):
        exps[3, 1] = e
        with pytest.raises(ValueError, match="exponents"):
            ddtree_sglang_ops.DDTreeDraftTopK(weight=mxfp4_head.Mxfp4Weight(codes, exps), block_size=8, num_modes=2, budget=17,
                                              max_bs=1)


@pytest.mark.parametrize("mxfp4", [True, False])
def test_candidates_belong_to_the_tensors_device(monkeypatch, mxfp4):
    """DDTreeDraftTopK launches on its tensors' GPU, whichever is current, and refuses hidden states of another device than the
    weight's. (One GPU: the current device is said to be another, and the change to the tensors' own is looked for.)"""
    import ddtree_sglang_ops
    import mfd_hip
    import mxfp4_head

    codes, exps = (t.cuda() for t in _weight(20001, 256, seed=14))
    weight = mxfp4_head.Mxfp4Weight(codes, exps)
    if not mxfp4:
        weight = mxfp4_head.dequantize(weight).to(torch.bfloat16)
    head = ddtree_sglang_ops.DDTreeDraftTopK(weight=weight, block_size=8, num_modes=2, budget=17, max_bs=1)
    x = torch.randn(16, 256, generator=torch.Generator().manual_seed(15)).to(torch.bfloat16).cuda()
    head(x)
    logp, ids = (t.clone() for t in head.outputs(1))
    monkeypatch.setattr(mfd_hip, "_current_device", lambda: 1)
    entered, device = [], torch.cuda.device
    monkeypatch.setattr(torch.cuda, "device", lambda index: entered.append(index) or device(index))
    head.top_logp.zero_()
    head(x)
    assert entered == [0]
    assert torch.equal(head.outputs(1)[0], logp) and torch.equal(head.outputs(1)[1], ids)
    with pytest.raises(ValueError, match="device"):
        head(x.cpu())
