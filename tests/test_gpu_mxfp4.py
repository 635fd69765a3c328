"""GPU parity of the 4-bit draft head with float64.

A product of a bf16 and an e2m1 value times a power of two is exact in fp32; a logit is a sum of `hidden` of them in fp32,
at most hidden 2^-24 of the sum of magnitudes (half a step each), and one rounding to bf16, 2^-8 of itself:
  |got - ref| <= 2^-8 |ref| (1 + 2^-8) + hidden 2^-24 (1 + 2^-8) sum |x w|
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _weight(vocab, hidden, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (vocab, hidden // 2), generator=g, dtype=torch.uint8)
    exps = torch.randint(100 if spread else 120, 124, (vocab, hidden // 32), generator=g, dtype=torch.uint8)
    return codes, exps


def _check(got, x, codes, exps):
    import mxfp4_head

    w = mxfp4_head.dequantize(mxfp4_head.Mxfp4Weight(codes, exps)).double()
    ref, mass = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    err = (got.cpu().double() - ref).abs() - (2.0 ** -8 * ref.abs() + x.shape[1] * 2.0 ** -24 * mass) * (1 + 2.0 ** -8)
    assert bool((err <= 0).all()), float(err.max())


@pytest.mark.parametrize("rows,vocab,hidden", [
    (1, 1, 128), (3, 17, 128), (16, 250, 256), (17, 4001, 384), (33, 100, 2560), (128, 515, 1024), (200, 77, 640),  # k-split
    (1, 16500, 128), (15, 20001, 384), (32, 33000, 256), (50, 50003, 512), (65, 70001, 384), (128, 17000, 640),     # wide
    (130, 99999, 256), (7, 163841, 128), (120, 170003, 128),                                                        # rounds
    (40, 18001, 256), (48, 100003, 128), (90, 20003, 384), (70, 140003, 128),                             # 48 and 96 rows
    (128, 98301, 128), (20, 196605, 128), (64, 163839, 128),               # a round that is full but for a few rows
])
def test_draft_head(rows, vocab, hidden):
    import mxfp4_head

    print(f"case: mxfp4 head rows={rows} vocab={vocab} hidden={hidden}", flush=True)
    codes, exps = _weight(vocab, hidden, seed=rows + vocab)
    x = torch.randn(rows, hidden, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    got = mxfp4_head.draft_head_mxfp4(x.cuda(), codes.cuda(), exps.cuda())
    torch.cuda.synchronize()
    assert tuple(got.shape) == (rows, vocab)
    _check(got, x, codes, exps)


def test_every_code_and_scale():
    """Each code under each scale of the format's range here (1 .. 252: from 253 on, 6 * 2^(e - 127) is infinite in bf16, and a
    zero in x times it is NaN; such scales are refused where the weight is laid out), met by a single one in x: the weight
    itself, exact but where it leaves bf16's normal range."""
    import mxfp4_head

    hidden, vocab = 128, 252
    codes = torch.arange(256, dtype=torch.uint8).view(-1)[torch.arange(vocab * 64) % 256].view(vocab, 64).contiguous()
    exps = torch.arange(1, 253, dtype=torch.uint8)[:, None].expand(vocab, 4).contiguous()
    x = torch.eye(128).to(torch.bfloat16)
    got = mxfp4_head.draft_head_mxfp4(x.cuda(), codes.cuda(), exps.cuda()).float().cpu()
    ref = mxfp4_head.dequantize(mxfp4_head.Mxfp4Weight(codes, exps)).t()
    normal = (ref.abs() >= 2.0 ** -126) | (ref == 0)
    assert torch.equal(got[normal], ref[normal].to(torch.bfloat16).float())


def test_strides_output_buffer_and_rows_left_alone():
    import mxfp4_head

    codes, exps = _weight(3001, 256, seed=5)
    base = torch.randn(40, 512, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    x = base[1:21, 128:384]
    buf = torch.full((24, 3016), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[2:22, :3001]
    got = mxfp4_head.draft_head_mxfp4(x, codes.cuda(), exps.cuda(), out=out)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    _check(got, x.cpu(), codes, exps)
    assert bool((buf[:2] == 7).all()) and bool((buf[22:] == 7).all()) and bool((buf[:, 3001:] == 7).all())
    # a base that is not 16-byte aligned is copied, not refused
    _check(mxfp4_head.draft_head_mxfp4(base[:, 1:257], codes.cuda(), exps.cuda()), base[:, 1:257].cpu(), codes, exps)
