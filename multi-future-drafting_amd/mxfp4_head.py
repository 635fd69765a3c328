"""The draft LM head with a 4-bit weight on MI355X (csrc/mxfp4_head.hip): a quarter of the draft step's largest stream.

The weight is in the OCP microscaling format MXFP4: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a
byte, low half first, and a power-of-two scale 2^(e - 127) for 32 weights of a row:
  codes  uint8 [vocab, hidden / 2],  exps  uint8 [vocab, hidden / 32],  hidden a multiple of 128.
quantize writes e of 1 .. 252: from 253 on 6 * 2^(e - 127) is infinite in bf16, and 255 is NaN. check_weight(values=True)
holds a weight to that, with ``ready_made`` also allowing 0, the format's 2^-127, which ready-made weights give their groups of
zeros (products with it are exact too). A call does not look at the values.
The product is exact in float32 (bf16 hidden states times such weights) and summed there; a logit is rounded once to bf16.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

import mfd_hip

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP = 32
MAX_EXP = 252


class Mxfp4Weight(NamedTuple):
    """An LM head in 4 bits; what DDTreeDraftTopK takes as its ``weight`` beside a bf16 matrix."""

    codes: torch.Tensor
    exps: torch.Tensor

    @property
    def device(self):
        return self.codes.device

    @property
    def shape(self):
        return self.codes.shape[0], self.codes.shape[1] * 2


def check_weight(codes: torch.Tensor, exps: torch.Tensor, values: bool = False, ready_made: bool = False) -> None:
    """The layout above, and with ``values`` (which waits for the device) the range of the scales; ValueError otherwise."""
    shape = codes.shape
    if codes.dtype is not torch.uint8 or exps.dtype is not torch.uint8 or len(shape) != 2 or \
            not codes.is_contiguous() or not exps.is_contiguous() or shape[1] % 64 or shape[0] < 1 or shape[1] < 1 or \
            tuple(exps.shape) != (shape[0], shape[1] // 16) or exps.get_device() != codes.get_device() or \
            codes.data_ptr() % 16 or exps.data_ptr() % 4:
        raise ValueError(f"codes must be contiguous uint8 [vocab, hidden / 2] with hidden % 128 == 0 and exps contiguous "
                         f"uint8 [vocab, hidden / {GROUP}] on the same device, got {codes.dtype} {tuple(codes.shape)} and "
                         f"{exps.dtype} {tuple(exps.shape)}")
    least = 0 if ready_made else 1
    if values and bool(((exps < least) | (exps > MAX_EXP)).any()):
        raise ValueError(f"scale exponents must be {least} .. {MAX_EXP}")


def quantize(weight: torch.Tensor, rows_at_once: int = 16384) -> Mxfp4Weight:
    """A finite float matrix [vocab, hidden] in 4 bits, once at load time: per group of 32 the scale under which the largest
    magnitude lies in (3.5, 7] (it rounds to 4 or 6), every weight to the nearest code (ties to the even one)."""
    vocab, hidden = weight.shape
    if hidden % 128:
        raise ValueError(f"hidden must be a multiple of 128, got {hidden}")
    codes = torch.empty((vocab, hidden // 2), dtype=torch.uint8, device=weight.device)
    exps = torch.empty((vocab, hidden // GROUP), dtype=torch.uint8, device=weight.device)
    # borders between neighbouring codes
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=weight.device)
    for lo in range(0, vocab, rows_at_once):
        w = weight[lo:lo + rows_at_once].double().view(-1, hidden // GROUP, GROUP)
        if not bool(torch.isfinite(w).all()):
            raise ValueError("weights must be finite")
        amax = w.abs().amax(-1)
        m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 7 = 0.875 * 2^3
        e = torch.where(m > 0.875, e - 2, e - 3)
        e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-126, MAX_EXP - 127)
        a = torch.ldexp(w.abs(), -e[..., None].to(w.dtype)).clamp(max=6.0)
        c = torch.bucketize(a, borders)                      # a border belongs to the code below it
        on = torch.bucketize(a, borders, right=True) != c    # on a border: c is below it, c + 1 above; the even one
        c = torch.where(on & (c % 2 == 1), c + 1, c)
        c = (c + 8 * torch.signbit(w).to(c.dtype)).view(-1, hidden)
        codes[lo:lo + rows_at_once] = (c[:, 0::2] + 16 * c[:, 1::2]).to(torch.uint8)
        exps[lo:lo + rows_at_once] = (e + 127).to(torch.uint8)
    return Mxfp4Weight(codes, exps)


def dequantize(weight: Mxfp4Weight) -> torch.Tensor:
    """The weight's values [vocab, hidden] in float32 (checks and tests)."""
    values = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=weight.device)
    c = torch.stack([weight.codes & 15, weight.codes >> 4], dim=-1).view(weight.shape).int()
    scale = torch.ldexp(torch.ones((), device=weight.device), weight.exps.int() - 127)
    return values[c] * scale.repeat_interleave(GROUP, dim=1)


def draft_head_mxfp4(x: torch.Tensor, codes: torch.Tensor, exps: torch.Tensor,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [rows, vocab] bf16 of hidden states x [rows, hidden] (bf16; rows may have a stride). Rows of the result are
    padded to a multiple of 8 elements, as tree_logits wants them; ``out``: a [rows, vocab] bf16 buffer with contiguous
    rows, their stride a multiple of 4."""
    check_weight(codes, exps)
    vocab, hidden = codes.shape[0], codes.shape[1] * 2
    if x.dtype is not torch.bfloat16 or x.dim() != 2 or x.shape[1] != hidden:
        raise ValueError(f"x must be bfloat16 [rows, {hidden}], got {x.dtype} {tuple(x.shape)}")
    device = x.get_device()
    if device < 0 or codes.get_device() != device or exps.get_device() != device or (
            out is not None and out.get_device() != device):
        raise ValueError(f"MFD kernels take GPU tensors of one device (x on {x.device}, codes on {codes.device})")
    # (one row has no stride: that of the tensor it was cut from says nothing)
    rows, stride = x.shape[0], x.stride()
    step = stride[0] if rows > 1 else hidden
    if stride[1] != 1 or step % 8 or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        step = hidden
    if out is None:
        out = x.new_empty((rows, (vocab + 7) // 8 * 8))
        pitch = out.stride(0)
        if out.shape[1] != vocab:
            out = out[:, :vocab]
    else:
        pitch = out.stride(0) if rows > 1 else (vocab + 7) // 8 * 8
        if out.dtype is not torch.bfloat16 or tuple(out.shape) != (rows, vocab) or (vocab > 1 and out.stride(1) != 1):
            raise ValueError(f"out must be bfloat16 [{rows}, {vocab}] with contiguous rows")
    mfd_hip.call_on(device, "mfd_draft_head_mxfp4", x.data_ptr(), step, rows or 1, 0, codes.data_ptr(),
                    exps.data_ptr(), rows, vocab, hidden, out.data_ptr(), pitch)
    return out
