"""Mode attention in bf16 with infinities among the block's values. A component that an infinity reaches is not finite (in the rows
that see its key; what the masked ones get there is not looked at); every other component is what it is without it.

Tolerance: probabilities in fp16 (2^-11 of each), a split's partial row in fp16 (2^-11 of a component, or 2^-24 of the row's
largest), scores and sums in fp32 (2^-12 at these sizes), the output in bf16 (2^-8):
  |out - ref| <= 2^-8 |ref| + (2^-11 + 2^-11 + 2^-12) sum p |v| + 2^-24 max over the row of sum p |v|
"""

import numpy as np
import pytest
import torch

from oracle import kv8

pytestmark = pytest.mark.gpu

D = 128


@pytest.mark.parametrize("ctx", [0, 300])
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("K,L,H,Hkv", [(4, 16, 4, 2), (8, 16, 8, 4)])
def test_an_infinity_leaves_its_neighbours(K, L, H, Hkv, splits, ctx):
    """Values of about 2^24, beyond what fp16 holds unscaled."""
    import mode_attention

    print(f"case: mode attention, infinity ctx={ctx} K={K} L={L} H={H} Hkv={Hkv} splits={splits}", flush=True)
    g = torch.Generator().manual_seed(K + ctx)
    KL, G, scaling = K * L, H // Hkv, D ** -0.5
    q = torch.randn(1, H, KL, D, generator=g).to(torch.bfloat16)
    k = torch.randn(1, Hkv, ctx + KL, D, generator=g).to(torch.bfloat16)
    v = (torch.randn(1, Hkv, ctx + KL, D, generator=g) * 2.0 ** 24).to(torch.bfloat16)
    v[0, 0, ctx + L, 5], v[0, 0, ctx + 2 * L - 1, 66] = 0, 0  # two keys of mode 1
    f = lambda t: t[0].transpose(0, 1).double().numpy()  # noqa: E731
    o, _, mass, _ = kv8.attention(f(q), f(k)[ctx:], f(v)[ctx:], f(k)[:ctx], f(v)[:ctx], K, L, scaling)
    v[0, 0, ctx + L, 5], v[0, 0, ctx + 2 * L - 1, 66] = float("inf"), -float("inf")
    got = mode_attention.mode_block_attention(q.cuda(), k.cuda(), v.cuda(), K, L, scaling, num_ctx_splits=splits)
    got = got[0].cpu().double().numpy()
    assert not np.isfinite(got[L:2 * L, :G][:, :, [5, 66]]).any()
    bound = 2.0 ** -8 * np.abs(o) + (2 * 2.0 ** -11 + 2.0 ** -12) * mass + 2.0 ** -24 * mass.max(-1, keepdims=True)
    others = np.ones((KL, H, D), bool)
    others[:, :G, [5, 66]] = False
    assert np.isfinite(got[others]).all() and (np.abs(got - o)[others] <= bound[others]).all()
