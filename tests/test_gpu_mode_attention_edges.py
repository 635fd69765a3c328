"""Mode attention in bf16 in batches of thousands, and with infinities among the block's values: a component that one reaches is
not finite (in the rows that see its key; what the masked ones get there is not looked at); every other is as without it.

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


@pytest.mark.parametrize("page", [1, 64])
def test_a_batch_of_thousands(page):
    """Thousands of requests in one call: the bits of the same requests in calls of 60."""
    import paged_mode_attention

    bs, K, L, H, Hkv = 3001, 2, 10, 4, 2
    print(f"case: mode attention of {bs} requests, page size {page}", flush=True)
    g = torch.Generator().manual_seed(page)
    KL, slots = K * L, 4096
    lens = torch.randint(0, 200, (bs,), generator=g).cuda()
    table = torch.randint(0, slots // page, (bs, -(-200 // page)), generator=g).int().cuda()
    kc, vc = (torch.randn(slots, Hkv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q, kn, vn = (torch.randn(bs * KL, n, D, generator=g).to(torch.bfloat16).cuda() for n in (H, Hkv, Hkv))
    rows = torch.arange(bs).cuda()
    call = lambda a, b: paged_mode_attention.paged_mode_block_attention(  # noqa: E731
        q=q[a * KL:b * KL], k_new=kn[a * KL:b * KL], v_new=vn[a * KL:b * KL], k_cache=kc, v_cache=vc, req_to_token=table,
        req_pool_indices=rows[a:b], ctx_lens=lens[a:b], num_modes=K, block_size=L, scaling=D ** -0.5, num_ctx_splits=0,
        page_size=page)
    out = call(0, bs)
    torch.cuda.synchronize()
    for a in range(0, bs, 60):
        b = min(a + 60, bs)
        assert torch.equal(call(a, b).view(torch.int16), out[a * KL:b * KL].view(torch.int16))
