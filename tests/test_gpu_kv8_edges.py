"""The 8-bit draft cache at the edges of what its calls allow: infinities beside very large and very small values in split
contexts. Tolerances: those of test_gpu_kv8 and test_gpu_kv8_use, derived there."""

import numpy as np
import pytest
import torch

from oracle import kv8
from test_gpu_kv8 import D, _gen, cache_args, check_attention, make_pool, oracle_attention, vals
from test_gpu_kv8_use import FORMS, SCALE, _attend, _bf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("size", [24, -30])
def test_an_infinity_leaves_its_neighbours(form, size):
    """Infinities in single components of one mode's block values, the others about 2^24 (beyond fp16's largest) or 2^-30 (below
    its smallest): whatever the number of splits, the infinite components are infinite in the rows that see them, and all others
    are what they are without it. The bound is test_value_scales_at_both_ends': a split's partial row is rounded to fp16 relative
    to its largest finite component."""
    K, L, H, Hkv, page, causal, _ = FORMS[form]
    print(f"case: kv8 infinity {FORMS[form]} 2^{size}", flush=True)
    lens, KL, G = [3 * page + 5, 0, 70], K * L, H // Hkv
    d = make_pool(lens, page, Hkv, seed=820 + form)
    d["v_scale"] *= 2.0 ** size
    g = _gen(821)
    T = len(lens) * KL
    q, kn, vn = _bf(g, T, H, D), _bf(g, T, Hkv, D), (torch.randn(T, Hkv, D, generator=g) * 2.0 ** size).to(torch.bfloat16)
    spots = [(b * KL + L, 0, c, s) for b in range(3) for c, s in ((5, 1), (66, -1))]  # the first key of every request's mode 1
    for t, h, c, s in spots:
        vn[t, h, c] = 0  # (the oracle's: a masked infinity would be 0 times infinity there)
    o, l, mass, most = oracle_attention(d, q, kn, vn, lens, K, L, SCALE, causal)
    for b, n in enumerate(lens):
        v = kv8.tokens(vals(d["v_cache"]), vals(d["v_scale"]), d["table"][d["rows"][b]].numpy(), n, page)
        m = mass[b * KL:(b + 1) * KL]
        more = np.abs(v).sum(0).repeat(G, 0) * 2.0 ** -23 + m.max(-1, keepdims=True) * 2.0 ** -24
        m += more / (2 * 2.0 ** -11 + 2.0 ** -12)
    bad = vn.clone()
    for t, h, c, s in spots:
        bad[t, h, c] = s * float("inf")
    for splits in (1, 2, 3):
        out, lse = _attend(d, cache_args(d), q.cuda(), kn.cuda(), bad.cuda(), K, L, num_ctx_splits=splits,
                           causal_in_block=causal)
        out = out.cpu().clone()
        for t, h, c, s in spots:
            seen = out[t:t + L, h * G:(h + 1) * G, c]
            assert bool((seen == s * float("inf")).all()), (splits, t, c)
            out[t:t + L, h * G:(h + 1) * G, c] = torch.from_numpy(o[t:t + L, h * G:(h + 1) * G, c]).to(torch.bfloat16)
        check_attention(out, lse, (o, l, mass, most))
