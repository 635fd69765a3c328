"""GPU parity of the 8-bit draft KV cache (store, attention, token weights, selection, compaction) with the float64 oracle.

Tolerances. Codes, scales and kept positions are exact. Attention: the probabilities are rounded to fp16 (half a step:
2^-11 of each), a split's partial row to fp16 again (2^-11 of the row), scores and sums are fp32 (a score of size B =
scale sum |q_d k_d|: 128 additions, 128 2^-24 B, at most 2^-12 at the sizes here), and the output to bf16 (2^-8 of itself):
  |out - ref| <= 2^-8 |ref| + (2^-11 + 2^-11 + 2^-12) sum p |v|
lse: the score's error, and the roundings of a sum, a logarithm and two products: 2^-24 (128 B + 8 |lse| + 8).
Weights: each probability carries its score's and its lse's error, and a few fp32 roundings of the exponential and sums.
"""

import numpy as np
import pytest
import torch

from oracle import kv8

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
D = 128


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def make_pool(lens, page, hkv, seed, spread=1.0, extra=0):
    """CPU tensors of a filled pool: codes, scales, page table (rows in reverse order, one row unused), and a second table
    of `extra` pages per request."""
    g = _gen(seed)
    need = [-(-max(n, 1) // page) for n in lens]
    total = sum(need) + extra * len(lens) + 3
    perm = torch.randperm(total, generator=g).to(torch.int32)
    width = max(need)
    table = torch.full((len(lens) + 1, width), 2 ** 30, dtype=torch.int32)  # entries past a request: never a page id
    dst = torch.full((len(lens) + 1, max(extra, 1)), 2 ** 30, dtype=torch.int32)
    rows = torch.arange(len(lens), 0, -1)
    at = 0
    for b, n in enumerate(need):
        table[rows[b], :n] = perm[at:at + n]
        at += n
        dst[rows[b], :extra] = perm[at:at + extra]
        at += extra
    d = dict(page=page, table=table, dst=dst, rows=rows, lens=torch.tensor(lens))
    for x in "kv":
        codes = (torch.randn(total * page, hkv, D, generator=g) * 60).clamp(-448, 448).to(F8)
        # scales a factor of 2^6 apart between neighbouring pages: the accumulators' unit changes all the time
        scale = torch.exp2(torch.randint(-8, -2, (total, hkv), generator=g).float()) * spread
        d[x + "_cache"], d[x + "_scale"] = codes, scale
    return d


def cache_args(d, dev="cuda"):
    return dict(k_cache=d["k_cache"].to(dev), v_cache=d["v_cache"].to(dev), k_scale=d["k_scale"].to(dev),
                v_scale=d["v_scale"].to(dev), page_size=d["page"], req_pool_indices=d["rows"].to(dev))


def vals(t):
    return t.cpu().float().numpy().astype(np.float64)


def oracle_attention(d, q, kn, vn, lens, K, L, scaling, causal):
    KL = K * L
    parts = []
    for b, n in enumerate(lens):
        kc = kv8.tokens(vals(d["k_cache"]), vals(d["k_scale"]), d["table"][d["rows"][b]].numpy(), n, d["page"])
        vc = kv8.tokens(vals(d["v_cache"]), vals(d["v_scale"]), d["table"][d["rows"][b]].numpy(), n, d["page"])
        r = slice(b * KL, (b + 1) * KL)
        parts.append(kv8.attention(vals(q[r]), vals(kn[r]) if kn is not None else None,
                                   vals(vn[r]) if vn is not None else None, kc, vc, K, L, scaling, causal))
    return [np.concatenate(x) for x in zip(*parts)]


def check_attention(out, lse, ref):
    o, l, mass, size = ref
    got, gl = vals(out), vals(lse)
    seen = np.isfinite(l)
    err = np.abs(got - o) - 2.0 ** -8 * np.abs(o) - (2 * 2.0 ** -11 + 2.0 ** -12) * mass
    assert np.isfinite(got).all() and (err <= 1e-30).all(), float(err.max())
    assert np.array_equal(np.isneginf(gl), ~seen)
    lerr = np.abs(np.where(seen, gl, 0) - np.where(seen, l, 0))
    assert (lerr <= 2.0 ** -24 * (128 * size + 8 * np.abs(np.where(seen, l, 0)) + 8)).all(), float(lerr.max())


ATTN = [
    # lens, K, L, H, Hkv, page, fresh, causal, splits
    ([1], 1, 1, 8, 8, 16, False, False, -1),                          # one key, one row
    ([0, 5], 1, 1, 8, 2, 16, False, False, -1),                       # a request without any key
    ([0, 0], 2, 3, 4, 2, 16, False, False, 3),
    ([0, 3], 1, 1, 4, 2, 64, True, False, 2),                         # its own key alone
    ([37, 64, 65, 31, 32, 33], 1, 1, 32, 8, 64, True, False, -1),     # tile borders, stream kernel
    ([700, 129, 1300], 1, 1, 40, 8, 16, False, False, 4),             # five rows a head, small pages, splits
    ([2000], 1, 1, 64, 8, 128, True, False, -1),
    ([300, 17], 1, 16, 4, 2, 32, True, True, -1),                     # 32 rows: the largest stream case; causal
    ([300, 17, 0], 4, 7, 8, 2, 32, True, False, 2),                   # 112 rows: four units, the last one padded
    ([129, 63, 64], 3, 16, 16, 8, 64, True, False, -1),               # 96 rows: an idle wave
    ([1000], 8, 16, 32, 8, 64, True, False, -1),                      # eight-wave workgroups
    ([1000, 0, 191], 8, 16, 32, 8, 64, True, True, 0),
    ([513, 64], 8, 16, 40, 8, 16, True, False, 3),                    # 20 units, 16-token pages
    ([130], 2, 40, 4, 2, 256, True, False, 1),                        # blocks of 40: modes cross units and tiles
    ([90], 1, 150, 2, 1, 32, True, True, 2),                          # one long causal block over three tiles
    ([200, 1], 1, 5, 26, 2, 64, False, False, -1),                    # 65 rows without block keys
    ([3000, 0, 700, 5000], 8, 16, 8, 2, 64, True, False, -1),               # splits measured out by the lengths
    ([0, 0, 0], 4, 16, 8, 2, 64, True, True, -1), ([9000, 1], 3, 16, 4, 1, 32, False, False, -1),
    ([i * 37 % 1500 for i in range(64)], 1, 40, 2, 1, 16, True, False, -1),  # .. of as many requests as a wave has lanes
    ([2000 * (i % 7) + i for i in range(16)], 1, 1, 32, 8, 64, True, False, -1),
    ([500 + i * 90 for i in range(65)], 1, 1, 8, 2, 64, False, False, -1),   # .. and one more than that
    ([64 + 7 * i for i in range(16)], 2, 16, 40, 8, 64, True, False, -1),   # a batch with idle waves: five units
    ([3 + 11 * i for i in range(16)], 1, 40, 40, 8, 32, True, True, 2),     # .. seven, small pages, splits
    ([1 + 17 * i % 97 for i in range(40)], 1, 1, 32, 8, 16, True, False, 1),  # plain decoding, more workgroups than CUs
    ([9 + 31 * i % 200 for i in range(40)], 1, 3, 32, 8, 64, False, False, -1),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(case):
    import kv8_cache

    lens, K, L, H, Hkv, page, fresh, causal, splits = ATTN[case]
    print(f"case: kv8 attention {ATTN[case]}", flush=True)
    d = make_pool(lens, page, Hkv, seed=case)
    g = _gen(100 + case)
    T = len(lens) * K * L
    q = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    kn = torch.randn(T, Hkv, D, generator=g).to(torch.bfloat16) if fresh else None
    vn = torch.randn(T, Hkv, D, generator=g).to(torch.bfloat16) if fresh else None
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = kv8_cache.paged_mode_block_attention_kv8(
        q=q.cuda(), k_new=kn.cuda() if fresh else None, v_new=vn.cuda() if fresh else None, page_table=d["table"].cuda(),
        ctx_lens=d["lens"].cuda(), num_modes=K, block_size=L, scaling=D ** -0.5, num_ctx_splits=splits,
        causal_in_block=causal, return_lse=True, err_flag=flag, **cache_args(d))
    torch.cuda.synchronize()
    assert int(flag) == 0
    check_attention(out, lse, oracle_attention(d, q, kn, vn, lens, K, L, D ** -0.5, causal))


WEIGHTS = [
    # lens, K, L, H, Hkv, page, width, decay
    ([1], 1, 1, 8, 8, 16, 1, 1.0),
    ([0, 5, 300], 1, 1, 8, 2, 16, 300, 0.5),
    ([256, 257, 255], 1, 5, 26, 2, 64, 400, 0.9),
    ([700, 64], 8, 16, 32, 8, 64, 700, 0.0),
    ([77, 500], 3, 16, 40, 8, 32, 501, 1.0),
    ([5003], 2, 16, 32, 8, 64, 5003, 0.5), ([4999], 1, 9, 32, 8, 16, 5100, 1.0),  # one request, more than one round of the smallest
    ([8500, 1, 130], 4, 16, 40, 8, 64, 8500, 1.0), ([130, 9001], 1, 33, 8, 8, 128, 9100, 0.7),  # more workgroups than CUs
    ([300], 1, 33, 2, 2, 64, 300, 0.3), ([100], 1, 161, 1, 1, 32, 200, 1.0),                   # two and six units
]


@pytest.mark.parametrize("case", range(len(WEIGHTS)))
def test_weights(case):
    import kv8_cache

    lens, K, L, H, Hkv, page, width, decay = WEIGHTS[case]
    print(f"case: kv8 weights {WEIGHTS[case]}", flush=True)
    d = make_pool(lens, page, Hkv, seed=50 + case)
    g = _gen(150 + case)
    KL = K * L
    q = torch.randn(len(lens) * KL, H, D, generator=g).to(torch.bfloat16)
    _, lse, _, size = oracle_attention(d, q, None, None, lens, K, L, D ** -0.5, False)
    lse32 = torch.from_numpy(lse).float()
    old = torch.rand(len(lens) + 1, Hkv, width + 3, generator=g)
    if decay == 0.0:
        old[:, :, 1] = float("nan")  # not read
    w = old.cuda()[:, :, :width]  # rows with a stride of their own
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = cache_args(d)
    del args["v_cache"], args["v_scale"]
    kv8_cache.attention_weights_kv8(q=q.cuda(), lse=lse32.cuda(), page_table=d["table"].cuda(), ctx_lens=d["lens"].cuda(),
                                    num_modes=K, block_size=L, scaling=D ** -0.5, weights=w, decay=decay, err_flag=flag,
                                    **args)
    torch.cuda.synchronize()
    assert int(flag) == 0
    got, before = vals(w), vals(old)[:, :, :width]
    for b, n in enumerate(lens):
        row = int(d["rows"][b])
        kc = kv8.tokens(vals(d["k_cache"]), vals(d["k_scale"]), d["table"][row].numpy(), n, page)
        add = kv8.weights(vals(q[b * KL:(b + 1) * KL]), vals(lse32[b * KL:(b + 1) * KL]), kc, D ** -0.5)
        ref = add + (decay * before[row, :, :n] if decay else 0)
        l = lse[b * KL:(b + 1) * KL]
        rel = 2.0 ** -24 * (128 * size[b * KL:(b + 1) * KL].max() + 8 * np.abs(l[np.isfinite(l)]).max(initial=0) + 16 + KL)
        assert (np.abs(got[row, :, :n] - ref) <= rel * ref + 1e-35).all(), (b, float(np.abs(got[row, :, :n] - ref).max()))
        assert np.array_equal(got[row, :, n:], before[row, :, n:], equal_nan=True)  # behind a request: as they were
    assert np.array_equal(got[0], before[0], equal_nan=True)  # the row of nobody


STORE = [
    # start, new, hkv, page
    ([0], [1], 2, 16), ([5, 0, 63, 64, 100], [1, 64, 1, 3, 29], 2, 64), ([0, 17], [300, 40], 4, 32),
    ([127, 3, 0], [130, 0, 128], 8, 128), ([250, 1], [10, 300], 2, 256), ([15, 16, 31], [1, 1, 40], 1, 16),
]


@pytest.mark.parametrize("case", range(len(STORE)))
def test_store(case):
    import kv8_cache

    start, new, hkv, page = STORE[case]
    print(f"case: kv8 store {STORE[case]}", flush=True)
    lens = [a + n for a, n in zip(start, new)]
    d = make_pool(lens, page, hkv, seed=200 + case)
    g = _gen(250 + case)
    N = sum(new)
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    # magnitudes from 2^-12 to 2^8 of the old scales', exact ties, zero rows, infinities and NaN among them
    x = {}
    for which in "kv":
        t = torch.randn(N + 2, hkv, D, generator=g) * torch.exp2(torch.randint(-12, 9, (N + 2, hkv, 1), generator=g).float())
        t[0, 0, :8] = torch.tensor([1.0, -1.0, 1.0625, 1.1875, 0.0, -0.0, 2.0 ** -9, 3 * 2.0 ** -11])
        t[N // 2, hkv - 1] = 0
        t[N - 1, 0, 5], t[N - 1, 0, 6], t[N - 1, 0, 7] = float("inf"), float("-inf"), float("nan")
        x[which] = t.to(torch.bfloat16)
    args = cache_args(d)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    dev = {w: x[w].cuda()[1:N + 1] if w == "v" else x[w].cuda()[:N] for w in "kv"}
    kv8_cache.kv8_store(k=dev["k"], v=dev["v"], page_table=d["table"].cuda(), start_lens=torch.tensor(start).cuda(),
                        cu_tokens=cu.cuda(), max_tokens=max(new), err_flag=flag, **args)
    torch.cuda.synchronize()
    assert int(flag) == 0
    for w in "kv":
        cache, scale = vals(d[w + "_cache"]), vals(d[w + "_scale"])
        kv8.store(vals(dev[w]), cache, scale, d["table"].numpy(), d["rows"].numpy(), start, cu.numpy(), page)
        assert np.array_equal(vals(args[w + "_scale"]), scale), w
        got = vals(args[w + "_cache"])
        assert np.array_equal(got, cache, equal_nan=True), (w, np.argwhere(~((got == cache) | np.isnan(cache)))[:4])


def test_store_token_by_token_is_attended_to():
    """A sequence written one token at a time holds, in each page, its tokens to within the type's half step of the page's
    scale, also where the scale grew on the way."""
    import kv8_cache

    page, hkv, n = 16, 2, 53
    d = make_pool([n], page, hkv, seed=300)
    g = _gen(301)
    x = (torch.randn(n, hkv, D, generator=g) * torch.linspace(0.01, 40, n)[:, None, None]).to(torch.bfloat16)
    args = cache_args(d)
    for t in range(n):
        row = x[t:t + 1].cuda()
        kv8_cache.kv8_store(k=row, v=-row, page_table=d["table"].cuda(), start_lens=torch.tensor([t]).cuda(),
                            cu_tokens=torch.tensor([0, 1], dtype=torch.int32).cuda(), max_tokens=1, **args)
    torch.cuda.synchronize()
    row = d["table"][d["rows"][0]].numpy()
    k = kv8.tokens(vals(args["k_cache"]), vals(args["k_scale"]), row, n, page)
    v = kv8.tokens(vals(args["v_cache"]), vals(args["v_scale"]), row, n, page)
    pages = row[np.arange(n) // page]
    s = vals(args["k_scale"])[pages][:, :, None]
    # every rounding is to a grid of which the next one is a part, but in the subnormal range, where each of the (at most
    # 15) regrowths adds half a step of 2^-9 scaled by its own, smaller, scale: their sum stays below one final step
    assert (np.abs(k - vals(x)) <= 2.0 ** -4 * np.abs(vals(x)) + 2.0 ** -9 * s).all()
    assert np.array_equal(v, -k)


def _weights_for_selection(g, rows, hkv, width, kind):
    if kind == "ties":
        return torch.randint(0, 3, (rows, hkv, width), generator=g).float()
    if kind == "zero":
        return torch.zeros(rows, hkv, width)
    w = torch.exp(3 * torch.randn(rows, hkv, width, generator=g))
    if kind == "odd":
        w[:, 0, ::7] = float("nan")
        w[:, 0, 3::11] = float("inf")
        w[:, hkv - 1, 5::13] = -1e30
        w[:, 0, 6::17] = -0.0
    return w


EVICT = [
    # lens, budget, sink, recent, hkv, page, weights
    ([100, 7, 0, 64], 20, 4, 8, 2, 16, "normal"), ([1000, 300, 301], 300, 4, 32, 8, 64, "ties"),
    ([500], 64, 0, 0, 1, 16, "zero"), ([4100, 5000], 1025, 4, 32, 2, 32, "normal"), ([77], 1, 0, 0, 3, 16, "normal"),
    ([300, 5], 40, 40, 0, 2, 64, "ties"), ([300], 36, 4, 32, 2, 128, "normal"), ([900, 640], 200, 3, 5, 2, 256, "odd"),
    ([8187, 9000], 3000, 4, 32, 9, 64, "ties"), ([9000, 16379], 2500, 4, 32, 2, 64, "odd"),  # keys in 8 and 16 registers
    ([20000, 16385, 900], 1500, 4, 32, 3, 64, "odd"), ([17000], 16000, 0, 1, 1, 128, "ties"),  # .. and in the workspace
]


@pytest.mark.parametrize("case", range(len(EVICT)))
def test_eviction(case):
    import kv8_cache

    lens, budget, sink, recent, hkv, page, kind = EVICT[case]
    print(f"case: kv8 eviction {EVICT[case]}", flush=True)
    d = make_pool(lens, page, hkv, seed=400 + case, extra=-(-budget // page))
    g = _gen(450 + case)
    width = max(lens) + 5
    w = _weights_for_selection(g, len(lens) + 1, hkv, width, kind)
    args = cache_args(d)
    dw = w.cuda()
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep, new = kv8_cache.evict_select(weights=dw, req_pool_indices=args["req_pool_indices"], ctx_lens=d["lens"].cuda(),
                                       budget=budget, sink=sink, recent=recent, err_flag=flag)
    kv8_cache.evict_compact_kv8(keep=keep, new_lens=new, ctx_lens=d["lens"].cuda(), src_table=d["table"].cuda(),
                                dst_table=d["dst"].cuda(), weights=dw, err_flag=flag, **args)
    torch.cuda.synchronize()
    assert int(flag) == 0
    ref_w = w.numpy().copy()
    for x in "kv":
        d[x + "_ref"] = (vals(d[x + "_cache"]), vals(d[x + "_scale"]))
    for b, n in enumerate(lens):
        row = int(d["rows"][b])
        kept = kv8.select(w[row].numpy(), n, budget, sink, recent)
        assert keep[b].tolist() == kept + [-1] * (budget - len(kept)) and int(new[b]) == len(kept), b
        for x in "kv":
            kv8.compact(*d[x + "_ref"], d["table"][row].numpy(), d["dst"][row].numpy(), kept, page)
        ref_w[row, :, :len(kept)] = w[row].numpy()[:, kept]
        ref_w[row, :, len(kept):n] = 0
    assert np.array_equal(dw.cpu().numpy(), ref_w, equal_nan=True)
    for x in "kv":
        assert np.array_equal(vals(args[x + "_cache"]), d[x + "_ref"][0], equal_nan=True), x
        assert np.array_equal(vals(args[x + "_scale"]), d[x + "_ref"][1]), x
