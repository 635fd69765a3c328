"""The 8-bit draft cache at the edges of what its calls allow: infinities beside very large and very small values in split
contexts, batches of thousands, counts and rows out of range, one workspace for many lengths, captured hooks, side streams.
Tolerances: those of test_gpu_kv8, with what _bounded derives."""

import numpy as np
import pytest
import torch

from oracle import kv8
from test_gpu_kv8 import D, F8, _gen, cache_args, check_attention, make_pool, oracle_attention, vals
from test_gpu_kv8_use import FORMS, SCALE, _attend, _bf, _guarded, _Step

pytestmark = pytest.mark.gpu


def _bounded(ref, d, lens, KL, G):
    """A reference whose ``mass`` covers fp16's subnormals too. Below 2^-14 half a step of fp16 is 2^-25. A probability p (of
    a row whose sum is at least 1) enters as fp16(p 2^q), q >= -2: off by 2^-23 of the sum at most, 2^-23 sum |v| over the
    cached keys. A split's partial row is rounded after a power of two has brought its largest finite component m into
    [1/2, 1): off by 2^-24 m there, and its share of that in the result, at most 2^-24 of the row's largest mass for each of
    up to four partials. check_attention takes (2 2^-11 + 2^-12) of ``mass``, so they are added divided by that."""
    o, lse, mass, most = ref
    for b, n in enumerate(lens):
        v = kv8.tokens(vals(d["v_cache"]), vals(d["v_scale"]), d["table"][d["rows"][b]].numpy(), n, d["page"])
        m = mass[b * KL:(b + 1) * KL]
        more = np.abs(v).sum(0).repeat(G, 0) * 2.0 ** -23 + m.max(-1, keepdims=True) * 2.0 ** -22
        m += more / (2 * 2.0 ** -11 + 2.0 ** -12)
    return o, lse, mass, most


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("size", [24, -30])
def test_an_infinity_leaves_its_neighbours(form, size):
    """Infinities in single components of one mode's block values, the others about 2^24 (beyond fp16's largest) or 2^-30 (below
    its smallest): whatever the number of splits, the infinite components are infinite in the rows that see them, and all others
    are what they are without it."""
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
    ref = _bounded(oracle_attention(d, q, kn, vn, lens, K, L, SCALE, causal), d, lens, KL, G)
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
            out[t:t + L, h * G:(h + 1) * G, c] = torch.from_numpy(ref[0][t:t + L, h * G:(h + 1) * G, c]).to(torch.bfloat16)
        check_attention(out, lse, ref)


@pytest.mark.parametrize("K,L,H,splits", [(1, 1, 4, 1), (1, 1, 4, 2), (2, 20, 2, 1), (2, 20, 2, 2)])
def test_a_batch_of_thousands(K, L, H, splits):
    """Thousands of requests in one call (every seventh compared)."""
    import kv8_cache

    bs, page, Hkv, KL = 3001, 16, 2, K * L
    print(f"case: kv8 attention of {bs} requests {K} x {L} splits={splits}", flush=True)
    g = _gen(830)
    lens = torch.randint(0, 200, (bs,), generator=g)
    pages = 200
    d = make_pool([page * pages], page, Hkv, seed=831)
    d.update(table=torch.randint(0, pages, (bs, -(-200 // page)), generator=g).int(), rows=torch.arange(bs))  # shared pages
    q, kn, vn = _bf(g, bs * KL, H, D), _bf(g, bs * KL, Hkv, D), _bf(g, bs * KL, Hkv, D)
    out, lse = kv8_cache.paged_mode_block_attention_kv8(
        q=q.cuda(), k_new=kn.cuda(), v_new=vn.cuda(), page_table=d["table"].cuda(), ctx_lens=lens.cuda(), num_modes=K,
        block_size=L, scaling=SCALE, num_ctx_splits=splits, max_ctx=200, return_lse=True, **cache_args(d))
    some = torch.arange(0, bs, 7)
    of = lambda t: t.cpu().view(bs, KL, -1, D)[some].reshape(len(some) * KL, -1, D)  # noqa: E731
    d["rows"], n = some, lens[some].tolist()
    ref = _bounded(oracle_attention(d, of(q), of(kn), of(vn), n, K, L, SCALE, False), d, n, KL, H // Hkv)
    check_attention(of(out), lse.cpu().view(bs, KL, H)[some].reshape(-1, H), ref)


def test_counts_rows_and_lengths_out_of_range_are_reported():
    """Whatever a call cuts to what its tensors hold, it says so in its error flag: the store's token counts and positions, the
    compaction's counts, lengths and rows (of the table, and of the sums), and rows of requests that have nothing to do. The other
    request's result keeps its bits, and nothing outside the tensors is written."""
    import kv8_cache
    import mfd_hip

    page, Hkv, H, lens, budget = 64, 2, 4, [300, 200], 100
    d = make_pool(lens, page, Hkv, seed=840, extra=2)
    g = _gen(841)
    k, v, q = _bf(g, 9, Hkv, D).cuda(), _bf(g, 9, Hkv, D).cuda(), _bf(g, 4, H, D).cuda()
    table, dst = d["table"].cuda(), d["dst"].cuda()
    keep = torch.stack([torch.arange(budget) * 2, torch.arange(budget)]).int().cuda()
    i64 = lambda *x: torch.tensor(x).cuda()  # noqa: E731

    def run(call, **kw):
        """(the flag, request 0's pages, request 0's sums)"""
        args, guards = {}, []
        for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
            args[name], buf = _guarded(d[name])
            guards.append(buf)
        w, buf = _guarded(kw.pop("sums", torch.ones(3, Hkv, 300)))
        guards.append(buf)
        args.update(page_size=page, req_pool_indices=d["rows"].cuda(), err_flag=torch.zeros(1, dtype=torch.int32).cuda())
        if call == "store":
            args.update(k=k, v=v, page_table=table, start_lens=i64(290, 60), max_tokens=9,
                        cu_tokens=torch.tensor([0, 3, 9], dtype=torch.int32).cuda())
            kv8_cache.kv8_store(**{**args, **kw})
        elif call == "compact":
            args.update(keep=keep, new_lens=i64(budget, budget), ctx_lens=i64(*lens), src_table=table, dst_table=dst, weights=w)
            kv8_cache.evict_compact_kv8(**{**args, **kw})
        else:
            args.update(q=q, page_table=table, ctx_lens=i64(*lens), num_modes=1, block_size=2, scaling=SCALE)
            if call == "attn":
                kv8_cache.paged_mode_block_attention_kv8(k_new=None, v_new=None, **{**args, **kw})
            else:
                del args["v_cache"], args["v_scale"]
                kv8_cache.attention_weights_kv8(lse=torch.ones(4, H).cuda(), weights=w, **{**args, **kw})
        torch.cuda.synchronize()
        for buf in guards:
            assert bool((buf[:4096] == 0x5A).all()) and bool((buf[-4096:] == 0x5A).all())
        pages = torch.cat([t[d["rows"][0].item()].long() for t in (d["table"][:, :5], d["dst"])]).cuda()
        caches = [args[x + "_cache"].view(torch.uint8).view(-1, page, Hkv, D)[pages] for x in "kv" if x + "_cache" in args]
        return int(args["err_flag"]), caches, w[2].clone()

    cu = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    r0 = int(d["rows"][0])
    rows = [i64(r0, r) for r in (-1, 3, 2 ** 40)]
    bad = {
        "store": [dict(cu_tokens=cu(0, 3, 10)), dict(cu_tokens=cu(0, 3, 2 ** 31 - 1)), dict(cu_tokens=cu(0, 3, 2)),
                  dict(cu_tokens=cu(0, 3, -5)), dict(start_lens=i64(290, -1), cu_tokens=cu(0, 3, 3)),
                  *(dict(req_pool_indices=r, cu_tokens=cu(0, 3, 3)) for r in rows)],
        "compact": [*(dict(new_lens=i64(budget, n)) for n in (-1, budget + 1, 2 ** 62, -2 ** 62)),
                    *(dict(ctx_lens=i64(300, n)) for n in (-1, 10 ** 6, 2 ** 62, -2 ** 62)),
                    *(dict(req_pool_indices=r, new_lens=i64(budget, 0)) for r in rows),
                    *(dict(req_pool_indices=r, new_lens=i64(budget, 0), ctx_lens=i64(300, 0), weights=None) for r in rows)],
        "attn": [dict(req_pool_indices=r, ctx_lens=i64(300, 0)) for r in rows],
        "weights": [dict(req_pool_indices=r, ctx_lens=i64(300, 0)) for r in rows],
    }
    for call, changes in bad.items():
        flag, caches, sums = run(call)
        assert flag == 0
        for change in changes:
            print(f"case: kv8 {call} out of range", {x: t if t is None else t.tolist() for x, t in change.items()}, flush=True)
            f, c, s = run(call, **change)
            assert f == mfd_hip.DEVERR_BAD_PAGE
            assert all(torch.equal(x, y) for x, y in zip(caches, c))
            assert "weights" in change or torch.equal(s, sums)
    # sums with fewer rows, or narrower ones, than the requests have
    assert run("compact", sums=torch.ones(3, Hkv, 299))[0] == mfd_hip.DEVERR_BAD_PAGE
    few = torch.ones(2, Hkv, 300).cuda()  # (request 0 is in row 2)
    assert run("compact", weights=few)[0] == mfd_hip.DEVERR_BAD_PAGE


@pytest.mark.parametrize("K,L,splits", [(1, 1, -1), (8, 16, -1), (8, 16, 32)])
def test_one_workspace_for_many_lengths(K, L, splits):
    """A buffer sized once, for one token more than the table's rows hold, serves calls without max_ctx and with smaller ones."""
    import kv8_cache

    page, Hkv, H = 64, 8, 32
    table_reach = 2048 if K == 1 else 16128
    print(f"case: kv8 workspace {K} x {L} splits={splits}", flush=True)
    d = make_pool([table_reach], page, Hkv, seed=850)
    g = _gen(851)
    T = K * L
    q, kn, vn = _bf(g, T, H, D).cuda(), _bf(g, T, Hkv, D).cuda(), _bf(g, T, Hkv, D).cuda()
    size = kv8_cache.workspace_bytes(bs=1, num_modes=K, block_size=L, num_heads=H, num_kv_heads=Hkv, with_block=True,
                                     max_ctx=table_reach + 1, num_ctx_splits=splits)
    ws = torch.full((size + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    args = cache_args(d)
    for n, most in ((table_reach, None), (table_reach, table_reach), (2047, 2048), (1000, 1900), (500, 2881), (0, 1)):
        d["lens"][0] = n
        o0, l0 = _attend(d, args, q, kn, vn, K, L, num_ctx_splits=splits, max_ctx=most)
        o1, l1 = _attend(d, args, q, kn, vn, K, L, num_ctx_splits=splits, max_ctx=most, workspace=ws[:size])
        assert torch.equal(o0.view(torch.int16), o1.view(torch.int16)) and torch.equal(l0, l1)
    assert bool((ws[size:] == 0x5A).all())


@pytest.mark.parametrize("K,L,H", [(1, 1, 8), (4, 16, 8)])
def test_a_captured_hook_splits_for_the_table(monkeypatch, K, L, H):
    """PagedModeAttention captured with the lengths of an empty batch (as engines capture it), replayed with others: the splits
    are those of what the table holds, not of the lengths at capture, and the results an eager call's."""
    import kv8_cache
    import paged_mode_attention

    page, Hkv, bs = 64, 2, 3
    d = make_pool([1500, 700, 1100], page, Hkv, seed=860)
    g = _gen(861)
    T, args = bs * K * L, cache_args(d)
    q, k, v = (_bf(g, T, n * D).cuda() for n in (H, Hkv, Hkv))
    pool = kv8_cache.Kv8Pool(num_layers=1, num_pages=d["k_scale"].shape[0], page_size=page, num_kv_heads=Hkv)
    pool.caches, pool.scales = [(args["k_cache"], args["v_cache"])], [(args["k_scale"], args["v_scale"])]
    lens = torch.ones(bs, dtype=torch.int64).cuda()
    batch = type("Batch", (), dict(req_pool_indices=d["rows"].cuda(), seq_lens=lens,
                                   seq_lens_cpu=torch.ones(bs, dtype=torch.int64)))
    hook = paged_mode_attention.PagedModeAttention(
        kv_pool=pool, req_to_token=d["table"].cuda(), num_modes=K, block_size=L, num_heads=H, num_kv_heads=Hkv, head_dim=D,
        scaling=SCALE, num_ctx_splits=-1, impl="hip", page_size=page)
    given, attention = [], kv8_cache.paged_mode_block_attention_kv8
    monkeypatch.setattr(kv8_cache, "paged_mode_block_attention_kv8",
                        lambda **kw: given.append(kw["max_ctx"]) or attention(**kw))
    hook(q, k, v, batch, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hook(q, k, v, batch, 0)
    assert given == [1, None]
    for now in ([1500, 700, 1100], [0, 64, 1], [1499, 0, 1100], [3, 3, 3]):
        lens.copy_(torch.tensor(now))
        batch.seq_lens_cpu = None
        eager = hook(q, k, v, batch, 0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))


def _operators():
    """{name: (inputs by name, what the call changes or returns, the call)} on one round's static buffers. Every input is one that
    is in range under both of its values below."""
    import ddtree_sglang_ops
    import kv8_cache
    import mxfp4_head
    import paged_mode_attention

    s = _Step(870)
    a = s.args
    cache = {x: a[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")}
    index = dict(page_size=s.page, req_pool_indices=a["req_pool_indices"])
    sizes = dict(num_modes=s.K, block_size=s.L, scaling=SCALE, page_table=s.table, ctx_lens=s.ctx)
    rows = s.out.view(-1, s.H * D)
    s.out.copy_(s.q)
    s.lse.fill_(6.0)
    s.w.copy_(torch.rand(s.w.shape, generator=_gen(871)))
    s.keep.copy_(torch.arange(100) * 3 % 300)
    s.keep.copy_(s.keep.sort(1).values.clamp(max=128))
    s.new.fill_(100)
    pool = kv8_cache.Kv8Pool(num_layers=1, num_pages=a["k_scale"].shape[0], page_size=s.page, num_kv_heads=s.Hkv)
    pool.caches, pool.scales = [(a["k_cache"], a["v_cache"])], [(a["k_scale"], a["v_scale"])]
    batch = type("Batch", (), dict(req_pool_indices=a["req_pool_indices"].int(), seq_lens=s.ctx.int()))
    hook = paged_mode_attention.PagedModeAttention(
        kv_pool=pool, req_to_token=s.table, num_modes=s.K, block_size=s.L, num_heads=s.H, num_kv_heads=s.Hkv, head_dim=D,
        scaling=SCALE, num_ctx_splits=3, impl="hip", page_size=s.page)
    head = ddtree_sglang_ops.DDTreeDraftTopK(weight=mxfp4_head.Mxfp4Weight(s.codes, s.exps), block_size=s.L, num_modes=s.K,
                                             budget=17, max_bs=2)
    flat = lambda t: t.view(t.shape[0], -1)  # noqa: E731
    qkv = dict(q=s.q, kn=s.kn, vn=s.vn)
    return {
        "attention": (dict(qkv, **cache), (s.out, s.lse), lambda: kv8_cache.paged_mode_block_attention_kv8(
            q=s.q, k_new=s.kn, v_new=s.vn, out=s.out, lse_out=s.lse, num_ctx_splits=3, **cache, **index, **sizes)),
        "hook": (dict(qkv, **cache), (), lambda: hook(flat(s.q), flat(s.kn), flat(s.vn), batch, 0)),
        "weights": (dict(q=s.q, lse=s.lse, w=s.w, k_cache=a["k_cache"], k_scale=a["k_scale"]), (s.w,),
                    lambda: kv8_cache.attention_weights_kv8(q=s.q, lse=s.lse, weights=s.w, decay=0.9, k_cache=a["k_cache"],
                                                            k_scale=a["k_scale"], **index, **sizes)),
        "store": (dict(kn=s.kn, vn=s.vn, **cache), tuple(cache.values()), lambda: kv8_cache.kv8_store(
            k=s.kn[:9], v=s.vn[:9], page_table=s.table, start_lens=s.ctx.int(), cu_tokens=s.cu, max_tokens=5, **cache, **index)),
        "select": (dict(w=s.w), (), lambda: torch.cat([t.flatten().long() for t in kv8_cache.evict_select(
            weights=s.w, req_pool_indices=a["req_pool_indices"], ctx_lens=s.ctx, budget=100)])),
        "select, narrow rows": (dict(w=s.w), (), lambda: kv8_cache.evict_select(
            weights=s.w[:, :, :300], req_pool_indices=a["req_pool_indices"].int(), ctx_lens=s.ctx, budget=100)[0]),
        "compact": (dict(keep=s.keep, w=s.w, **cache), (s.w, *cache.values()), lambda: kv8_cache.evict_compact_kv8(
            keep=s.keep, new_lens=s.new, ctx_lens=s.ctx, src_table=s.table, dst_table=s.dst, weights=s.w, **cache, **index)),
        "evict": (dict(w=s.w, **cache), (s.w, *cache.values()), lambda: pool.evict(
            weights=s.w, page_table=s.table, dst_table=s.dst, req_pool_indices=a["req_pool_indices"], ctx_lens=s.ctx,
            budget=100)[0]),
        "head": (dict(x=s.out), (), lambda: mxfp4_head.draft_head_mxfp4(rows, s.codes, s.exps)),
        "head of an unaligned view": (dict(x=s.out), (), lambda: mxfp4_head.draft_head_mxfp4(
            rows.view(-1)[1:-(s.H * D) + 1].view(-1, s.H * D), s.codes, s.exps)),
        "candidates": (dict(x=s.out), (head.top_logp, head.top_ids, head.log_z), lambda: head(rows)),
    }


NAMES = ["attention", "hook", "weights", "store", "select", "select, narrow rows", "compact", "evict", "head",
         "head of an unaligned view", "candidates"]


@pytest.mark.parametrize("name", NAMES)
def test_each_operator_runs_on_the_current_stream(name):
    """An operator on a side stream behind a long wait and the copies that bring its inputs: a launch on any other stream would
    read what the inputs held before, which gives another result (the first assertion)."""
    print(f"case: side stream, {name}", flush=True)
    inputs, changed, call = _operators()[name]
    true = {k: t.clone() for k, t in inputs.items()}

    def other(k, t):
        if k == "keep":
            return (t + 1).clamp(max=128)
        return t.view(torch.uint8).flip(0).view(t.dtype) if t.dtype == F8 else t.flip(0)

    false = {k: other(k, t) for k, t in true.items()}

    def run():
        res = call()
        return [t.clone().view(torch.uint8) for t in (*changed, *([res] if torch.is_tensor(res) else []))]

    def put(values):
        for k, t in inputs.items():
            t.view(torch.uint8).copy_(values[k].view(torch.uint8))

    put(false)
    wrong = run()
    put(true)
    right = run()
    put(false)
    for t in changed:
        if not any(t is x for x in inputs.values()):
            t.zero_()
    torch.cuda.synchronize()
    assert any(not torch.equal(x, y) for x, y in zip(wrong, right))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        put(true)
        got = run()
    assert not side.query()  # (it still waits: nothing above has begun)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(right, got))


def test_one_token_and_one_head_have_no_stride():
    """Slices of one token out of a projection of odd width, and of one head: the strides of axes with one entry mean nothing. The
    bits are those of contiguous tensors."""
    import kv8_cache

    page = 64
    print("case: kv8 one token, one head", flush=True)
    d = make_pool([300], page, 1, seed=880)
    g = _gen(881)
    index = dict(page_table=d["table"].cuda(), req_pool_indices=d["rows"].cuda())
    wide = _bf(g, 1, 3 * D + 1).cuda()
    one = lambda i: wide[:, i * D:(i + 1) * D].as_strided((1, 1, D), (3 * D + 1, 3 * D + 1, 1), i * D)  # noqa: E731
    results = []
    for q, k, v in ((one(0), one(1), one(2)), tuple(one(i).clone(memory_format=torch.contiguous_format) for i in range(3))):
        args = cache_args(d)
        buf = torch.full((2, 3 * D + 1), 3.0, dtype=torch.bfloat16, device="cuda")
        out = buf.as_strided((1, 1, D), (3 * D + 1, 3 * D + 1, 1))
        _, lse = _attend(d, args, q, k, v, 1, 1, out=out)
        assert bool((buf[0, D:] == 3).all()) and bool((buf[1] == 3).all())
        w = torch.zeros(2, 1, 300, device="cuda")
        wargs = {x: args[x] for x in ("k_cache", "k_scale", "page_size")}
        kv8_cache.attention_weights_kv8(q=q, lse=lse, ctx_lens=d["lens"].cuda(), num_modes=1, block_size=1, scaling=SCALE,
                                        weights=w, **wargs, **index)
        kv8_cache.kv8_store(k=k, v=v, start_lens=torch.tensor([290]).cuda(), max_tokens=1, **index,
                            cu_tokens=torch.tensor([0, 1], dtype=torch.int32).cuda(),
                            **{x: y for x, y in args.items() if x != "req_pool_indices"})
        results.append([t.clone().contiguous().view(torch.uint8) for t in (
            out, lse, w, args["k_cache"], args["v_cache"], args["k_scale"], args["v_scale"])])
    assert all(torch.equal(x, y) for x, y in zip(*results))
