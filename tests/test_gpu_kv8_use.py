"""The 8-bit draft cache and the 4-bit head as they are used: captured in graphs and on another stream, through
PagedModeAttention and DDTreeDraftTopK, all operators in one run; and what must not matter to them: garbage in masked places,
ids and lengths out of range, strides and index types, caches beyond 4 GiB. Tolerances: those of test_gpu_kv8."""

import numpy as np
import pytest
import torch

from oracle import kv8
from test_gpu_kv8 import ATTN, D, F8, _gen, cache_args, check_attention, make_pool, oracle_attention, vals

pytestmark = pytest.mark.gpu

SCALE = D ** -0.5


def _bf(g, *shape):
    return torch.randn(*shape, generator=g).to(torch.bfloat16)


def _attend(d, args, q, kn, vn, K, L, **kw):
    import kv8_cache

    given = dict(page_table=d["table"].cuda(), ctx_lens=d["lens"].cuda(), num_modes=K, block_size=L, scaling=SCALE,
                 return_lse=True)
    return kv8_cache.paged_mode_block_attention_kv8(q=q, k_new=kn, v_new=vn, **{**given, **args, **kw})


def _same(a, b):
    return torch.equal(a.cpu().view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32),
                       b.cpu().view(torch.int16 if b.dtype == torch.bfloat16 else torch.int32))


FORMS = [  # K, L, H, Hkv, page, causal, splits: stream kernel; four waves, small and large pages; eight waves, likewise
    (4, 2, 8, 2, 16, False, 1), (2, 5, 4, 2, 64, True, 2), (4, 16, 4, 2, 32, False, 2), (3, 16, 8, 4, 64, True, 1),
    (8, 16, 8, 4, 32, True, 2), (8, 16, 8, 4, 128, False, 1), (2, 70, 2, 2, 64, True, 2),
]


@pytest.mark.parametrize("form", range(len(FORMS)))
def test_garbage_in_masked_places(form):
    """NaN in slots behind a request, in pages of nobody and in their scales; infinities and NaN in one mode's block keys and
    values: rows that do not see them keep their bits, rows that see a value get it in its own component."""
    K, L, H, Hkv, page, causal, splits = FORMS[form]
    print(f"case: kv8 garbage {FORMS[form]}", flush=True)
    lens = [130, 77, 0]
    d = make_pool(lens, page, Hkv, seed=600 + form)
    g = _gen(650 + form)
    KL = K * L
    q, kn, vn = _bf(g, 3 * KL, H, D), _bf(g, 3 * KL, Hkv, D), _bf(g, 3 * KL, Hkv, D)
    clean = cache_args(d)
    kw = dict(num_ctx_splits=splits, causal_in_block=causal)
    o0, l0 = _attend(d, clean, q.cuda(), kn.cuda(), vn.cuda(), K, L, **kw)

    bad = {k: v.clone() if torch.is_tensor(v) else v for k, v in d.items()}
    used = torch.zeros(d["k_cache"].shape[0], dtype=torch.bool)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        used[d["table"][d["rows"][b]].long()[t // page] * page + t % page] = True
    for x in "kv":
        bad[x + "_cache"].view(torch.uint8)[~used] = 0x7F
        bad[x + "_scale"][~used.view(-1, page).any(1)] = float("nan")
    v2, k2 = vn.clone(), kn.clone()
    first = KL + L  # request 1, mode 1
    v2[first, 0, 3], v2[first + L - 1, 0, 3], v2[first, Hkv - 1, 127] = float("inf"), float("-inf"), float("nan")
    o1, l1 = _attend(d, cache_args(bad), q.cuda(), kn.cuda(), v2.cuda(), K, L, **kw)
    assert _same(l0, l1)
    o0c, o1c = o0.cpu().clone(), o1.cpu().clone()
    rows, G = slice(first, first + L), H // Hkv
    seen = o1c[rows, :G, 3].float()
    last = seen[-1:] if causal else seen  # they see both infinities
    assert bool(last.isnan().all()) and bool((seen[:-1] == float("inf")).all() if causal else True)
    assert bool(o1c[rows, H - G:, 127].isnan().all())
    for o in (o0c, o1c):
        o[rows, :G, 3] = 0
        o[rows, H - G:, 127] = 0
    assert _same(o0c, o1c)

    k2[first, :, 9] = float("nan")  # a key of mode 1: its rows are lost, no other
    o2, l2 = _attend(d, cache_args(bad), q.cuda(), k2.cuda(), vn.cuda(), K, L, **kw)
    assert bool(o2[rows].isnan().all()) and bool(l2[rows].isnan().all())
    keep = torch.ones(3 * KL, dtype=torch.bool)
    keep[rows] = False
    assert _same(o0.cpu()[keep], o2.cpu()[keep]) and _same(l0.cpu()[keep], l2.cpu()[keep])


def test_a_nan_code_reaches_the_rows_that_see_it():
    d = make_pool([100, 90], 64, 2, seed=700)
    g = _gen(701)
    q, kn, vn = _bf(g, 2 * 64, 4, D), _bf(g, 2 * 64, 2, D), _bf(g, 2 * 64, 2, D)
    clean = cache_args(d)
    o0, _ = _attend(d, clean, q.cuda(), kn.cuda(), vn.cuda(), 4, 16)
    slot = int(d["table"][d["rows"][0]][0]) * 64 + 40
    d["v_cache"].view(torch.uint8)[slot, 1, 17] = 0x7F
    o1, l1 = _attend(d, cache_args(d), q.cuda(), kn.cuda(), vn.cuda(), 4, 16)
    assert bool(o1[:64, 2:, 17].isnan().all()) and bool(l1.isfinite().all())
    o0[:64, 2:, 17] = o1[:64, 2:, 17] = 0
    assert _same(o0, o1)


@pytest.mark.parametrize("form", range(len(FORMS)))
def test_value_scales_at_both_ends(form):
    """Neighbouring pages whose values are a factor of 2^80 apart, the scales' whole range, in both orders and alone: the
    accumulators change their unit with each.

    Here probabilities far below the row's largest decide the result, and fp16 has fewer bits for those. A probability p enters
    as fp16(p 2^q), q >= -2 the quotient of the page's scale and the unit, p relative to a maximum that the row has met, so that
    the row's sum is at least 1. Below 2^-14 half a step is 2^-25: p / sum is off by 2^-25 2^-q <= 2^-23 at most, beside its
    2^-11. Over the cached keys that is 2^-23 sum |v| on top of the bound elsewhere. A split's partial row is rounded to fp16
    after a power of two has brought its largest component m into [1/2, 1): components below 2^-14 are off by 2^-25 there, 2^-24 m
    in the row at most. (With one page deciding, single codes of very different size make up a row.)"""
    K, L, H, Hkv, page, causal, splits = FORMS[form]
    for ends in ((-40, 40), (40, -40), (-40, -40), (40, 40), (0, -40)):
        lens = [5 * page + 3, page + 1]
        d = make_pool(lens, page, Hkv, seed=780 + form)
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                d["v_scale"][int(d["table"][d["rows"][b]][i])] = 2.0 ** ends[i % 2]
        g = _gen(790)
        T = 2 * K * L
        q, kn, vn = _bf(g, T, H, D), _bf(g, T, Hkv, D), _bf(g, T, Hkv, D)
        o, l = _attend(d, cache_args(d), q.cuda(), kn.cuda(), vn.cuda(), K, L, num_ctx_splits=splits, causal_in_block=causal)
        ref = oracle_attention(d, q, kn, vn, lens, K, L, SCALE, causal)
        for b, n in enumerate(lens):
            v = kv8.tokens(vals(d["v_cache"]), vals(d["v_scale"]), d["table"][d["rows"][b]].numpy(), n, page)
            mass = ref[2][b * K * L:(b + 1) * K * L]
            more = np.abs(v).sum(0).repeat(H // Hkv, 0) * 2.0 ** -23 + mass.max(-1, keepdims=True) * 2.0 ** -24
            mass += more / (2 * 2.0 ** -11 + 2.0 ** -12)
        check_attention(o, l, ref)


def test_weights_of_rows_taken_out():
    """Rows whose lse is -inf add nothing, whatever their q holds."""
    import kv8_cache

    for K, L, H in ((1, 3, 4), (4, 16, 4), (8, 16, 8)):
        d = make_pool([300, 70], 32, 2, seed=710 + H)
        g = _gen(711)
        T = 2 * K * L
        q = _bf(g, T, H, D)
        _, lse, _, _ = oracle_attention(d, q, None, None, [300, 70], K, L, SCALE, False)
        lse = torch.from_numpy(lse).float()
        lse[K * L - 1], lse[0] = float("-inf"), float("-inf")
        res = []
        for fill in (0.0, float("nan"), float("inf")):
            q[K * L - 1], q[0] = fill, fill
            args = cache_args(d)
            del args["v_cache"], args["v_scale"]
            w = torch.zeros(3, 2, 300).cuda()
            kv8_cache.attention_weights_kv8(q=q.cuda(), lse=lse.cuda(), page_table=d["table"].cuda(), ctx_lens=d["lens"].cuda(),
                                            num_modes=K, block_size=L, scaling=SCALE, weights=w, **args)
            res.append(w)
        assert bool(res[0].isfinite().all()) and _same(res[0], res[1]) and _same(res[0], res[2])


def _guarded(t, dev="cuda"):
    """t in the middle of a larger buffer; the buffer."""
    flat = t.contiguous().view(torch.uint8).reshape(-1)
    buf = torch.full((flat.numel() + 8192,), 0x5A, dtype=torch.uint8, device=dev)
    buf[4096:-4096] = flat.to(dev)
    return buf[4096:-4096].view(t.dtype).view(t.shape), buf


def test_ids_and_lengths_out_of_range_are_reported():
    """Page ids, table rows and lengths that nobody checked: the call says so in its error flag, writes nothing outside its
    tensors, and the other requests' results keep their bits."""
    import kv8_cache
    import mfd_hip

    page, Hkv, H = 64, 2, 4
    lens = [300, 200, 150]
    for form, (KK, LL) in enumerate(((4, 16), (1, 2))):
        d = make_pool(lens, page, Hkv, seed=720, extra=2)
        g = _gen(721)
        T = 3 * KK * LL
        q, kn, vn = _bf(g, T, H, D), _bf(g, T, Hkv, D), _bf(g, T, Hkv, D)
        o0, l0 = _attend(d, cache_args(d), q.cuda(), kn.cuda(), vn.cuda(), KK, LL, num_ctx_splits=2)
        args = cache_args(d)
        bad = dict(page_in_table=[-1, 2 ** 30], row=[-1, 4, 2 ** 40], length=[-1, 10 ** 6, 2 ** 62, -2 ** 62])
        for what, values in bad.items():
            for value in values:
                print(f"case: kv8 ids out of range {form} {what} {value}", flush=True)
                e = {k: v.clone() if torch.is_tensor(v) else v for k, v in d.items()}
                if what == "page_in_table":
                    e["table"][e["rows"][1], 1] = value
                elif what == "row":
                    e["rows"][1] = value
                else:
                    e["lens"][1] = value
                guards, a = {}, {}
                for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
                    a[name], guards[name] = _guarded(d[name])
                a.update(page_size=page, req_pool_indices=e["rows"].cuda())
                before = {name: buf.clone() for name, buf in guards.items()}
                flags = torch.zeros(5, dtype=torch.int32, device="cuda")
                o1, l1 = _attend(e, a, q.cuda(), kn.cuda(), vn.cuda(), KK, LL, num_ctx_splits=2, err_flag=flags[0:1])
                w, wbuf = _guarded(torch.ones(4, Hkv, 300))
                wargs = {k: v for k, v in a.items() if k not in ("v_cache", "v_scale")}
                kv8_cache.attention_weights_kv8(q=q.cuda(), lse=l0, page_table=e["table"].cuda(), ctx_lens=e["lens"].cuda(),
                                                num_modes=KK, block_size=LL, scaling=SCALE, weights=w, err_flag=flags[1:2],
                                                **wargs)
                assert all(torch.equal(guards[n], before[n]) for n in guards)  # so far everything only read
                keep, new = kv8_cache.evict_select(weights=w, req_pool_indices=a["req_pool_indices"],
                                                   ctx_lens=e["lens"].cuda(), budget=100, sink=2, recent=8, err_flag=flags[2:3])
                kv8_cache.evict_compact_kv8(keep=keep, new_lens=new, ctx_lens=e["lens"].cuda(), src_table=e["table"].cuda(),
                                            dst_table=e["dst"].cuda(), weights=w, err_flag=flags[3:4], **a)
                kv8_cache.kv8_store(k=kn.cuda()[:3], v=vn.cuda()[:3], page_table=e["table"].cuda(),
                                    start_lens=torch.tensor([5, 70 if what != "length" else value, 5]).cuda(),
                                    cu_tokens=torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda(), max_tokens=1,
                                    err_flag=flags[4:5], **a)
                torch.cuda.synchronize()
                f = flags.tolist()
                assert f[0] == f[1] == mfd_hip.DEVERR_BAD_PAGE and f[4] == f[0], (what, value, f)
                assert (f[2] != 0) == (what != "page_in_table") and (f[3] != 0 or what != "page_in_table"), f
                for buf in [*guards.values(), wbuf]:
                    assert bool((buf[:4096] == 0x5A).all()) and bool((buf[-4096:] == 0x5A).all())
                n = KK * LL
                for r in (slice(0, n), slice(2 * n, 3 * n)):
                    assert _same(o0[r].contiguous(), o1[r].contiguous()) and _same(l0[r].contiguous(), l1[r].contiguous())


def test_strides_index_types_and_a_buffer_for_the_result():
    """q, k and v as slices of one fused projection, K and V interleaved in one cache with a slot of their own, int32 indices that
    are longer than the batch, the result into a strided buffer: the same bits as contiguous ones."""
    import kv8_cache

    lens, K, L, H, Hkv, page = [300, 65], 4, 16, 8, 2, 64
    d = make_pool(lens, page, Hkv, seed=730, extra=2)
    g = _gen(731)
    T = 2 * K * L
    fused = _bf(g, T, (H + 2 * Hkv) * D + 64).cuda()
    q = fused[:, :H * D].view(T, H, D)
    kn, vn = (fused[:, (H + i * Hkv) * D:(H + (i + 1) * Hkv) * D].view(T, Hkv, D) for i in range(2))
    o0, l0 = _attend(d, cache_args(d), q.contiguous(), kn.contiguous(), vn.contiguous(), K, L)
    slots = d["k_cache"].shape[0]
    both = torch.zeros(slots, Hkv, 2, 160, dtype=torch.uint8, device="cuda").view(F8)
    kc, vc = both[:, :, 0, :D], both[:, :, 1, 16:16 + D]
    kc.copy_(d["k_cache"].cuda())
    vc.copy_(d["v_cache"].cuda())
    args = dict(cache_args(d), k_cache=kc, v_cache=vc, req_pool_indices=torch.cat([d["rows"], torch.tensor([9])]).int().cuda())
    out = torch.full((T, H + 1, 144), 3.0, dtype=torch.bfloat16, device="cuda")
    d32 = dict(d, lens=torch.cat([d["lens"], torch.tensor([7])]).int())
    table = torch.full((3, d["table"].shape[1] + 5), 2 ** 30, dtype=torch.int32)
    table[:, 2:-3] = d["table"]
    o1, l1 = _attend(d32, args, q, kn, vn, K, L, out=out[:, 1:, 8:136], page_table=table.cuda()[:, 2:-3],
                     max_ctx=d["table"].shape[1] * page)
    assert _same(o0, o1.contiguous()) and _same(l0, l1)
    assert bool((out[:, 0] == 3).all()) and bool((out[:, :, :8] == 3).all()) and bool((out[:, :, 136:] == 3).all())
    w0, w1 = torch.zeros(3, Hkv, 304).cuda(), torch.zeros(3, Hkv, 304).cuda()
    for w, qq, a in ((w0, q.contiguous(), cache_args(d)), (w1, q, args)):
        a = {k: v for k, v in a.items() if k not in ("v_cache", "v_scale")}
        kv8_cache.attention_weights_kv8(q=qq, lse=l0, page_table=d["table"].cuda(), ctx_lens=d["lens"].cuda(), num_modes=K,
                                        block_size=L, scaling=SCALE, weights=w,
                                        **{**a, "req_pool_indices": d["rows"].int().cuda()})
    assert _same(w0, w1)
    plain = cache_args(d)
    for a in (plain, args):
        kv8_cache.kv8_store(k=kn[:40], v=vn[:40], page_table=d["table"].cuda(), start_lens=torch.tensor([290, 0]).int().cuda(),
                            cu_tokens=torch.tensor([0, 10, 40], dtype=torch.int32).cuda(), max_tokens=40, **a)
        keep = torch.arange(100, dtype=torch.int32).repeat(2, 1).cuda() * 2
        kv8_cache.evict_compact_kv8(keep=keep, new_lens=torch.tensor([100, 30]).int().cuda(), ctx_lens=d["lens"].int().cuda(),
                                    src_table=d["table"].cuda(), dst_table=d["dst"].cuda(), **a)
    for x in "kv":
        assert torch.equal(plain[x + "_cache"].view(torch.uint8), args[x + "_cache"].contiguous().view(torch.uint8))
        assert torch.equal(plain[x + "_scale"], args[x + "_scale"])
    assert bool((both[:, :, 0, D:].view(torch.uint8) == 0).all())


def test_nothing_to_do():
    import kv8_cache
    import mxfp4_head

    d = make_pool([5], 16, 2, seed=740, extra=1)
    args = cache_args(d)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    args["req_pool_indices"] = none
    e = dict(d, lens=none)
    empty = torch.empty(0, 2, D, dtype=torch.bfloat16, device="cuda")
    o, l = _attend(e, args, torch.empty(0, 4, D, dtype=torch.bfloat16, device="cuda"), empty, empty, 2, 4)
    assert tuple(o.shape) == (0, 4, D) and tuple(l.shape) == (0, 4)
    kv8_cache.kv8_store(k=empty, v=empty, page_table=d["table"].cuda(), start_lens=none,
                        cu_tokens=torch.zeros(1, dtype=torch.int32, device="cuda"), max_tokens=0, **args)
    keep, new = kv8_cache.evict_select(weights=torch.zeros(2, 2, 8, device="cuda"), req_pool_indices=none, ctx_lens=none, budget=4,
                                       sink=1, recent=1)
    assert tuple(keep.shape) == (0, 4) and tuple(new.shape) == (0,)
    kv8_cache.evict_compact_kv8(keep=keep, new_lens=new, ctx_lens=none, src_table=d["table"].cuda(),
                                dst_table=d["dst"].cuda(), **args)
    x = torch.empty(0, 128, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(7, 64, dtype=torch.uint8, device="cuda"), torch.full((7, 4), 127, dtype=torch.uint8, device="cuda")
    assert tuple(mxfp4_head.draft_head_mxfp4(x, *w).shape) == (0, 7)
    torch.cuda.synchronize()


def test_results_repeat():
    import kv8_cache

    for case in (5, 8, 12):
        lens, K, L, H, Hkv, page, fresh, causal, splits = ATTN[case]
        d = make_pool(lens, page, Hkv, seed=750 + case)
        g = _gen(751)
        T = len(lens) * K * L
        q = _bf(g, T, H, D).cuda()
        kn, vn = (_bf(g, T, Hkv, D).cuda(), _bf(g, T, Hkv, D).cuda()) if fresh else (None, None)
        args = cache_args(d)
        wargs = {k: v for k, v in args.items() if k not in ("v_cache", "v_scale")}
        first = None
        for _ in range(4):
            o, l = _attend(d, args, q, kn, vn, K, L, num_ctx_splits=3)
            w = torch.zeros(len(lens) + 1, Hkv, max(lens)).cuda()
            kv8_cache.attention_weights_kv8(q=q, lse=l, page_table=d["table"].cuda(), ctx_lens=d["lens"].cuda(), num_modes=K,
                                            block_size=L, scaling=SCALE, weights=w, **wargs)
            first = first or (o, l, w)
            assert _same(first[0], o) and _same(first[1], l) and _same(first[2], w)


class _Step:
    """One draft round on static buffers, every workspace handed in: attention, token weights, new tokens, selection,
    compaction, and the 4-bit head on the attention's rows."""

    def __init__(self, seed):
        import kv8_cache

        self.K, self.L, self.H, self.Hkv, self.page = 4, 16, 8, 2, 64
        self.lens = [300, 129]
        d = make_pool(self.lens, self.page, self.Hkv, seed=seed, extra=2)
        g = _gen(seed + 1)
        T = 2 * self.K * self.L
        self.d = d
        self.start = cache_args(d)
        self.args = {k: v.clone() if torch.is_tensor(v) else v for k, v in self.start.items()}
        self.table, self.dst, self.ctx = d["table"].cuda(), d["dst"].cuda(), d["lens"].cuda()
        self.q, self.kn, self.vn = _bf(g, T, self.H, D).cuda(), _bf(g, T, self.Hkv, D).cuda(), _bf(g, T, self.Hkv, D).cuda()
        self.out, self.lse = torch.zeros_like(self.q), torch.zeros(T, self.H, device="cuda")
        self.w = torch.zeros(3, self.Hkv, 20000, device="cuda")  # wide: selection through its workspace
        self.cu = torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda")
        self.keep = torch.zeros(2, 100, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(2, dtype=torch.int64, device="cuda")
        self.flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        size = kv8_cache.workspace_bytes(bs=2, num_modes=self.K, block_size=self.L, num_heads=self.H, num_kv_heads=self.Hkv,
                                         with_block=True, max_ctx=300, num_ctx_splits=3)
        self.ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        self.ws2 = torch.zeros(2 * 20000 * 4, dtype=torch.uint8, device="cuda")
        self.codes = torch.randint(0, 256, (20001, self.H * D // 2), generator=g, dtype=torch.uint8).cuda()
        self.exps = torch.randint(118, 124, (20001, self.H * D // 32), generator=g, dtype=torch.uint8).cuda()
        self.logits = torch.zeros(T, 20008, dtype=torch.bfloat16, device="cuda")[:, :20001]

    def refill(self, seed):
        g = _gen(seed)
        for t in (self.q, self.kn, self.vn):
            t.copy_(_bf(g, *t.shape))
        for k, v in self.start.items():
            if torch.is_tensor(v):
                self.args[k].view(torch.uint8).copy_(v.view(torch.uint8))
        self.w.zero_()

    def run(self):
        import kv8_cache
        import mxfp4_head

        common = dict(num_modes=self.K, block_size=self.L, scaling=SCALE, page_table=self.table, ctx_lens=self.ctx,
                      err_flag=self.flag)
        wargs = {k: v for k, v in self.args.items() if k not in ("v_cache", "v_scale")}
        kv8_cache.paged_mode_block_attention_kv8(q=self.q, k_new=self.kn, v_new=self.vn, out=self.out, lse_out=self.lse,
                                                 num_ctx_splits=3, max_ctx=300, workspace=self.ws, **self.args, **common)
        kv8_cache.attention_weights_kv8(q=self.q, lse=self.lse, weights=self.w, decay=0.9, **wargs, **common)
        kv8_cache.kv8_store(k=self.kn[:9], v=self.vn[:9], page_table=self.table, start_lens=self.ctx - 5, cu_tokens=self.cu,
                            max_tokens=5, err_flag=self.flag, **self.args)
        kv8_cache.evict_select(weights=self.w, req_pool_indices=self.args["req_pool_indices"], ctx_lens=self.ctx, budget=100,
                               keep_out=self.keep, new_lens_out=self.new, workspace=self.ws2, err_flag=self.flag)
        kv8_cache.evict_compact_kv8(keep=self.keep, new_lens=self.new, ctx_lens=self.ctx, src_table=self.table,
                                    dst_table=self.dst, weights=self.w, err_flag=self.flag, **self.args)
        mxfp4_head.draft_head_mxfp4(self.out.view(-1, self.H * D), self.codes, self.exps, out=self.logits)

    def state(self):
        torch.cuda.synchronize()
        assert int(self.flag) == 0
        return [t.clone().contiguous().view(torch.uint8) for t in (
            self.out, self.lse, self.w, self.keep, self.new, self.logits, self.args["k_cache"], self.args["v_cache"],
            self.args["k_scale"], self.args["v_scale"])]


def test_a_captured_round_replays():
    """Two rounds captured in graphs that share their workspaces, replayed in turn with other inputs, eager work and
    synchronizations between: each replay leaves what the eager round leaves."""
    a, b = _Step(760), _Step(770)
    b.ws, b.ws2 = a.ws, a.ws2
    graphs = []
    for s in (a, b):
        s.run()  # first use of every kernel
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run()
        graphs.append(graph)
    for turn in range(4):
        for s, graph in zip((a, b), graphs):
            s.refill(780 + turn)
            s.run()
            eager = s.state()
            s.refill(780 + turn)
            torch.cuda.synchronize()
            for t in (s.out, s.lse, s.keep, s.new, s.logits):
                t.zero_()
            graph.replay()
            assert all(torch.equal(x, y) for x, y in zip(eager, s.state()))


def test_a_captured_attention_follows_the_lengths():
    """Captured with one batch's lengths and replayed with others, none among them: splits are measured out on the device."""
    import kv8_cache

    for K, L, H in ((4, 16, 8), (1, 2, 32)):
        bs, page, Hkv = 9, 64, 8
        most = [900 + 300 * b for b in range(bs)]
        d = make_pool(most, page, Hkv, seed=795)
        g = _gen(796)
        T = bs * K * L
        q, kn, vn = _bf(g, T, H, D).cuda(), _bf(g, T, Hkv, D).cuda(), _bf(g, T, Hkv, D).cuda()
        args, table, lens = cache_args(d), d["table"].cuda(), d["lens"].cuda()
        out, lse = torch.zeros_like(q), torch.zeros(T, H, device="cuda")
        size = kv8_cache.workspace_bytes(bs=bs, num_modes=K, block_size=L, num_heads=H, num_kv_heads=Hkv, with_block=True,
                                         max_ctx=max(most))
        assert size > 0
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        run = lambda **kw: kv8_cache.paged_mode_block_attention_kv8(  # noqa: E731
            q=q, k_new=kn, v_new=vn, page_table=table, ctx_lens=lens, num_modes=K, block_size=L, scaling=SCALE,
            max_ctx=max(most), return_lse=True, **kw, **args)
        run(out=out, lse_out=lse, workspace=ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(out=out, lse_out=lse, workspace=ws)
        for turn in range(4):
            now = [0] * bs if turn == 2 else [(n * (turn + 3) * (b + 2)) % (n + 1) for b, n in enumerate(most)]
            lens.copy_(torch.tensor(now))
            o, l = run()
            torch.cuda.synchronize()
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert _same(o, out) and _same(l, lse)
            check_attention(out, lse, oracle_attention(d, q.cpu(), kn.cpu(), vn.cpu(), now, K, L, SCALE, False))


def test_on_another_stream():
    s = _Step(790)
    s.refill(791)
    s.run()
    eager = s.state()
    s.refill(791)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1000000)  # whatever ran on the default stream instead would be ahead of the inputs below
        s.q.mul_(1)
        s.run()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, s.state()))


def test_a_cache_beyond_4_gib():
    """Pages whose bytes lie more than 2^32 behind the cache's first, as the bits of the same pages in a small cache."""
    import kv8_cache

    page, Hkv, H = 64, 8, 32
    lens = [200, 129]
    for K, L in ((1, 4), (8, 16)):
        d = make_pool(lens, page, Hkv, seed=800, extra=2)
        pages = d["k_scale"].shape[0]
        total = 70001  # 4.59 GB of K, and of V
        far = torch.arange(pages) * 3 + (total - 3 * pages)
        far[0] = 1
        big = dict(page_size=page, req_pool_indices=d["rows"].cuda())
        for x in "kv":
            cache = torch.empty(total * page, Hkv, D, dtype=torch.uint8, device="cuda")
            scale = torch.full((total, Hkv), 1.0, device="cuda")
            cache.view(total, page, Hkv, D)[far.cuda()] = d[x + "_cache"].view(torch.uint8).view(pages, page, Hkv, D).cuda()
            scale[far.cuda()] = d[x + "_scale"].cuda()
            big[x + "_cache"], big[x + "_scale"] = cache.view(F8), scale
        move = lambda t: torch.where(t < pages, far[t.clamp(max=pages - 1).long()].int(), t)  # noqa: E731
        e = dict(d, table=move(d["table"]), dst=move(d["dst"]))
        g = _gen(801)
        T = 2 * K * L
        q, kn, vn = _bf(g, T, H, D).cuda(), _bf(g, T, Hkv, D).cuda(), _bf(g, T, Hkv, D).cuda()
        res = []
        for dd, a in ((d, cache_args(d)), (e, big)):
            tables = dict(page_table=dd["table"].cuda())
            kv8_cache.kv8_store(k=kn[:8], v=vn[:8], start_lens=torch.tensor([190, 60]).cuda(), max_tokens=6,
                                cu_tokens=torch.tensor([0, 2, 8], dtype=torch.int32).cuda(), **tables, **a)
            o, l = _attend(dd, a, q, kn, vn, K, L)
            w = torch.zeros(3, Hkv, 200, device="cuda")
            wargs = {k: v for k, v in a.items() if k not in ("v_cache", "v_scale")}
            kv8_cache.attention_weights_kv8(q=q, lse=l, ctx_lens=d["lens"].cuda(), num_modes=K, block_size=L, scaling=SCALE,
                                            weights=w, **tables, **wargs)
            keep, new = kv8_cache.evict_select(weights=w, req_pool_indices=a["req_pool_indices"], ctx_lens=d["lens"].cuda(),
                                               budget=100)
            kv8_cache.evict_compact_kv8(keep=keep, new_lens=new, ctx_lens=d["lens"].cuda(), src_table=dd["table"].cuda(),
                                        dst_table=dd["dst"].cuda(), **a)
            ids = torch.arange(pages) if dd is d else far
            res.append([o.view(torch.int16), l, w, keep, new] + [
                t for x in "kv" for t in (a[x + "_cache"].view(torch.uint8).view(-1, page, Hkv, D)[ids.cuda()],
                                          a[x + "_scale"][ids.cuda()])])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(*res))
        del big, res


def test_a_draft_run_of_all_operators():
    """Prompts stored, drafted against with token weights collected over two layers, accepted tokens stored, the requests cut to
    a budget, and drafted against again, through the pool and PagedModeAttention: each step against the oracle's."""
    import kv8_cache
    import paged_mode_attention

    page, Hkv, H, K, L, layers, budget = 32, 2, 8, 4, 8, 2, 64
    bs, prompt, accepted = 2, [150, 70], [3, 1]
    KL = K * L
    g = _gen(810)
    pool = kv8_cache.Kv8Pool(num_layers=layers, num_pages=24, page_size=page, num_kv_heads=Hkv)
    perm = torch.randperm(24, generator=g).int()
    table, dst = torch.zeros(3, 6, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32)
    table[2, :5], table[1, :3] = perm[:5], perm[5:8]
    dst[2, :3], dst[1, :3] = perm[8:11], perm[11:14]  # (one page to grow)
    rows = torch.tensor([2, 1])
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    common = dict(req_pool_indices=rows.cuda(), err_flag=flag)
    mine = []  # the oracle's caches
    for layer in range(layers):
        mine.append({x: (vals(c), vals(s)) for x, c, s in zip("kv", pool.get_kv_buffer(layer), pool.get_kv_scale(layer))})

    def store(start, new, tab):
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        for layer in range(layers):
            x = {w: _bf(g, int(cu[-1]), Hkv, D) * 3 for w in "kv"}
            pool.store(layer, k=x["k"].cuda(), v=x["v"].cuda(), page_table=tab.cuda(), start_lens=torch.tensor(start).cuda(),
                       cu_tokens=cu.cuda(), max_tokens=max(new), **common)
            for w in "kv":
                kv8.store(vals(x[w]), *mine[layer][w], tab.numpy(), rows.numpy(), start, cu.numpy(), page)

    def same_caches():
        torch.cuda.synchronize()
        for layer in range(layers):
            for x, c, s in zip("kv", pool.get_kv_buffer(layer), pool.get_kv_scale(layer)):
                assert np.array_equal(vals(c), mine[layer][x][0]) and np.array_equal(vals(s), mine[layer][x][1])

    def draft(lens, tab, weights):
        batch = type("Batch", (), dict(req_pool_indices=rows.cuda(), seq_lens=torch.tensor(lens).cuda(),
                                       seq_lens_cpu=torch.tensor(lens)))()
        hook = paged_mode_attention.PagedModeAttention(
            kv_pool=pool, req_to_token=tab.cuda(), num_modes=K, block_size=L, num_heads=H, num_kv_heads=Hkv, head_dim=D,
            scaling=SCALE, num_ctx_splits=-1, impl="hip", page_size=page)
        for layer in range(layers):
            q, kn, vn = _bf(g, bs * KL, H, D), _bf(g, bs * KL, Hkv, D), _bf(g, bs * KL, Hkv, D)
            d = dict(table=tab, rows=rows, page=page)
            for i, x in enumerate("kv"):
                d[x + "_cache"], d[x + "_scale"] = (torch.from_numpy(t) for t in mine[layer][x])
            ref = oracle_attention(d, q, kn, vn, lens, K, L, SCALE, False)
            out, lse = pool.attention(layer, q=q.cuda(), k_new=kn.cuda(), v_new=vn.cuda(), page_table=tab.cuda(),
                                      ctx_lens=batch.seq_lens, num_modes=K, block_size=L, scaling=SCALE, return_lse=True,
                                      **common)
            check_attention(out, lse, ref)
            got = hook(*(t.cuda().view(bs * KL, -1) for t in (q, kn, vn)), batch, layer)
            check_attention(got.view(-1, H, D), lse, ref)
            if weights is not None:
                pool.add_weights(layer, q=q.cuda(), lse=lse, page_table=tab.cuda(), ctx_lens=batch.seq_lens, num_modes=K,
                                 block_size=L, scaling=SCALE, weights=weights, decay=0.5 if layer == 0 else 1.0, **common)
                for b, n in enumerate(lens):
                    r = slice(b * KL, (b + 1) * KL)
                    k = kv8.tokens(*mine[layer]["k"], tab[rows[b]].numpy(), n, page)
                    expected[b] = expected[b] * (0.5 if layer == 0 else 1.0) + kv8.weights(vals(q[r]), ref[1][r], k, SCALE)

    weights = torch.zeros(3, Hkv, 200, device="cuda")
    expected = [np.zeros((Hkv, n)) for n in prompt]
    store([0, 0], prompt, table)
    same_caches()
    draft(prompt, table, weights)
    for b, n in enumerate(prompt):
        got = vals(weights)[int(rows[b]), :, :n]
        # a probability's relative error: its score's and its lse's (sizes below 64, |lse| below 32) and its own roundings
        assert (np.abs(got - expected[b]) <= 2.0 ** -24 * (256 * 64 + 16 * 32 + 64) * expected[b] + 1e-35).all()
    store(prompt, accepted, table)
    same_caches()
    lens = [n + a for n, a in zip(prompt, accepted)]
    before = weights.cpu().numpy().copy()
    keep, new = pool.evict(weights=weights, page_table=table.cuda(), dst_table=dst.cuda(), ctx_lens=torch.tensor(lens).cuda(),
                           budget=budget, sink=4, recent=8, **common)
    for b, n in enumerate(lens):
        row = int(rows[b])
        kept = kv8.select(before[row], n, budget, 4, 8)
        assert keep[b].tolist() == kept + [-1] * (budget - len(kept)) and int(new[b]) == len(kept)
        for layer in range(layers):
            for x in "kv":
                kv8.compact(*mine[layer][x], table[row].numpy(), dst[row].numpy(), kept, page)
        assert np.array_equal(weights.cpu().numpy()[row, :, :len(kept)], before[row][:, kept])
    same_caches()
    draft(new.tolist(), dst, None)
    store(new.tolist(), accepted, dst)
    same_caches()
    draft([int(n) + a for n, a in zip(new.tolist(), accepted)], dst, None)
    assert int(flag) == 0


@pytest.mark.parametrize("vocab_ids", [False, True])
def test_draft_topk_with_a_4_bit_head(vocab_ids):
    """DDTreeDraftTopK over an Mxfp4Weight: the rows' logits as draft_head_mxfp4 forms them, and the top-k of those."""
    import ddtree_sglang_ops
    import mxfp4_head

    hidden, vocab, L, K, bs, budget = 256, 20001, 8, 3, 2, 17
    g = _gen(820)
    w = mxfp4_head.quantize((torch.randn(vocab, hidden, generator=g) * 0.05).cuda())
    ids = torch.randperm(2 * vocab, generator=g)[:vocab].int().cuda() if vocab_ids else None
    head = ddtree_sglang_ops.DDTreeDraftTopK(weight=w, block_size=L, num_modes=K, budget=budget, max_bs=4, vocab_ids=ids)
    x = _bf(g, bs * K * L, hidden).cuda()
    head(x)
    torch.cuda.synchronize()
    n = bs * K * (L - 1)
    rows = x.view(-1, L, hidden)[:, 1:].reshape(n, hidden)
    logits = mxfp4_head.draft_head_mxfp4(rows, w.codes, w.exps)
    assert torch.equal(head.logits[:n].view(torch.int16), logits.view(torch.int16))
    ref = rows.cpu().double() @ mxfp4_head.dequantize(w).cpu().double().t()
    mass = rows.cpu().double().abs() @ mxfp4_head.dequantize(w).cpu().double().abs().t()
    bound = (2.0 ** -8 * ref.abs() + hidden * 2.0 ** -24 * mass) * (1 + 2.0 ** -8)
    assert bool(((logits.cpu().double() - ref).abs() <= bound).all())
    logp, top = head.outputs(bs)
    f = logits.cpu().float()
    want, at = f.sort(dim=1, descending=True, stable=True)  # ties: the lowest column
    want, at = want[:, :budget], at[:, :budget]
    log_z = torch.logsumexp(f.double(), dim=1, keepdim=True)
    got = logp.reshape(n, budget).cpu().double() + head.log_z[:n].cpu().double()[:, None]
    assert bool(((got - want.double()).abs() <= 2.0 ** -22 * (want.abs() + log_z.abs())).all())
    assert bool(((head.log_z[:n].cpu().double()[:, None] - log_z).abs() <= 1e-5 * log_z.abs() + 1e-5).all())
    columns = top.reshape(n, budget).cpu()
    assert torch.equal(columns, (at.int() if ids is None else ids.cpu()[at]))
