"""What the 8-bit draft cache and the 4-bit head do without a GPU: the oracle's number formats against torch's, the refusals of
the C entry points and of the Python ones (no kernel is launched), quantisation of the head, the float32 checking path of
PagedModeAttention over an 8-bit pool, and the choice of context splits."""

import numpy as np
import pytest
import torch

import kv8_cache
import mfd_hip
import mxfp4_head
import paged_mode_attention
from oracle import kv8

F8 = torch.float8_e4m3fn


def test_oracle_rounding_is_the_types():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-13, 10, (20000,), generator=g).float())
    x = torch.cat([x, torch.arange(-460, 460).float() / 1024, torch.arange(0, 4000).float() / 8])
    ref = x.clamp(-448, 448).to(F8).float().double().numpy()
    assert np.array_equal(kv8.e4m3(x.double().numpy()), ref)
    codes = torch.arange(256, dtype=torch.uint8).view(F8).float().double().numpy()
    assert np.array_equal(kv8.e4m3(codes), codes, equal_nan=True)


@pytest.mark.parametrize("amax", [0.0, 1e-30, 448 * 2.0 ** -40, 447.9, 448.0, 448.1, 3e-3, 1.0, 0.875, 0.8751, 1e20])
def test_page_scale_is_the_smallest_that_holds(amax):
    s = kv8.page_scale(amax)
    assert np.log2(s) == int(np.log2(s)) and 2.0 ** -40 <= s <= 2.0 ** 40
    assert amax <= 448 * s or s == 2.0 ** 40
    assert s == 2.0 ** -40 or amax > 448 * s / 2


# ------------------------------------------------------------------------------------------- refusals, C entry points

P = 1 << 20  # stands for a 16-byte aligned device pointer; no call below gets as far as using it


def _store(**kw):
    d = dict(k=P, v=P, kn=(1024, 128), vn=(1024, 128), kc=P, vc=P, kcs=(1024, 128), vcs=(1024, 128), ks=P, vs=P, pages=10,
             table=P, ts=8, rows=4, width=8, page=64, idx=P, starts=P, cu=P, N=5, bs=2, most=4, heads=8, D=128)
    d.update(kw)
    return mfd_hip.lib().mfd_kv8_store(d["k"], d["v"], *d["kn"], *d["vn"], d["kc"], d["vc"], *d["kcs"], *d["vcs"], d["ks"],
                                       d["vs"], d["pages"], d["table"], d["ts"], d["rows"], d["width"], d["page"], d["idx"],
                                       d["starts"], d["cu"], d["N"], d["bs"], d["most"], d["heads"], d["D"], None, None)


def _attn(**kw):
    d = dict(q=P, qs=(4096, 128), kn=P, vn=P, kns=(1024, 128), vns=(1024, 128), kc=P, vc=P, kcs=(1024, 128), vcs=(1024, 128),
             ks=P, vs=P, pages=10, table=P, ts=8, rows=4, width=8, page=64, idx=P, lens=P, bs=2, K=2, L=4, H=32, heads=8,
             D=128, scale=0.1, causal=0, splits=1, keys=0, out=P, os=(4096, 128), lse=P, ws=None, nws=0)
    d.update(kw)
    return mfd_hip.lib().mfd_kv8_attn(d["q"], *d["qs"], d["kn"], d["vn"], *d["kns"], *d["vns"], d["kc"], d["vc"], *d["kcs"],
                                      *d["vcs"], d["ks"], d["vs"], d["pages"], d["table"], d["ts"], d["rows"], d["width"],
                                      d["page"], d["idx"], d["lens"], d["bs"], d["K"], d["L"], d["H"], d["heads"], d["D"],
                                      d["scale"], d["causal"], d["splits"], d["keys"], d["out"], *d["os"], d["lse"], d["ws"],
                                      d["nws"], None, None)


def _weigh(**kw):
    d = dict(q=P, qs=(4096, 128), lse=P, kc=P, kcs=(1024, 128), ks=P, pages=10, table=P, ts=8, rows=4, width=8, page=64, idx=P,
             lens=P, bs=2, K=2, L=4, H=32, heads=8, D=128, scale=0.1, decay=1.0, w=P, ws=(800, 100), wrows=4, wwidth=100)
    d.update(kw)
    return mfd_hip.lib().mfd_kv8_weights(d["q"], *d["qs"], d["lse"], d["kc"], *d["kcs"], d["ks"], d["pages"], d["table"],
                                         d["ts"], d["rows"], d["width"], d["page"], d["idx"], d["lens"], d["bs"], d["K"],
                                         d["L"], d["H"], d["heads"], d["D"], d["scale"], d["decay"], d["w"], *d["ws"],
                                         d["wrows"], d["wwidth"], None, None)


def _select(**kw):
    d = dict(w=P, ws=(800, 100), wrows=4, width=100, heads=8, idx=P, lens=P, bs=2, budget=40, sink=4, recent=32, keep=P, new=P,
             wsp=P, nws=1 << 20)
    d.update(kw)
    return mfd_hip.lib().mfd_evict_select(d["w"], *d["ws"], d["wrows"], d["width"], d["heads"], d["idx"], d["lens"],
                                          d["bs"], d["budget"], d["sink"], d["recent"], d["keep"], d["new"], d["wsp"],
                                          d["nws"], None, None)


def _compact(**kw):
    d = dict(keep=P, budget=40, new=P, lens=P, kc=P, vc=P, kcs=(1024, 128), vcs=(1024, 128), ks=P, vs=P, pages=10, src=P,
             dst=P, page=64, idx=P, w=P, bs=2, heads=8, D=128)
    d.update(kw)
    return mfd_hip.lib().mfd_evict_compact_kv8(d["keep"], d["budget"], d["new"], d["lens"], d["kc"], d["vc"], *d["kcs"],
                                               *d["vcs"], d["ks"], d["vs"], d["pages"], d["src"], 8, 4, 8, d["dst"], 8, 4, 8,
                                               d["page"], d["idx"], d["w"], 800, 100, 4, 100, d["bs"], d["heads"], d["D"],
                                               None, None)


def _head(**kw):
    d = dict(x=P, rs=2560, rpg=15, gs=2560, c=P, e=P, M=15, N=1000, K=2560, out=P, os=1000)
    d.update(kw)
    return mfd_hip.lib().mfd_draft_head_mxfp4(d["x"], d["rs"], d["rpg"], d["gs"], d["c"], d["e"], d["M"], d["N"], d["K"],
                                              d["out"], d["os"], None)


INVALID, UNSUPPORTED = -1, -2
CACHE = [(dict(D=64), UNSUPPORTED, "head dim"), (dict(page=1), UNSUPPORTED, "page_size"),
         (dict(page=48), UNSUPPORTED, "page_size"), (dict(page=512), UNSUPPORTED, "page_size"), (dict(heads=0), INVALID, "sizes"),
         (dict(kc=P + 8), UNSUPPORTED, "alignment"), (dict(kcs=(1024, 100)), UNSUPPORTED, "alignment"),
         (dict(kcs=(1 << 26, 128)), UNSUPPORTED, "strides"), (dict(pages=1 << 27), UNSUPPORTED, "2^31")]


EVERY = [(f, kw, c, w) for f in (_store, _attn, _weigh, _compact) for kw, c, w in CACHE]


@pytest.mark.parametrize("call,kw,code,word", EVERY + [
    (_store, dict(table=None), INVALID, "table"), (_store, dict(k=None), INVALID, "null"),
    (_store, dict(kn=(1020, 128)), UNSUPPORTED, "16-byte"), (_store, dict(v=P + 2), UNSUPPORTED, "16-byte"),
    (_store, dict(bs=-1), INVALID, "sizes"), (_store, dict(most=-1), INVALID, "sizes"), (_store, dict(cu=None), INVALID, "null"),
    (_attn, dict(H=30), INVALID, "sizes"), (_attn, dict(K=0), INVALID, "sizes"), (_attn, dict(K=1 << 17), UNSUPPORTED, "65536"),
    (_attn, dict(scale=0.0), INVALID, "scale"), (_attn, dict(scale=float("nan")), INVALID, "scale"),
    (_attn, dict(q=P + 4), UNSUPPORTED, "16-byte"), (_attn, dict(os=(4096, 12)), UNSUPPORTED, "16-byte"),
    (_attn, dict(kn=None), INVALID, "null"), (_attn, dict(vn=None), INVALID, "null"), (_attn, dict(lens=None), INVALID, "null"),
    (_attn, dict(splits=0), INVALID, "num_ctx_splits"), (_attn, dict(splits=4, keys=100), INVALID, "split_keys"),
    (_attn, dict(splits=4, keys=0, bs=65), INVALID, "split_keys"), (_attn, dict(splits=4, keys=64), INVALID, "workspace"),
    (_attn, dict(splits=4, keys=64, ws=P, nws=100), INVALID, "workspace"),
    (_attn, dict(splits=4, keys=64, ws=P + 8, nws=1 << 30), INVALID, "workspace"),
    (_weigh, dict(decay=-0.1), INVALID, "decay"), (_weigh, dict(decay=float("nan")), INVALID, "decay"),
    (_weigh, dict(lse=None), INVALID, "null"), (_weigh, dict(qs=(1 << 28, 128)), UNSUPPORTED, "2^30"),
    (_select, dict(budget=0), INVALID, "budget"), (_select, dict(sink=20, recent=21), INVALID, "budget"),
    (_select, dict(sink=-1), INVALID, "budget"), (_select, dict(keep=None), INVALID, "null"),
    (_select, dict(nws=100, width=20000), INVALID, "workspace"), (_select, dict(heads=0), INVALID, "sizes"),
    (_compact, dict(budget=0), INVALID, "sizes"), (_compact, dict(keep=None), INVALID, "null"),
    (_compact, dict(src=None), INVALID, "table"), (_compact, dict(dst=None), INVALID, "table"),
    (_head, dict(K=2624), UNSUPPORTED, "128"), (_head, dict(c=P + 8), UNSUPPORTED, "alignment"),
    (_head, dict(e=P + 2), UNSUPPORTED, "alignment"),
    (_head, dict(x=None), INVALID, "null"), (_head, dict(os=999), UNSUPPORTED, "alignment"), (_head, dict(N=0), INVALID, "sizes"),
    (_head, dict(M=-1), INVALID, "sizes"), (_head, dict(rpg=0), INVALID, "sizes"),
])
def test_c_entry_refuses(call, kw, code, word):
    assert call(**kw) == code
    assert word.encode() in mfd_hip.lib().mfd_last_error()


def test_c_entries_with_nothing_to_do():
    assert _store(bs=0) == 0 and _store(N=0) == 0 and _attn(bs=0) == 0 and _weigh(bs=0) == 0 and _select(bs=0) == 0
    assert _compact(bs=0) == 0 and _head(M=0) == 0 and _weigh(wwidth=0) == 0
    lib = mfd_hip.lib()
    assert lib.mfd_kv8_attn_workspace_bytes(2, 8, 16, 32, 8, 1, 1) == 0
    # 4 splits and the block's partial, 2 x 32 x 128 rows: fp16 rows of 128, lse, scale exponent
    assert lib.mfd_kv8_attn_workspace_bytes(2, 8, 16, 32, 8, 1, 4) == 5 * 2 * 32 * 128 * (256 + 8) + 2 * 4
    assert lib.mfd_kv8_attn_workspace_bytes(2, 1, 1, 32, 8, 1, 4) == 4 * 2 * 32 * (256 + 8) + 2 * 4
    assert lib.mfd_evict_select_workspace_bytes(3, 16384) == 0  # (keys in registers)
    assert lib.mfd_evict_select_workspace_bytes(3, 16385) == 3 * 16388 * 4


# ------------------------------------------------------------------------------------------ refusals, Python entry points


def _cache(heads=2, pages=4, page=16):
    d = dict(page_size=page)
    for x in "kv":
        d[x + "_cache"] = torch.zeros(pages * page, heads, 128, dtype=torch.uint8).view(F8)
        d[x + "_scale"] = torch.ones(pages, heads)
    return d


TABLE = torch.zeros(3, 2, dtype=torch.int32)
ROWS = torch.tensor([0, 1])
LENS = torch.tensor([5, 9])


def _good(kind):
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    cache = _cache()
    if kind == "store":
        return kv8_cache.kv8_store, dict(cache, k=bf(3, 2, 128), v=bf(3, 2, 128), page_table=TABLE, req_pool_indices=ROWS,
                                         start_lens=LENS, cu_tokens=torch.tensor([0, 1, 3], dtype=torch.int32), max_tokens=2)
    if kind == "attn":
        return kv8_cache.paged_mode_block_attention_kv8, dict(
            cache, q=bf(8, 4, 128), k_new=bf(8, 2, 128), v_new=bf(8, 2, 128), page_table=TABLE, req_pool_indices=ROWS,
            ctx_lens=LENS, num_modes=2, block_size=2, scaling=0.1)
    if kind == "weights":
        del cache["v_cache"], cache["v_scale"]
        return kv8_cache.attention_weights_kv8, dict(
            cache, q=bf(8, 4, 128), lse=torch.zeros(8, 4), page_table=TABLE, req_pool_indices=ROWS, ctx_lens=LENS, num_modes=2,
            block_size=2, scaling=0.1, weights=torch.zeros(3, 2, 32))
    if kind == "select":
        return kv8_cache.evict_select, dict(weights=torch.zeros(3, 2, 32), req_pool_indices=ROWS, ctx_lens=LENS, budget=8,
                                            sink=1, recent=2)
    return kv8_cache.evict_compact_kv8, dict(cache, keep=torch.zeros(2, 8, dtype=torch.int32), new_lens=LENS, ctx_lens=LENS,
                                             src_table=TABLE, dst_table=TABLE, req_pool_indices=ROWS,
                                             weights=torch.zeros(3, 2, 32))


BAD = [
    ("store", dict(k=torch.zeros(3, 2, 128))), ("store", dict(v=torch.zeros(2, 2, 128, dtype=torch.bfloat16))),
    ("store", dict(cu_tokens=torch.tensor([0, 1, 3]))), ("store", dict(start_lens=torch.tensor([5.0, 9.0]))),
    ("store", dict(page_table=TABLE.long())), ("store", dict(page_size=24)), ("store", dict(page_size=32)),
    ("store", dict(k_scale=torch.ones(4, 2, dtype=torch.float64))), ("store", dict(v_scale=torch.ones(2, 4).t())),
    ("store", dict(k_cache=torch.zeros(64, 2, 128))), ("store", dict(v_cache=torch.zeros(64, 1, 128).to(F8))),
    ("attn", dict(q=torch.zeros(7, 4, 128, dtype=torch.bfloat16))),
    ("attn", dict(q=torch.zeros(8, 3, 128, dtype=torch.bfloat16))),
    ("attn", dict(q=torch.zeros(8, 4, 64, dtype=torch.bfloat16))), ("attn", dict(q=torch.zeros(8, 4, 128))),
    ("attn", dict(k_new=None)), ("attn", dict(v_new=torch.zeros(4, 2, 128, dtype=torch.bfloat16))),
    ("attn", dict(num_modes=0)), ("attn", dict(ctx_lens=torch.tensor([5]))),
    ("attn", dict(req_pool_indices=torch.tensor([[0, 1]]))),
    ("weights", dict(lse=torch.zeros(4, 8))), ("weights", dict(lse=torch.zeros(8, 4).double())),
    ("weights", dict(weights=torch.zeros(3, 4, 32))), ("weights", dict(weights=torch.zeros(3, 2, 32).bfloat16())),
    ("select", dict(weights=torch.zeros(3, 32, 2).transpose(1, 2))), ("select", dict(weights=torch.zeros(64))),
    ("select", dict(ctx_lens=torch.tensor(5))), ("select", dict(keep_out=torch.zeros(2, 8))),
    ("compact", dict(keep=torch.zeros(2, 8))), ("compact", dict(dst_table=TABLE.t())),
    ("compact", dict(weights=torch.zeros(3, 3, 32))),
]


@pytest.mark.parametrize("kind,change", BAD)
def test_python_entry_refuses(kind, change):
    call, args = _good(kind)
    with pytest.raises(ValueError) as e:
        call(**{**args, **change})
    assert "GPU tensors" not in str(e.value)  # the change is what is refused, not the CPU tensors


@pytest.mark.parametrize("kind", ["store", "attn", "weights", "select", "compact"])
def test_cpu_tensors_are_refused_last(kind):
    call, args = _good(kind)
    with pytest.raises(ValueError, match="GPU tensors"):
        call(**args)


# ------------------------------------------------------------------------------------------------------ the 4-bit head


def test_quantize_takes_the_nearest_code():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(40, 256, generator=g) * torch.exp2(torch.randint(-20, 20, (40, 1), generator=g).float())
    w[3] = 0
    w[5, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])  # borders: the even code
    w[5, 8:32] = 0
    q = mxfp4_head.quantize(w)
    mxfp4_head.check_weight(*q, values=True)
    back = mxfp4_head.dequantize(q).double()
    assert back[3].abs().max() == 0 and back[5, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    scale = torch.exp2(q.exps.double() - 127).repeat_interleave(32, 1)
    grid = torch.tensor(mxfp4_head.E2M1, dtype=torch.float64)
    best = ((w.double().abs() / scale)[..., None] - grid).abs().amin(-1) * scale
    assert bool(((back - w.double()).abs() <= best * (1 + 1e-12)).all())
    top = (w.double().abs() / scale).view(40, -1, 32).amax(-1)
    assert bool(((top > 3.5) & (top <= 7) | (top == 0)).all())


def test_head_refusals():
    codes, exps = torch.zeros(10, 64, dtype=torch.uint8), torch.full((10, 4), 120, dtype=torch.uint8)
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    for bad in (dict(codes=codes.int()), dict(exps=exps[:, :3]), dict(codes=codes[:, :32]), dict(codes=codes.t()),
                dict(x=x.float()), dict(x=x[:, :64])):
        with pytest.raises(ValueError) as e:
            mxfp4_head.draft_head_mxfp4(**{**dict(x=x, codes=codes, exps=exps), **bad})
        assert "GPU tensors" not in str(e.value)
    with pytest.raises(ValueError, match="GPU tensors"):
        mxfp4_head.draft_head_mxfp4(x, codes, exps)
    for e in (0, 253, 255):
        exps[2, 1] = e
        with pytest.raises(ValueError, match="exponents"):
            mxfp4_head.check_weight(codes, exps, values=True)
    with pytest.raises(ValueError, match="128"):
        mxfp4_head.quantize(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="finite"):
        mxfp4_head.quantize(torch.full((4, 128), float("inf")))


# ------------------------------------------------------------------------------------------------ pool, reference, splits


def test_reference_path_over_an_8_bit_pool():
    """PagedModeAttention(impl="reference") over a Kv8Pool whose pages were filled by the oracle's store."""
    page, heads, H, K, L = 16, 2, 4, 2, 3
    pool = kv8_cache.Kv8Pool(num_layers=2, num_pages=9, page_size=page, num_kv_heads=heads, device="cpu")
    g = torch.Generator().manual_seed(11)
    lens = [37, 16]
    table = torch.tensor([[0, 0, 0], [4, 1, 7], [3, 0, 0]], dtype=torch.int32)
    for x, cache, scale in zip("kv", pool.get_kv_buffer(1), pool.get_kv_scale(1)):
        values, s = cache.float().double().numpy(), scale.double().numpy()
        kv8.store(torch.randn(53, heads, 128, generator=g).double().numpy(), values, s, table.numpy(), [1, 2], [0, 0],
                  [0, 37, 53], page)
        cache.copy_(torch.from_numpy(values).float().to(F8))
        scale.copy_(torch.from_numpy(s).float())
    T = 2 * K * L
    q, k, v = (torch.randn(T, n * 128, generator=g) for n in (H, heads, heads))
    batch = type("Batch", (), dict(req_pool_indices=torch.tensor([1, 2]), seq_lens=torch.tensor(lens)))()
    attn = paged_mode_attention.PagedModeAttention(
        kv_pool=pool, req_to_token=table, num_modes=K, block_size=L, num_heads=H, num_kv_heads=heads, head_dim=128,
        scaling=128 ** -0.5, num_ctx_splits=-1, impl="reference", page_size=page)
    got = attn(q, k, v, batch, 1).view(T, H, 128)
    f = lambda t: t.double().numpy()  # noqa: E731
    for b, n in enumerate(lens):
        ctx = [kv8.tokens(f(c.float()), f(s), table[b + 1].numpy(), n, page)
               for c, s in zip(pool.get_kv_buffer(1), pool.get_kv_scale(1))]
        r = slice(b * K * L, (b + 1) * K * L)
        ref = kv8.attention(f(q[r].view(-1, H, 128)), f(k[r].view(-1, heads, 128)), f(v[r].view(-1, heads, 128)), *ctx, K, L,
                            128 ** -0.5)[0]
        assert np.abs(f(got[r]) - ref).max() <= 1e-5 * np.abs(ref).max()


def test_pool_refuses_page_sizes():
    with pytest.raises(ValueError, match="page_size"):
        kv8_cache.Kv8Pool(num_layers=1, num_pages=2, page_size=100, num_kv_heads=1, device="cpu")


@pytest.mark.parametrize("bs,heads,rows", [(1, 8, 4), (16, 8, 5), (64, 8, 4), (1, 8, 512), (16, 8, 640), (4, 2, 64), (65, 1, 3)])
def test_split_choice_covers_the_context(monkeypatch, bs, heads, rows):
    monkeypatch.setattr(mfd_hip, "cu_count", lambda device: 256)
    for ctx in (1, 63, 64, 65, 1000, 8192, 100001):
        splits, keys = kv8_cache._auto_splits(bs, heads, rows, True, ctx, None)
        if keys == 0:  # one pass, or measured out on the device
            assert splits == 1 or 1 < bs <= 64 and 1 < splits <= 32
        else:
            assert splits > 1 and keys % 64 == 0 and (splits - 1) * keys < ctx <= splits * keys
        for want in (2, 3, 64):
            s, k = kv8_cache._splits_of(want, ctx)
            assert 1 <= s <= want and k % 64 == 0 and (s - 1) * k < ctx <= s * k
