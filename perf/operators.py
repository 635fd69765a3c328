"""Performance cases of the draft step in fewer bits on one MI355X: an 8-bit draft KV cache, its eviction, and a 4-bit
draft head.

A draft token that lost precision costs an accepted token and never a wrong one (the target verifies it), so the
drafter's cache, its length and its LM head are where a serving loop saves bytes. ``prepare`` makes what the loop holds
before the call, ``run`` makes one pass: in plain torch, or through the public entry points where ``own`` is true.

Kinds of work (``case["kind"]``):
  store      new keys and values of a batch rounded into the paged 8-bit cache, a scale for each page and head
  attn       mode attention of a batch over that cache (one mode of one token: plain decoding), with its log-sum-exp
  weights    attention weight that each cached token received in the step, added to its running sum
  evict      the tokens to keep by those sums, then cache and sums compacted to them (into fresh pages)
  head       drafted hidden states times an LM head in 4 bits (e2m1, a power-of-two scale for 32 weights)

The cache holds e4m3 codes [slots, KV heads, 128] and float32 scales [pages, KV heads], powers of two between 2^-40 and
2^40: the smallest that puts the page's largest magnitude at or below 448, never shrinking while a page fills.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False  # set by the tools: whether run() calls the framework's operators

D = 128  # head dim of every configuration
DEV = "cuda"
F8 = torch.float8_e4m3fn
SCALING = D ** -0.5
_MIN_EXP, _MAX_EXP = -40, 40

# Context lengths of 16 running requests, uniform over 1024 .. 8192 (the batch of the paged attention's configuration),
# and the tokens that a round of them accepted.
_CTX16 = "7316,1903,5221,2874,6650,1187,4096,8033,3519,5902,1466,7704,2333,4777,6128,3050"
_NEW16 = "5,1,9,3,16,2,7,1,4,12,1,6,3,8,2,10"


def _package():
    """The framework's modules (its directory on the path as a user puts it)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "multi-future-drafting_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import kv8_cache
    import mxfp4_head

    return kv8_cache, mxfp4_head


def listed():
    return [
        # A verified round's accepted tokens of 16 requests go into the cache: the smallest store, latency.
        dict(name="store_round16", kind="store", start=_CTX16, new=_NEW16, hkv=8, page=64),
        # Prompts of four requests enter the cache, one of them behind a shared prefix that ends inside a page.
        dict(name="store_prompts", kind="store", start="0,0,1000,0", new="8192,4096,3001,1187", hkv=8, page=64),
        # One user's plain decode step (no draft modes): the smallest attention, where launches count.
        dict(name="attn_one_token", kind="attn", ctx="1187", modes=1, block=1, h=32, hkv=8, page=64, fresh=True),
        # Plain decoding of a continuous batch at longer contexts: the stream of the cache.
        dict(name="attn_decode16", kind="attn", modes=1, block=1, h=40, hkv=8, page=64, fresh=True,
             ctx="29264,7612,20884,11496,26600,4748,16384,32132,14076,23608,5864,30816,9332,19108,24512,12200"),
        # One request's draft step: 8 modes x 16 tokens over 4096 context tokens.
        dict(name="attn_ctx4096", kind="attn", ctx="4096", modes=8, block=16, h=32, hkv=8, page=64, fresh=True),
        # The continuous batch's draft step: 16 requests, 40 heads over 8.
        dict(name="attn_16", kind="attn", ctx=_CTX16, modes=8, block=16, h=40, hkv=8, page=64, fresh=True),
        # What that draft step's queries attended to, for one request and for the batch.
        dict(name="weights_ctx4096", kind="weights", ctx="4096", modes=8, block=16, h=32, hkv=8, page=64),
        dict(name="weights_16", kind="weights", ctx=_CTX16, modes=8, block=16, h=40, hkv=8, page=64),
        # One request cut from 8192 tokens to 2048; a batch cut to 1024 each (some of it shorter).
        dict(name="evict_8192", kind="evict", ctx="8192", budget=2048, hkv=8, page=64),
        dict(name="evict_16", kind="evict", ctx=_CTX16 + "," + _CTX16.replace("1187", "900"), budget=1024, hkv=8, page=64),
        # The draft head over the full vocabulary: one mode of 16 tokens, and the 8 modes of one request.
        dict(name="head_15", kind="head", rows=15, hidden=2560, vocab=151936),
        dict(name="head_120", kind="head", rows=120, hidden=2560, vocab=151936),
    ]


# ---------------------------------------------------------------------------------------------- drawn cases


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    """One more case of the same ranges, odd and ragged sizes among them."""
    kind = rng.choice(["store", "store", "attn", "attn", "attn", "weights", "weights", "evict", "evict", "head", "head"])
    page = rng.choice([16, 32, 64, 64, 64, 128])
    hkv = rng.choice([2, 4, 8, 8])
    text = lambda v: ",".join(map(str, v))  # noqa: E731
    if kind == "store":
        bs = _log_int(rng, 1, 24)
        top = rng.choice([1, 16, 16, 8192])
        new = [_log_int(rng, 1, top) for _ in range(bs)]
        while sum(new) > 16000:
            new.pop()
        return dict(kind=kind, start=text(rng.choice([0, _log_int(rng, 1, 8192)]) for _ in new), new=text(new), hkv=hkv,
                    page=page)
    if kind in ("attn", "weights"):
        modes, block = rng.choice([(1, 1), (1, 1), (1, 16), (3, 16), (4, 7), (8, 16), (8, 16)])
        h = hkv * rng.choice([1, 2, 4, 4, 5, 8])
        cost = 0
        ctx = []
        for _ in range(_log_int(rng, 1, 16)):
            ctx.append(_log_int(rng, 16, 32768 if modes * block == 1 else 8192))
            cost += ctx[-1] * h * modes * block
            if cost > 3.5e8 and len(ctx) > 1:  # (16 requests of the listed batch: 3.7e8)
                ctx.pop()
                break
        case = dict(kind=kind, ctx=text(ctx), modes=modes, block=block, h=h, hkv=hkv, page=page)
        return dict(case, fresh=modes * block > 1 or rng.random() < 0.5) if kind == "attn" else case
    if kind == "evict":
        ctx = [_log_int(rng, 64, 16384) for _ in range(_log_int(rng, 1, 24))]
        return dict(kind=kind, ctx=text(ctx), budget=_log_int(rng, 64, 2048), hkv=hkv, page=page)
    vocab = _log_int(rng, 4000, 151936)
    if rng.random() < 0.5:
        vocab = vocab // 64 * 64
    return dict(kind=kind, rows=_log_int(rng, 1, 128), hidden=rng.choice([1024, 2048, 2560, 4096]) if vocab < 90000
                else 2560, vocab=vocab)


# ---------------------------------------------------------------------------------------------- inputs


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _dev(values, dtype):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _pages(case, lens, g, more=0):
    """A pool of pages for these lengths in random order, with one page in eight unused, and the page table. Rows 0 and
    1 of the table belong to nobody, as in a serving pool. ``more``: pages of a second table, disjoint from the first."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    extra = [-(-more // page)] * len(lens) if more else []
    total = (sum(need) + sum(extra)) * 9 // 8 + 2
    perm = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    tables, at = [], 0
    for counts in (need, extra):
        if counts:
            table = torch.zeros(len(lens) + 2, max(counts), dtype=torch.int32, device=DEV)
            for b, n in enumerate(counts):
                table[b + 2, :n] = perm[at:at + n]
                at += n
            tables.append(table)
    return total, tables


def _cache(pages, hkv, page, spread, g):
    """Codes and scales of a filled cache: values of about ``spread``, head sizes a factor of a few apart."""
    size = torch.exp2(torch.randint(-1, 3, (pages, hkv), device=DEV, generator=g).float()) * spread / 448 * 4
    scale = torch.exp2(torch.ceil(torch.log2(size)))
    x = _randn(g, pages, page, hkv, D) * 96  # four deviations fit the type's 448
    return x.clamp_(-448, 448).to(F8).view(pages * page, hkv, D), scale


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = dict(case=dict(case))
    if kind == "head":
        V, H = case["vocab"], case["hidden"]
        s["x"] = _randn(g, case["rows"], H).to(torch.bfloat16)
        s["codes"] = torch.randint(0, 256, (V, H // 2), device=DEV, generator=g, dtype=torch.uint8)
        s["exps"] = torch.randint(117, 122, (V, H // 32), device=DEV, generator=g, dtype=torch.uint8)
        return s
    hkv, page = case["hkv"], case["page"]
    lens = _ints(case["ctx"]) if kind != "store" else [a + n for a, n in zip(_ints(case["start"]), _ints(case["new"]))]
    bs = len(lens)
    total, tables = _pages(case, lens, g, more=case["budget"] if kind == "evict" else 0)
    s["table"] = tables[0]
    s["k_cache"], s["k_scale"] = _cache(total, hkv, page, 2.0, g)
    s["v_cache"], s["v_scale"] = _cache(total, hkv, page, 1.0, g)
    s["rows"] = torch.arange(2, bs + 2, device=DEV)
    if kind == "store":
        new = _ints(case["new"])
        n = sum(new)
        # keys carry a few large channels, as they do in practice
        gain = torch.exp2(torch.randint(-2, 3, (1, hkv, D), device=DEV, generator=g).float())
        s["k"] = (_randn(g, n, hkv, D) * gain).to(torch.bfloat16)
        s["v"] = _randn(g, n, hkv, D).to(torch.bfloat16)
        s["start"] = _dev(_ints(case["start"]), torch.int64)
        s["cu"] = _dev([0] + torch.tensor(new).cumsum(0).tolist(), torch.int32)
        s["max_new"] = max(new)
        return s
    s["lens"] = _dev(lens, torch.int64)
    if kind == "evict":
        s["dst_table"] = tables[1]
        # running sums: heavy-tailed over the tokens, and a head of its own taste
        width = max(lens)
        s["weights"] = torch.exp(_randn(g, bs + 2, hkv, width) + 2 * _randn(g, bs + 2, 1, width))
        return s
    KL = case["modes"] * case["block"]
    T = bs * KL
    s["q"] = _randn(g, T, case["h"], D).to(torch.bfloat16)
    if kind == "weights":
        s["lse"] = _plain_attention(s, case, blocks=False)[1]
        s["weights"] = torch.rand(bs + 2, hkv, max(lens), device=DEV, generator=g) * 4
        return s
    s["fresh"] = case["fresh"]
    s["k_new"] = (_randn(g, T, hkv, D) * 2).to(torch.bfloat16)
    s["v_new"] = _randn(g, T, hkv, D).to(torch.bfloat16)
    return s


# ---------------------------------------------------------------------------------------------- plain forms


def _codes(x, scale):
    """e4m3 codes of x / scale (the division is exact: scales are powers of two)."""
    return (x / scale).clamp(-448, 448).to(F8)


def _page_scale(amax):
    """The smallest power of two s with amax / s <= 448, within the cache's range."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(amax > 0, torch.where(m > 0.875, e - 8, e - 9), torch.full_like(e, _MIN_EXP))
    return torch.exp2(e.clamp(_MIN_EXP, _MAX_EXP).float())


def _plain_store(x, cache, scale, pages, offsets, page):
    """x [n, hkv, D] into entry offsets[i] of page pages[i], the scales grown and the older entries of a page rounded
    again where its scale grew."""
    hkv = x.shape[1]
    x = x.float()
    n_pages = scale.shape[0]
    where = pages[:, None].expand(-1, hkv)
    amax = torch.zeros(n_pages, hkv, device=DEV).scatter_reduce_(0, where, x.abs().amax(-1), "amax")
    first = torch.full((n_pages,), page, device=DEV).scatter_reduce_(0, pages, offsets, "amin")  # page: untouched
    old = torch.where((first == 0)[:, None], torch.zeros_like(scale), scale)  # a page begun anew forgets its scale
    new = torch.where((first < page)[:, None], torch.maximum(old, _page_scale(amax)), scale)
    touched = torch.unique(pages)
    paged = cache.view(torch.uint8).view(n_pages, page, hkv, D)
    kept = paged[touched].view(F8).float() * scale[touched][:, None, :, None]
    kept = _codes(kept, new[touched][:, None, :, None]).view(torch.uint8)
    older = torch.arange(page, device=DEV)[None] < first[touched][:, None]
    paged[touched] = torch.where(older[:, :, None, None], kept, paged[touched])
    scale.copy_(new)
    paged[pages, offsets] = _codes(x, scale[pages][:, :, None]).view(torch.uint8)


def _run_store(s, case):
    page = case["page"]
    cu = s["cu"].long()
    i = torch.arange(s["k"].shape[0], device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    pos = s["start"][b] + i - cu[b]
    pages, offsets = s["table"][s["rows"][b], pos // page].long(), pos % page
    _plain_store(s["k"], s["k_cache"], s["k_scale"], pages, offsets, page)
    _plain_store(s["v"], s["v_cache"], s["v_scale"], pages, offsets, page)
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _slots(s, lens, page, width):
    """Slots [bs, width] of the requests' tokens (past a length: the last one) and whether there is a token."""
    t = torch.arange(width, device=DEV)
    there = t[None] < lens[:, None]
    at = torch.minimum(t[None], (lens - 1).clamp(min=0)[:, None])
    return s["table"][s["rows"][:, None], at // page].long() * page + at % page, there


def _values(cache, scale, slots, page):
    """Decoded rows [bs, hkv, width, D] in float32."""
    x = cache.view(torch.uint8)[slots].view(F8).float() * scale[slots // page][..., None]
    return x.transpose(1, 2).contiguous()


def _grouped(q, bs, KL, hkv):
    """q [bs KL, H, D] as [bs, hkv, G KL, D] float32."""
    G = q.shape[1] // hkv
    return q.float().view(bs, KL, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(bs, hkv, G * KL, D)


def _plain_attention(s, case, blocks):
    """(output [T, H, D] float32, natural log-sum-exp [T, H]) over the cache and, with ``blocks``, each mode's own
    keys."""
    K, L, hkv, page = case["modes"], case["block"], case["hkv"], case["page"]
    KL, H = K * L, case["h"]
    G, bs = H // hkv, s["lens"].numel()
    slots, there = _slots(s, s["lens"], page, s["table"].shape[1] * page)
    q = _grouped(s["q"], bs, KL, hkv)
    k = _values(s["k_cache"], s["k_scale"], slots, page)
    v = _values(s["v_cache"], s["v_scale"], slots, page)
    sc = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(SCALING)
    sc.masked_fill_(~there[:, None, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    if blocks:
        own_k = s["k_new"].float().view(bs, K, L, hkv, D).permute(0, 3, 1, 2, 4)[:, :, None]  # [bs, hkv, 1, K, L, D]
        own_v = s["v_new"].float().view(bs, K, L, hkv, D).permute(0, 3, 1, 2, 4)[:, :, None]
        sb = torch.matmul(q.view(bs, hkv, G, K, L, D), own_k.transpose(-1, -2).contiguous()) * SCALING
        m = torch.maximum(m, sb.amax(-1).view(m.shape))
    p = sc.sub_(m).exp_()
    total, out = p.sum(-1, keepdim=True), torch.matmul(p, v)
    if blocks:
        pb = torch.exp(sb - m.view(bs, hkv, G, K, L, 1))
        total = total + pb.sum(-1).view(m.shape)
        out = out + torch.matmul(pb, own_v).view(out.shape)
    back = lambda x: x.view(bs, hkv, G, KL, -1).permute(0, 3, 1, 2, 4).reshape(bs * KL, H, -1)  # noqa: E731
    return back(out / total), back(m + torch.log(total))[..., 0].contiguous()


def _run_attn(s, case):
    o, lse = _plain_attention(s, case, s["fresh"])
    return o.to(torch.bfloat16), lse


def _run_weights(s, case):
    hkv, page, H = case["hkv"], case["page"], case["h"]
    KL, bs = case["modes"] * case["block"], s["lens"].numel()
    width = s["weights"].shape[-1]
    slots, there = _slots(s, s["lens"], page, width)
    k = _values(s["k_cache"], s["k_scale"], slots, page)
    sc = torch.matmul(_grouped(s["q"], bs, KL, hkv), k.transpose(-1, -2).contiguous()).mul_(SCALING)
    lse = s["lse"].view(bs, KL, hkv, H // hkv).permute(0, 2, 3, 1).reshape(bs, hkv, -1, 1)
    w = sc.sub_(lse).exp_().sum(2)
    before = s["weights"][s["rows"]]
    s["weights"][s["rows"]] = torch.where(there[:, None, :], 0.9 * before + w, before)
    return s["weights"]


_SINK, _RECENT = 4, 32


def _plain_select(w, lens, budget):
    """Indices of the kept tokens, ascending, -1 behind them, and their number. ``w`` [bs, hkv, width]."""
    width = w.shape[-1]
    t = torch.arange(width, device=DEV)[None]
    score = w.double().sum(1).float()
    recent = (lens - _RECENT)[:, None]
    always = (t < _SINK) | (t >= recent)
    key = torch.where(always, torch.full_like(score, math.inf), score)
    key = torch.where(t < lens[:, None], key, torch.full_like(score, -math.inf))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :budget]
    n = torch.minimum(lens, torch.full_like(lens, budget))
    kept = torch.arange(order.shape[1], device=DEV)[None] < n[:, None]
    keep = torch.sort(torch.where(kept, order, torch.full_like(order, width)), dim=1).values
    keep = torch.where(keep < width, keep, torch.full_like(keep, -1)).to(torch.int32)
    if keep.shape[1] < budget:
        keep = torch.nn.functional.pad(keep, (0, budget - keep.shape[1]), value=-1)
    return keep, n


def _plain_move(cache, scale, src, dst_pages, there, page):
    """Kept rows [bs, m] (slots src) into pages dst_pages [bs, m / page], rounded with the pages' own scales."""
    bs, m = src.shape
    hkv = cache.shape[1]
    x = cache.view(torch.uint8)[src].view(F8).float() * scale[src // page][..., None]
    x = torch.where(there[:, :, None, None], x, torch.zeros_like(x)).view(bs, m // page, page, hkv, D)
    new = _page_scale(x.abs().amax((2, 4)))
    codes = _codes(x, new[:, :, None, :, None]).view(torch.uint8)
    used = there.view(bs, m // page, page)
    paged = cache.view(torch.uint8).view(-1, page, hkv, D)
    pages = dst_pages[used[:, :, 0]]  # the pages that get a token
    paged[pages] = torch.where(used[used[:, :, 0]][:, :, None, None], codes[used[:, :, 0]], paged[pages])
    scale[pages] = new[used[:, :, 0]]


def _run_evict(s, case):
    page, budget = case["page"], case["budget"]
    rows, lens, weights = s["rows"], s["lens"], s["weights"]
    keep, n = _plain_select(weights[rows], lens, budget)
    m = s["dst_table"].shape[1] * page
    at = torch.nn.functional.pad(keep, (0, m - budget), value=-1).long()
    there = at >= 0
    at = at.clamp(min=0)
    src = s["table"][rows[:, None], at // page].long() * page + at % page
    dst = s["dst_table"][rows].long()
    _plain_move(s["k_cache"], s["k_scale"], src, dst, there, page)
    _plain_move(s["v_cache"], s["v_scale"], src, dst, there, page)
    width = weights.shape[-1]
    old = weights[rows]
    moved = torch.gather(old, 2, at[:, None, :min(m, width)].expand(-1, old.shape[1], -1))
    moved = torch.nn.functional.pad(moved, (0, width - moved.shape[2]))
    t = torch.arange(width, device=DEV)[None, None]
    new = torch.where(t < n[:, None, None], moved, torch.zeros_like(moved))
    weights[rows] = torch.where(t < lens[:, None, None], new, old)
    return keep, n, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], weights


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _run_head(s, case):
    V, H = case["vocab"], case["hidden"]
    values = torch.tensor(_E2M1, device=DEV)
    pair = torch.stack([values.repeat(16), values.repeat_interleave(16)], dim=1)  # low half first
    w = pair[s["codes"].int()].view(V, H // 32, 32) * torch.exp2(s["exps"].float() - 127)[:, :, None]
    return torch.matmul(s["x"].float(), w.view(V, H).t()).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------- one pass


def _own(s, case):
    kv8_cache, mxfp4_head = _package()
    kind = case["kind"]
    if kind == "head":
        return mxfp4_head.draft_head_mxfp4(s["x"], s["codes"], s["exps"])
    cache = dict(k_cache=s["k_cache"], v_cache=s["v_cache"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                 page_size=case["page"], req_pool_indices=s["rows"])
    if kind == "store":
        kv8_cache.kv8_store(k=s["k"], v=s["v"], page_table=s["table"], start_lens=s["start"], cu_tokens=s["cu"],
                            max_tokens=s["max_new"], **cache)
        return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if kind == "attn":
        return kv8_cache.paged_mode_block_attention_kv8(
            q=s["q"], k_new=s["k_new"] if s["fresh"] else None, v_new=s["v_new"] if s["fresh"] else None,
            page_table=s["table"], ctx_lens=s["lens"], num_modes=case["modes"], block_size=case["block"],
            scaling=SCALING, max_ctx=max(_ints(case["ctx"])), return_lse=True, **cache)
    if kind == "weights":
        kv8_cache.attention_weights_kv8(
            q=s["q"], lse=s["lse"], k_cache=s["k_cache"], k_scale=s["k_scale"], page_size=case["page"],
            page_table=s["table"], req_pool_indices=s["rows"], ctx_lens=s["lens"], num_modes=case["modes"],
            block_size=case["block"], scaling=SCALING, weights=s["weights"], decay=0.9)
        return s["weights"]
    keep, n = kv8_cache.evict_select(weights=s["weights"], req_pool_indices=s["rows"], ctx_lens=s["lens"],
                                     budget=case["budget"], sink=_SINK, recent=_RECENT)
    kv8_cache.evict_compact_kv8(keep=keep, new_lens=n, ctx_lens=s["lens"], src_table=s["table"],
                                dst_table=s["dst_table"], weights=s["weights"], **cache)
    return keep, n, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["weights"]


def run(state):
    case = state["case"]
    return _own(state, case) if own else globals()["_run_" + case["kind"]](state, case)


# ---------------------------------------------------------------------------------------------- what a pass needs


def work(case):
    kind = case["kind"]
    if kind == "head":
        M, V, H = case["rows"], case["vocab"], case["hidden"]
        return dict(bytes=V * H // 2 + V * H // 32 + 2 * M * H + 2 * M * V, flops=2.0 * M * V * H)
    hkv = case["hkv"]
    if kind == "store":
        # new keys and values read in bf16, written in 8 bits (with it, the entries of begun pages once each way)
        page = case["page"]
        older = sum(a % page for a in _ints(case["start"]))
        n = sum(_ints(case["new"]))
        return dict(bytes=2 * hkv * D * (3 * n + 2 * older), flops=4.0 * hkv * D * n)
    lens = _ints(case["ctx"])
    if kind == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        return dict(bytes=4 * hkv * (sum(lens) * 2 + kept) + 4 * hkv * D * kept, flops=float(hkv * sum(lens)))
    KL, H = case["modes"] * case["block"], case["h"]
    T = len(lens) * KL
    if kind == "weights":
        return dict(bytes=sum(lens) * hkv * (D + 8) + T * H * (2 * D + 4), flops=2.0 * H * KL * D * sum(lens))
    L = case["block"] if case["fresh"] else 0
    return dict(bytes=2 * sum(lens) * hkv * D + T * (4 * H * D + 4 * H + (4 * hkv * D if L else 0)),
                flops=4.0 * H * KL * D * sum(n + L for n in lens))


# ---------------------------------------------------------------------------------------------- from the definition


def _exact_scale(amax):
    """Power-of-two scales of float64 magnitudes by comparison with the 81 there are."""
    steps = torch.exp2(torch.arange(_MIN_EXP, _MAX_EXP + 1, device=DEV, dtype=torch.float64))
    return steps[torch.searchsorted(steps[:-1] * 448, amax.contiguous())]


def _exact_codes(x):
    """x (float64) rounded to e4m3, ties to even, as float64 values."""
    a = x.abs().clamp(max=448)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(a / step) * step, x)


def _tokens64(s, b, n, page, cache, scale):
    """Decoded rows [n, hkv, D] of request b."""
    t = torch.arange(n, device=DEV)
    pages = s["table"][b + 2].long()[t // page]
    return cache.double()[pages * page + t % page] * scale.double()[pages][:, :, None]


def _exact_store(s, case):
    page, hkv = case["page"], case["hkv"]
    start, new = _ints(case["start"]), _ints(case["new"])
    out = []
    for which in "kv":
        x, cache, scale = s[which].double(), s[which + "_cache"].double(), s[which + "_scale"].double()
        at = 0
        for b, (a, n) in enumerate(zip(start, new)):
            for p in range(a // page, -(-(a + n) // page)):
                lo, hi = max(a, p * page), min(a + n, (p + 1) * page)
                pg = int(s["table"][b + 2, p])
                rows = x[at + lo - a:at + hi - a]
                sc = _exact_scale(rows.abs().amax((0, 2)))
                before = lo - p * page
                if before:
                    sc = torch.maximum(sc, scale[pg])
                    older = cache[pg * page:pg * page + before] * scale[pg][None, :, None]
                    cache[pg * page:pg * page + before] = _exact_codes(older / sc[None, :, None])
                cache[pg * page + before:pg * page + hi - p * page] = _exact_codes(rows / sc[None, :, None])
                scale[pg] = sc
            at += n
        out.append((cache, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attn(s, case):
    K, L, H, hkv, page = case["modes"], case["block"], case["h"], case["hkv"], case["page"]
    KL, G = K * L, H // hkv
    lens = _ints(case["ctx"])
    out = torch.zeros(len(lens) * KL, H, D, device=DEV, dtype=torch.float64)
    lse = torch.zeros(len(lens) * KL, H, device=DEV, dtype=torch.float64)
    mode = torch.arange(KL, device=DEV) // L
    for b, n in enumerate(lens):
        rows = slice(b * KL, (b + 1) * KL)
        k = _tokens64(s, b, n, page, s["k_cache"], s["k_scale"])
        v = _tokens64(s, b, n, page, s["v_cache"], s["v_scale"])
        if s["fresh"]:
            k, v = torch.cat([k, s["k_new"][rows].double()]), torch.cat([v, s["v_new"][rows].double()])
        for h in range(H):
            sc = s["q"][rows, h].double() @ k[:, h // G].t() * SCALING
            if s["fresh"]:
                sc[:, n:].masked_fill_(mode[:, None] != mode[None], -math.inf)
            lse[rows, h] = torch.logsumexp(sc, -1)
            out[rows, h] = torch.softmax(sc, -1) @ v[:, h // G]
    return out, lse


def _exact_weights(s, case):
    KL, G = case["modes"] * case["block"], case["h"] // case["hkv"]
    w = s["weights"].double()
    for b, n in enumerate(_ints(case["ctx"])):
        k = _tokens64(s, b, n, case["page"], s["k_cache"], s["k_scale"])
        w[b + 2, :, :n] *= 0.9
        for h in range(case["h"]):
            sc = s["q"][b * KL:(b + 1) * KL, h].double() @ k[:, h // G].t() * SCALING
            w[b + 2, h // G, :n] += torch.exp(sc - s["lse"][b * KL:(b + 1) * KL, h, None].double()).sum(0)
    return w


def _exact_evict(s, case):
    page, budget, hkv = case["page"], case["budget"], case["hkv"]
    lens = _ints(case["ctx"])
    keep = torch.full((len(lens), budget), -1, dtype=torch.int32, device=DEV)
    weights = s["weights"].double()
    new = {x: [s[x + "_cache"].double(), s[x + "_scale"].double()] for x in "kv"}
    counts = []
    for b, n in enumerate(lens):
        score = s["weights"][b + 2, :, :n].double().sum(0).float().tolist()
        ends = [t for t in range(n) if t < _SINK or t >= n - _RECENT][:budget]
        rest = sorted((t for t in range(_SINK, n - _RECENT)), key=lambda t: (-score[t], t))
        kept = sorted(ends + rest[:max(0, budget - len(ends))])
        counts.append(len(kept))
        idx = torch.tensor(kept, device=DEV)
        keep[b, :len(kept)] = idx.int()
        for x in "kv":
            rows = _tokens64(s, b, n, page, s[x + "_cache"], s[x + "_scale"])[idx]
            for p in range(0, len(kept), page):
                part = rows[p:p + page]
                pg = int(s["dst_table"][b + 2, p // page])
                sc = _exact_scale(part.abs().amax((0, 2)))
                new[x][0][pg * page:pg * page + len(part)] = _exact_codes(part / sc[None, :, None])
                new[x][1][pg] = sc
        weights[b + 2, :, :len(kept)] = s["weights"][b + 2].double()[:, idx]
        weights[b + 2, :, len(kept):n] = 0
    return (keep, torch.tensor(counts, device=DEV), new["k"][0], new["v"][0], new["k"][1], new["v"][1], weights)


def _exact_head(s, case):
    x = s["x"].double()
    lut = torch.tensor(_E2M1, device=DEV, dtype=torch.float64)
    parts = []
    for lo in range(0, case["vocab"], 16384):
        c = s["codes"][lo:lo + 16384].long()
        w = torch.empty(c.shape[0], case["hidden"], device=DEV, dtype=torch.float64)
        w[:, 0::2], w[:, 1::2] = lut[c & 15], lut[c >> 4]
        w *= torch.exp2(s["exps"][lo:lo + 16384].double() - 127).repeat_interleave(32, dim=1)
        parts.append(x @ w.t())
    return torch.cat(parts, dim=1)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed), case)
