"""The draft KV cache in 8 bits on MI355X: its store, the mode attention that reads it, and its eviction by the attention
weight that each token received (csrc/kv8_cache.hip, csrc/kv8_attn.hip).

A draft token that lost precision costs an accepted token and never a wrong one: the target verifies it. So the
drafter's cache is where half the bytes and a bounded length are free of risk. The cache is paged: token t of request b
lies at slot page_table[req_pool_indices[b], t // page_size] * page_size + t % page_size of
  k_cache, v_cache  [slots, KV heads, 128]  torch.float8_e4m3fn codes
  k_scale, v_scale  [pages, KV heads]       float32, a power of two between 2^-40 and 2^40; a value is code * scale
page_size is 16, 32, 64, 128 or 256. Index arguments: page tables int32, the others int64 (int32 is converted).

``err_flag`` (optional, int32 [1] on the device) gets mfd_hip.DEVERR_BAD_PAGE OR-ed in where a page id, table row,
length or token count lies outside its bounds; nothing out of bounds is read or written. Every call works on the tensors'
own device and its current stream, synchronises nothing, and can be captured in a graph (lengths are read on the device).
"""

from __future__ import annotations

from typing import Optional

import torch

import mfd_hip

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128, 256)
CODE_DTYPE = torch.float8_e4m3fn
UNIT = 32        # query rows of a unit of the kernels
TILE_KEYS = 64   # split_keys come in multiples of it


# ------------------------------------------------------------------------------------------------ argument checks
# A draft step calls these for every layer, with kernels of 5 to 30 us behind them: each check reads a tensor's attributes
# once (0.04 us each), dtypes are compared by identity.


def _cache_args(k_cache, v_cache, k_scale, v_scale, page_size: int):
    """(k pointer, v pointer, slot and head strides of both, scale pointers, pages) of a cache, and its KV heads."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
    shape, scales = k_cache.shape, k_scale.shape
    ks, vs = k_cache.stride(), v_cache.stride()
    if k_cache.dtype is not CODE_DTYPE or v_cache.dtype is not CODE_DTYPE or len(shape) != 3 or shape[2] != HEAD_DIM or \
            v_cache.shape != shape or ks[2] != 1 or vs[2] != 1:
        raise ValueError(f"k_cache and v_cache must be {CODE_DTYPE} [slots, KV heads, {HEAD_DIM}] with contiguous rows, got "
                         f"{k_cache.dtype} {tuple(shape)} and {v_cache.dtype} {tuple(v_cache.shape)}")
    heads = shape[1]
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or len(scales) != 2 or \
            v_scale.shape != scales or scales[1] != heads or scales[0] * page_size != shape[0] or \
            not k_scale.is_contiguous() or not v_scale.is_contiguous():
        raise ValueError(f"k_scale and v_scale must be contiguous float32 [{shape[0]} / {page_size}, {heads}], got "
                         f"{k_scale.dtype} {tuple(scales)} and {v_scale.dtype} {tuple(v_scale.shape)}")
    return (k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], vs[0], vs[1], k_scale.data_ptr(), v_scale.data_ptr(),
            scales[0]), heads


def _table_args(table):
    shape, stride = table.shape, table.stride()
    if table.dtype is not torch.int32 or len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"a page table is int32 [rows, pages] with contiguous rows, got {table.dtype} {tuple(shape)}")
    return table.data_ptr(), stride[0], shape[0], shape[1]


def _index(t, n: int, name: str):
    """The first n entries of an index tensor as contiguous int64."""
    shape, dtype = t.shape, t.dtype
    if dtype is torch.int64 and len(shape) == 1 and shape[0] == n and t.is_contiguous():
        return t
    if len(shape) != 1 or shape[0] < n or dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32 [{n}], got {dtype} {tuple(shape)}")
    return t[:n].to(torch.int64).contiguous()


def _rows(t, count: int, heads: int, name: str):
    """Strides of bf16 rows [count, heads, 128] (of an axis with one entry: 0, what it has there says nothing)."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1 or shape[0] != count or \
            shape[1] != heads:
        raise ValueError(f"{name} must be bfloat16 [{count}, {heads}, {HEAD_DIM}] with contiguous rows, got {t.dtype} "
                         f"{tuple(shape)}")
    if count == 1 or heads == 1:
        return stride[0] if count > 1 else 0, stride[1] if heads > 1 else 0, 1
    return stride


def _query(q, heads: int, num_modes: int, block_size: int):
    """(requests, query heads, strides) of a batch's queries."""
    shape, KL = q.shape, num_modes * block_size
    if num_modes < 1 or block_size < 1 or len(shape) != 3 or shape[0] % KL or heads < 1 or shape[1] % heads:
        raise ValueError(f"q {tuple(shape)} is not bs * {num_modes} * {block_size} rows of a multiple of {heads} heads")
    return shape[0] // KL, shape[1], _rows(q, shape[0], shape[1], "q")


def _weights_args(weights, heads: int):
    shape, stride = weights.shape, weights.stride()
    if weights.dtype is not torch.float32 or len(shape) != 3 or shape[1] != heads or (stride[2] != 1 and shape[2] > 1):
        raise ValueError(f"weights must be float32 [rows, {heads}, tokens] with contiguous rows, got {weights.dtype} "
                         f"{tuple(shape)}")
    return weights.data_ptr(), stride[0], stride[1], shape[0], shape[2]


def _device_of(*tensors) -> int:
    """The GPU of the tensors, the same for all of them."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index or index < 0:
            raise ValueError(f"MFD kernels take GPU tensors of one device (got tensors on {tensors[0].device} and "
                             f"{t.device})")
    return index


def _err(err_flag):
    if err_flag is None:
        return None
    if err_flag.dtype is not torch.int32 or err_flag.numel() < 1:
        raise ValueError(f"err_flag must be int32, got {err_flag.dtype}")
    return err_flag.data_ptr()


def _scratch(workspace, need: int, like):
    """The caller's workspace if it is given and large enough, else a new one."""
    if workspace is None:
        return like.new_empty(need, dtype=torch.uint8)
    if workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous() or workspace.data_ptr() % 16:
        raise ValueError(f"a contiguous, 16-byte aligned workspace of {need} bytes is needed")
    return workspace


# ----------------------------------------------------------------------------------------------------------- store


def kv8_store(*, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, page_table: torch.Tensor, req_pool_indices: torch.Tensor, start_lens: torch.Tensor,
              cu_tokens: torch.Tensor, max_tokens: int, page_size: int, err_flag: Optional[torch.Tensor] = None) -> None:
    """New tokens of a batch into the cache, in place. k, v [N, KV heads, 128] bf16, request b's tokens being rows
    cu_tokens[b] : cu_tokens[b + 1] (int32 [bs + 1]); they go to its positions start_lens[b], start_lens[b] + 1, ...
    ``max_tokens``: an upper bound of one request's new tokens.

    A page's scale is the smallest power of two s with amax / s <= 448. A page whose first token is stored begins anew; in a
    page begun earlier the scale only grows, and the entries before the new ones are rounded again when it does. Entries
    behind the new ones keep their bits. Infinities become +-448 s, NaN stays NaN. Two requests must not store into one
    page in the same call (nor two calls that may overlap)."""
    cache, heads = _cache_args(k_cache, v_cache, k_scale, v_scale, page_size)
    n, bs = k.shape[0], cu_tokens.numel() - 1
    ks, vs = _rows(k, n, heads, "k"), _rows(v, n, heads, "v")
    if cu_tokens.dtype is not torch.int32 or cu_tokens.dim() != 1 or bs < 0 or not cu_tokens.is_contiguous():
        raise ValueError(f"cu_tokens must be contiguous int32 [bs + 1], got {cu_tokens.dtype} {tuple(cu_tokens.shape)}")
    table = _table_args(page_table)
    rows, starts = _index(req_pool_indices, bs, "req_pool_indices"), _index(start_lens, bs, "start_lens")
    device = _device_of(k, v, k_cache, v_cache, k_scale, v_scale, page_table, req_pool_indices, start_lens, cu_tokens,
                        err_flag)
    mfd_hip.call_on(device, "mfd_kv8_store", k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], *cache,
                    *table, page_size, rows.data_ptr(), starts.data_ptr(), cu_tokens.data_ptr(), n, bs,
                    max_tokens, heads, HEAD_DIM, _err(err_flag))


# ------------------------------------------------------------------------------------------------------- attention


def _auto_count(bs: int, heads: int, rows: int, with_block: bool, max_ctx: int, device) -> tuple[int, bool]:
    """For num_ctx_splits < 0: the most splits of a request, growing with max_ctx, and whether they are parts of max_ctx. From
    what the kernels' workgroup slots hold (two workgroups per CU, one of eight waves) and the programs (request, KV head, group
    of units) that there are without a split.

    A single request's splits fill one round of slots, less the block partial's. A batch's (up to 64 requests) are measured out
    on the device (keys 0), as long as makes all of them together fill the rounds whatever the lengths: 4 requests of 700 ..
    8000 tokens, 32 heads, 8 x 16 queries, 62 us against 87 with a third of the longest each; 3 of 1024 .. 8192 45 against 60;
    equal lengths as before. Plain decoding (a program is one unit) of few requests keeps a workgroup per CU, or parts of 2048
    tokens where those are more: the device's search and one more load in the merge cost 2 us (4 requests of up to 8192 tokens
    22.7 us against 25.3; 16 56.0 against 43.7). At least 128 keys per split there and 192 else (32768 tokens, one request:
    28 us in 32 parts, 34 in 64).

    Short contexts stay whole: splits cost the block's own partial, the merge and its launch. Plain decoding up to 640 tokens
    (600: 12.9 us against 12.0 on the device, but 16.3 against 21.2 with the call's host time); else the longer the more of the
    slots the whole programs fill (8 x 16 queries, 32 heads: one request of 200 tokens 17.4 us split, 22.6 whole; 6 of 600 42.6
    and 36.7, of 1500 52.5 and 60.7; 12 of 1500 93.5 and 66.7)."""
    units = -(-rows // UNIT)
    cus = mfd_hip.cu_count(device)
    waves = 8 if units % 8 == 0 or units > 4 and 2 * bs * heads * -(-units // 8) >= cus else 4  # (as mfd_kv8_attn does)
    slots = cus * (1 if waves == 8 else 2)
    programs = max(1, bs * heads * -(-units // waves))
    if units == 1:
        short = 640
    else:
        short = 5120 * programs // slots - 1024 if 3 * programs > slots else 1536 * programs // slots
    if programs >= slots or max_ctx <= short:
        return 1, True
    least = 128 if units == 1 else 192
    if bs == 1 or bs > 64 or units == 1 and 8 * programs < slots:
        splits = slots // programs - (1 if with_block and units > 1 else 0)
        if units == 1 and bs > 1:
            splits = min(3 * slots // programs, max(cus // programs, max_ctx // 2048))
        return max(1, min(splits, -(-max_ctx // least), 32 if units == 1 else 64)), True
    # the pairs (request, partial) that mfd_kv8_attn deals out; one request's splits at most what the others leave
    extra = 1 if with_block and units > 1 else 0
    per, need = programs // bs, bs * (2 + extra)
    pairs = max(need, -(-need * per // slots) * slots // per)
    return max(1, min(pairs - extra * bs - bs + 1, -(-max_ctx // least), 32 if units == 1 else 16)), False


def _auto_splits(bs: int, heads: int, rows: int, with_block: bool, max_ctx: int, device) -> tuple[int, int]:
    """(num_ctx_splits, split_keys) for num_ctx_splits < 0; split_keys 0: measured out on the device."""
    splits, parts = _auto_count(bs, heads, rows, with_block, max_ctx, device)
    return _splits_of(splits, max_ctx) if parts and splits > 1 else (splits, 0)


def _splits_of(splits: int, max_ctx: int) -> tuple[int, int]:
    keys = -(-max(1, -(-max_ctx // splits)) // TILE_KEYS) * TILE_KEYS
    return max(1, -(-max_ctx // keys)), keys


def paged_mode_block_attention_kv8(
    *,
    q: torch.Tensor,
    k_new: Optional[torch.Tensor],
    v_new: Optional[torch.Tensor],
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    page_table: torch.Tensor,
    req_pool_indices: torch.Tensor,
    ctx_lens: torch.Tensor,
    num_modes: int,
    block_size: int,
    scaling: float,
    page_size: int,
    num_ctx_splits: int = -1,
    max_ctx: Optional[int] = None,
    causal_in_block: bool = False,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    lse_out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    err_flag: Optional[torch.Tensor] = None,
):
    """paged_mode_attention.paged_mode_block_attention over the 8-bit cache: q [T, H, 128] bf16 with T = bs * num_modes *
    block_size (mode-major per request), every query attending to its request's ctx_lens[b] cached tokens and to the
    block_size rows of k_new / v_new [T, KV heads, 128] (bf16) of its own mode.

    k_new = v_new = None: the cache alone, e.g. plain decoding with num_modes = block_size = 1 after the token was stored.
    A row that sees no key gets output 0 and lse -inf.

    Returns out [T, H, 128] bf16, and with ``return_lse`` (or ``lse_out`` given) also the natural log-sum-exp of each row's
    scaled scores, [T, H] float32.

    num_ctx_splits: > 1 splits contexts of ``max_ctx`` tokens in that many parts (a shorter context has fewer, a longer one
    a longer last part), joined by log-sum-exp; 0 or 1: one pass; < 0: by the batch's sizes. ``max_ctx`` (default: what the
    page table's rows hold) only tunes the splits. With num_ctx_splits < 0 those of 2 to 64 requests are measured
    out from the lengths on the device; those of one request, of more than 64 and of a few in plain decoding are equal parts of
    max_ctx, which should be near the longest length then (one request of 4096 tokens, 32 heads, bound 131072: 8 x 16 queries
    120 us against 29, plain decoding 42 against 19). ``workspace``: a uint8 buffer of workspace_bytes(...), for capture without
    allocation; one buffer must not serve two calls that may overlap."""
    cache, heads = _cache_args(k_cache, v_cache, k_scale, v_scale, page_size)
    bs, H, qs = _query(q, heads, num_modes, block_size)
    T = q.shape[0]
    fresh = k_new is not None
    if fresh != (v_new is not None):
        raise ValueError("k_new and v_new go together")
    if fresh:
        ks, vs = _rows(k_new, T, heads, "k_new"), _rows(v_new, T, heads, "v_new")
        new = (k_new.data_ptr(), v_new.data_ptr(), ks[0], ks[1], vs[0], vs[1])
    else:
        new = (None, None, 0, 0, 0, 0)
    table = _table_args(page_table)
    rows, lens = _index(req_pool_indices, bs, "req_pool_indices"), _index(ctx_lens, bs, "ctx_lens")
    device = _device_of(q, k_new, v_new, k_cache, v_cache, k_scale, v_scale, page_table, req_pool_indices, ctx_lens, out,
                        lse_out, workspace, err_flag)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, H, HEAD_DIM))
    os = _rows(out, T, H, "out")
    if lse_out is not None:
        if lse_out.dtype is not torch.float32 or tuple(lse_out.shape) != (T, H) or not lse_out.is_contiguous():
            raise ValueError(f"lse_out must be contiguous float32 [{T}, {H}], got {lse_out.dtype} {tuple(lse_out.shape)}")
    elif return_lse:
        lse_out = q.new_empty((T, H), dtype=torch.float32)
    if bs:
        cap = max(1, table[3] * page_size)
        max_ctx = cap if max_ctx is None else max(1, min(max_ctx, cap))
        if num_ctx_splits < 0:
            splits, keys = _auto_splits(bs, heads, H // heads * num_modes * block_size, fresh, max_ctx, q.device)
        else:
            splits, keys = _splits_of(num_ctx_splits, max_ctx) if num_ctx_splits > 1 else (1, 0)
        need = 0
        if splits > 1:
            need = mfd_hip.lib().mfd_kv8_attn_workspace_bytes(bs, num_modes, block_size, H, heads, fresh, splits)
            workspace = _scratch(workspace, need, q)
        mfd_hip.call_on(device, "mfd_kv8_attn", q.data_ptr(), qs[0], qs[1], *new, *cache, *table, page_size,
                        rows.data_ptr(), lens.data_ptr(), bs, num_modes, block_size, H, heads, HEAD_DIM, scaling,
                        1 if causal_in_block else 0, splits, keys, out.data_ptr(), os[0], os[1],
                        None if lse_out is None else lse_out.data_ptr(), workspace.data_ptr() if need else None, need,
                        _err(err_flag))
    return (out, lse_out) if lse_out is not None else out


def workspace_bytes(*, bs: int, num_modes: int, block_size: int, num_heads: int, num_kv_heads: int, with_block: bool,
                    max_ctx: int, num_ctx_splits: int = -1, device=None) -> int:
    """Bytes of paged_mode_block_attention_kv8's workspace for these sizes, enough for every call whose ``max_ctx`` (or what its
    page table's rows hold, where that is less or none is given) is at most this one. (Parts are whole tiles, so a longer context
    can have fewer of them: what counts is how many were asked for, which only grows.)"""
    max_ctx = max(1, max_ctx)
    if bs < 1:
        return 0
    if num_ctx_splits < 0:
        device = torch.device("cuda") if device is None else torch.device(device)
        splits, _ = _auto_count(bs, num_kv_heads, num_heads // num_kv_heads * num_modes * block_size, with_block, max_ctx, device)
    else:
        splits = min(num_ctx_splits, -(-max_ctx // TILE_KEYS))
    return mfd_hip.lib().mfd_kv8_attn_workspace_bytes(bs, num_modes, block_size, num_heads, num_kv_heads, with_block, splits)


def decode(cache: torch.Tensor, scale: torch.Tensor, page_size: int) -> torch.Tensor:
    """The cache's values [slots, KV heads, 128] in float32 (checks and tests)."""
    return cache.float() * scale.repeat_interleave(page_size, dim=0)[:, :, None]


# -------------------------------------------------------------------------------------------------------- eviction


def attention_weights_kv8(*, q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                          page_table: torch.Tensor, req_pool_indices: torch.Tensor, ctx_lens: torch.Tensor, num_modes: int,
                          block_size: int, scaling: float, page_size: int, weights: torch.Tensor, decay: float = 1.0,
                          err_flag: Optional[torch.Tensor] = None) -> None:
    """The attention weight that each cached token received, added to its running sum in place: for t < ctx_lens[b]

        weights[row, h, t] = decay * weights[row, h, t] + sum over KV head h's query rows of exp(scaling q.k_t - lse)

    with row = req_pool_indices[b]. q and ``lse`` [T, H] as paged_mode_block_attention_kv8 took and returned them (rows of
    lse -inf add nothing). weights: float32 [rows, KV heads, tokens], zero before a request's first call. With page tables
    that all layers share, one ``weights`` collects every layer's call: decay in the first, 1 in the others. decay 0 does not
    read the old sums. A row of ``weights`` belongs to one request of the call. Results repeat bit for bit."""
    cache, heads = _cache_args(k_cache, k_cache, k_scale, k_scale, page_size)
    bs, H, qs = _query(q, heads, num_modes, block_size)
    if lse.dtype is not torch.float32 or tuple(lse.shape) != (q.shape[0], H) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous float32 [{q.shape[0]}, {H}], got {lse.dtype} {tuple(lse.shape)}")
    table, sums = _table_args(page_table), _weights_args(weights, heads)
    rows, lens = _index(req_pool_indices, bs, "req_pool_indices"), _index(ctx_lens, bs, "ctx_lens")
    device = _device_of(q, lse, k_cache, k_scale, page_table, req_pool_indices, ctx_lens, weights, err_flag)
    mfd_hip.call_on(device, "mfd_kv8_weights", q.data_ptr(), qs[0], qs[1], lse.data_ptr(), cache[0], cache[2], cache[3],
                    cache[6], cache[8], *table, page_size, rows.data_ptr(), lens.data_ptr(), bs, num_modes, block_size, H,
                    heads, HEAD_DIM, scaling, decay, *sums, _err(err_flag))


def evict_select(*, weights: torch.Tensor, req_pool_indices: torch.Tensor, ctx_lens: torch.Tensor, budget: int,
                 sink: int = 4, recent: int = 32, keep_out: Optional[torch.Tensor] = None,
                 new_lens_out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                 err_flag: Optional[torch.Tensor] = None):
    """The tokens to keep of each request: all of one that has at most ``budget``; else its first ``sink``, its last
    ``recent``, and of the rest those whose weights, summed over the KV heads (in float64, rounded once to float32), are
    largest (ties: the lowest position; NaN below everything). Returns (keep [bs, budget] int32: positions ascending, -1
    behind them; new_lens [bs] int64). bs is ctx_lens' length."""
    bs, heads = ctx_lens.numel(), weights.shape[1] if weights.dim() == 3 else -1
    sums = _weights_args(weights, heads)
    rows, lens = _index(req_pool_indices, bs, "req_pool_indices"), _index(ctx_lens, bs, "ctx_lens")
    keep = weights.new_empty((bs, budget), dtype=torch.int32) if keep_out is None else keep_out
    new_lens = weights.new_empty(bs, dtype=torch.int64) if new_lens_out is None else new_lens_out
    if keep.dtype is not torch.int32 or tuple(keep.shape) != (bs, budget) or not keep.is_contiguous() or \
            new_lens.dtype is not torch.int64 or tuple(new_lens.shape) != (bs,) or not new_lens.is_contiguous():
        raise ValueError(f"keep_out must be contiguous int32 [{bs}, {budget}] and new_lens_out int64 [{bs}]")
    device = _device_of(weights, req_pool_indices, ctx_lens, keep_out, new_lens_out, workspace, err_flag)
    need = mfd_hip.lib().mfd_evict_select_workspace_bytes(bs, sums[4])
    workspace = _scratch(workspace, need, weights)
    mfd_hip.call_on(device, "mfd_evict_select", *sums, heads, rows.data_ptr(), lens.data_ptr(), bs, budget, sink, recent,
                    keep.data_ptr(), new_lens.data_ptr(), workspace.data_ptr() if need else None, need, _err(err_flag))
    return keep, new_lens


def evict_compact_kv8(*, keep: torch.Tensor, new_lens: torch.Tensor, ctx_lens: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, src_table: torch.Tensor,
                      dst_table: torch.Tensor, req_pool_indices: torch.Tensor, page_size: int,
                      weights: Optional[torch.Tensor] = None, err_flag: Optional[torch.Tensor] = None) -> None:
    """The kept tokens (evict_select's answer) moved, in order, from their pages in src_table to those of dst_table, rounded
    with each new page's own scale; the old pages are then free. New pages must not be among the old ones of the call's
    requests, but may be shared by nobody. Entries behind the last kept token keep their bits. ``weights``: the running sums
    move along in place, and those of positions new_lens[b] : ctx_lens[b] become 0. With several layers on the same tables,
    every layer's cache is compacted with the same ``keep`` and one call of them takes ``weights``."""
    cache, heads = _cache_args(k_cache, v_cache, k_scale, v_scale, page_size)
    bs, budget = keep.shape
    if keep.dtype is not torch.int32 or not keep.is_contiguous():
        raise ValueError(f"keep must be contiguous int32 [bs, budget], got {keep.dtype}")
    src, dst = _table_args(src_table), _table_args(dst_table)
    sums = _weights_args(weights, heads) if weights is not None else (None, 0, 0, 0, 0)
    new, lens = _index(new_lens, bs, "new_lens"), _index(ctx_lens, bs, "ctx_lens")
    rows = _index(req_pool_indices, bs, "req_pool_indices")
    device = _device_of(keep, new_lens, ctx_lens, k_cache, v_cache, k_scale, v_scale, src_table, dst_table,
                        req_pool_indices, weights, err_flag)
    mfd_hip.call_on(device, "mfd_evict_compact_kv8", keep.data_ptr(), budget, new.data_ptr(), lens.data_ptr(), *cache,
                    *src, *dst, page_size, rows.data_ptr(), *sums, bs, heads, HEAD_DIM, _err(err_flag))


# ------------------------------------------------------------------------------------------------------------ pool


class Kv8Pool:
    """The drafter's KV pool in 8 bits, in the form paged_mode_attention.PagedModeAttention takes as its ``kv_pool``
    (``get_kv_buffer(layer)``, and ``get_kv_scale(layer)`` beside it). All layers share the page tables; which pages belong
    to whom is the caller's allocator's business."""

    def __init__(self, *, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, device="cuda"):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
        self.page_size, self.num_pages = int(page_size), int(num_pages)
        slots = self.num_pages * self.page_size
        codes = lambda: torch.zeros(slots, num_kv_heads, HEAD_DIM, dtype=torch.uint8, device=device).view(CODE_DTYPE)
        scales = lambda: torch.ones(self.num_pages, num_kv_heads, dtype=torch.float32, device=device)
        self.caches = [(codes(), codes()) for _ in range(num_layers)]
        self.scales = [(scales(), scales()) for _ in range(num_layers)]

    def get_kv_buffer(self, layer_id: int):
        return self.caches[layer_id]

    def get_kv_scale(self, layer_id: int):
        return self.scales[layer_id]

    def _layer(self, layer_id: int) -> dict:
        (k, v), (ks, vs) = self.caches[layer_id], self.scales[layer_id]
        return dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, page_size=self.page_size)

    def store(self, layer_id: int, **kwargs) -> None:
        """kv8_store into a layer (its arguments without the cache's)."""
        kv8_store(**self._layer(layer_id), **kwargs)

    def attention(self, layer_id: int, **kwargs):
        """paged_mode_block_attention_kv8 over a layer (its arguments without the cache's)."""
        return paged_mode_block_attention_kv8(**self._layer(layer_id), **kwargs)

    def add_weights(self, layer_id: int, **kwargs) -> None:
        """attention_weights_kv8 of a layer (its arguments without the cache's)."""
        attention_weights_kv8(k_cache=self.caches[layer_id][0], k_scale=self.scales[layer_id][0], page_size=self.page_size,
                              **kwargs)

    def evict(self, *, weights: torch.Tensor, page_table: torch.Tensor, dst_table: torch.Tensor,
              req_pool_indices: torch.Tensor, ctx_lens: torch.Tensor, budget: int, sink: int = 4, recent: int = 32,
              err_flag: Optional[torch.Tensor] = None):
        """Cut the requests to ``budget`` tokens by ``weights``, in every layer, into the pages of dst_table; returns
        (keep, new_lens) as evict_select does."""
        keep, new_lens = evict_select(weights=weights, req_pool_indices=req_pool_indices, ctx_lens=ctx_lens, budget=budget,
                                      sink=sink, recent=recent, err_flag=err_flag)
        for layer in range(len(self.caches)):
            evict_compact_kv8(keep=keep, new_lens=new_lens, ctx_lens=ctx_lens, src_table=page_table, dst_table=dst_table,
                              req_pool_indices=req_pool_indices, weights=weights if layer == 0 else None,
                              err_flag=err_flag, **self._layer(layer))
        return keep, new_lens
