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


def _cache_args(cache, scale, name: str, page_size: int):
    """(pointer, slot stride, head stride, scale pointer) of one side of the cache."""
    if cache.dtype != CODE_DTYPE or cache.dim() != 3 or cache.shape[2] != HEAD_DIM or cache.stride(2) != 1:
        raise ValueError(f"{name}_cache must be {CODE_DTYPE} [slots, KV heads, {HEAD_DIM}] with contiguous rows, got "
                         f"{cache.dtype} {tuple(cache.shape)}")
    pages, heads = scale.shape
    if scale.dtype != torch.float32 or not scale.is_contiguous() or heads != cache.shape[1] or \
            pages * page_size != cache.shape[0]:
        raise ValueError(f"{name}_scale must be contiguous float32 [{cache.shape[0]} / {page_size}, {cache.shape[1]}], got "
                         f"{scale.dtype} {tuple(scale.shape)}")
    return cache.data_ptr(), cache.stride(0), cache.stride(1), scale.data_ptr()


def _check_page_size(page_size: int) -> None:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")


def _table_args(table):
    if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"a page table is int32 [rows, pages] with contiguous rows, got {table.dtype} "
                         f"{tuple(table.shape)}")
    return table.data_ptr(), table.stride(0), table.shape[0], table.shape[1]


def _index(t, n: int, name: str):
    """The first n entries of an index tensor as contiguous int64."""
    if t.dim() != 1 or t.numel() < n or t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    t = t[:n] if t.numel() != n else t
    t = t if t.dtype == torch.int64 else t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def _rows3(t, heads: Optional[int], name: str, dtype=torch.bfloat16):
    if t.dtype != dtype or t.dim() != 3 or t.shape[2] != HEAD_DIM or t.stride(2) != 1 or \
            (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be {dtype} [rows, heads, {HEAD_DIM}] with contiguous rows, got {t.dtype} "
                         f"{tuple(t.shape)}")


def _weights_args(weights, heads: int):
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[1] != heads or \
            (weights.shape[2] > 1 and weights.stride(2) != 1):
        raise ValueError(f"weights must be float32 [rows, {heads}, tokens] with contiguous rows, got {weights.dtype} "
                         f"{tuple(weights.shape)}")
    return weights.data_ptr(), weights.stride(0), weights.stride(1), weights.shape[0], weights.shape[2]


def _same_device(*tensors):
    """The tensors' GPU, the same for all of them."""
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"MFD kernels take GPU tensors (got a tensor on {device})")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}")
    return device


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
    page in the same call."""
    _check_page_size(page_size)
    heads = k_cache.shape[1]
    _rows3(k, heads, "k")
    _rows3(v, heads, "v")
    if v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    bs = cu_tokens.numel() - 1
    if cu_tokens.dtype != torch.int32 or cu_tokens.dim() != 1 or bs < 0 or not cu_tokens.is_contiguous():
        raise ValueError(f"cu_tokens must be contiguous int32 [bs + 1], got {cu_tokens.dtype} {tuple(cu_tokens.shape)}")
    device = _same_device(k, v, k_cache, v_cache, k_scale, v_scale, page_table, req_pool_indices, start_lens, cu_tokens,
                          err_flag)
    kp, kss, ksh, ksp = _cache_args(k_cache, k_scale, "k", page_size)
    vp, vss, vsh, vsp = _cache_args(v_cache, v_scale, "v", page_size)
    if k_scale.shape != v_scale.shape:
        raise ValueError("the K and V caches have different sizes")
    rows, starts = _index(req_pool_indices, bs, "req_pool_indices"), _index(start_lens, bs, "start_lens")
    mfd_hip.call_on(device, "mfd_kv8_store", k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), kp, vp,
          kss, ksh, vss, vsh, ksp, vsp, k_scale.shape[0], *_table_args(page_table), page_size, rows.data_ptr(),
          starts.data_ptr(), cu_tokens.data_ptr(), k.shape[0], bs, int(max_tokens), heads, HEAD_DIM,
          mfd_hip.ptr(err_flag))


# ------------------------------------------------------------------------------------------------------- attention


def _auto_splits(bs: int, heads: int, rows: int, with_block: bool, max_ctx: int, device) -> tuple[int, int]:
    """(num_ctx_splits, split_keys) for num_ctx_splits < 0: enough parts of the longest context for two rounds of workgroup
    slots if all were as long (contexts of a batch differ, and short workgroups behind long ones even that out), of at least
    256 keys each."""
    units = -(-rows // UNIT)
    waves = 8 if units % 8 == 0 else 4
    slots = mfd_hip.cu_count(device) * (1 if units > 1 and waves == 8 else 2)
    programs = max(1, bs * heads * -(-units // waves))
    want = slots * (1 if bs == 1 else 2)
    splits = want // programs if bs == 1 else -(-want // programs)
    if bs == 1 and with_block and units > 1:
        splits -= 1
    splits = min(splits, -(-max_ctx // 256), 64)
    if splits <= 1:
        return 1, 0
    return _splits_of(splits, max_ctx)


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
    page table's rows hold) only tunes the splits. ``workspace``: a uint8 buffer of workspace_bytes(...), for capture
    without allocation; one buffer must not serve two calls that may overlap."""
    _check_page_size(page_size)
    T, H, _ = q.shape
    heads = k_cache.shape[1]
    KL = num_modes * block_size
    if num_modes < 1 or block_size < 1 or T % KL or H % heads:
        raise ValueError(f"q {tuple(q.shape)} is not bs * {num_modes} * {block_size} rows of a multiple of {heads} heads")
    _rows3(q, None, "q")
    bs = T // KL
    fresh = k_new is not None
    if fresh != (v_new is not None):
        raise ValueError("k_new and v_new go together")
    if fresh:
        _rows3(k_new, heads, "k_new")
        _rows3(v_new, heads, "v_new")
        if k_new.shape[0] != T or v_new.shape[0] != T:
            raise ValueError(f"k_new and v_new must have q's {T} rows")
        fresh_args = (k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_new.stride(1), v_new.stride(0),
                      v_new.stride(1))
    else:
        fresh_args = (None, None, 0, 0, 0, 0)
    device = _same_device(q, k_new, v_new, k_cache, v_cache, k_scale, v_scale, page_table, req_pool_indices, ctx_lens, out,
                          lse_out, workspace, err_flag)
    kp, kss, ksh, ksp = _cache_args(k_cache, k_scale, "k", page_size)
    vp, vss, vsh, vsp = _cache_args(v_cache, v_scale, "v", page_size)
    if k_scale.shape != v_scale.shape:
        raise ValueError("the K and V caches have different sizes")
    if out is None:
        out = torch.empty((T, H, HEAD_DIM), device=device, dtype=torch.bfloat16)
    else:
        _rows3(out, H, "out")
        if out.shape[0] != T:
            raise ValueError(f"out must have q's {T} rows")
    if lse_out is None and return_lse:
        lse_out = torch.empty((T, H), device=device, dtype=torch.float32)
    elif lse_out is not None and (lse_out.dtype != torch.float32 or tuple(lse_out.shape) != (T, H) or
                                  not lse_out.is_contiguous()):
        raise ValueError(f"lse_out must be contiguous float32 [{T}, {H}]")
    if bs:
        cap = page_table.shape[1] * page_size
        max_ctx = cap if max_ctx is None else max(1, min(int(max_ctx), cap))
        if num_ctx_splits < 0:
            splits, keys = _auto_splits(bs, heads, H // heads * KL, fresh, max_ctx, device)
        else:
            splits, keys = _splits_of(num_ctx_splits, max_ctx) if num_ctx_splits > 1 else (1, 0)
        need = 0
        if splits > 1:
            need = mfd_hip.lib().mfd_kv8_attn_workspace_bytes(bs, num_modes, block_size, H, heads, fresh, splits)
            if workspace is None:
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
            elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
                raise ValueError(f"a contiguous workspace of {need} bytes is needed")
        rows, lens = _index(req_pool_indices, bs, "req_pool_indices"), _index(ctx_lens, bs, "ctx_lens")
        mfd_hip.call_on(device, "mfd_kv8_attn", q.data_ptr(), q.stride(0), q.stride(1), *fresh_args, kp, vp, kss, ksh, vss, vsh,
              ksp, vsp, k_scale.shape[0], *_table_args(page_table), page_size, rows.data_ptr(), lens.data_ptr(), bs,
              num_modes, block_size, H, heads, HEAD_DIM, float(scaling), 1 if causal_in_block else 0, splits, keys,
              out.data_ptr(), out.stride(0), out.stride(1), mfd_hip.ptr(lse_out), workspace.data_ptr() if need else None,
              need, mfd_hip.ptr(err_flag))
    return (out, lse_out) if lse_out is not None else out


def workspace_bytes(*, bs: int, num_modes: int, block_size: int, num_heads: int, num_kv_heads: int, with_block: bool,
                    max_ctx: int, num_ctx_splits: int = -1, device=None) -> int:
    """Bytes of paged_mode_block_attention_kv8's workspace for these sizes (its ``max_ctx`` the same)."""
    if num_ctx_splits < 0:
        device = torch.device("cuda") if device is None else torch.device(device)
        splits, _ = _auto_splits(bs, num_kv_heads, num_heads // num_kv_heads * num_modes * block_size, with_block,
                                 max(1, max_ctx), device)
    else:
        splits = _splits_of(num_ctx_splits, max(1, max_ctx))[0] if num_ctx_splits > 1 else 1
    return mfd_hip.lib().mfd_kv8_attn_workspace_bytes(bs, num_modes, block_size, num_heads, num_kv_heads, with_block,
                                                      splits)


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
    read the old sums. Results repeat bit for bit."""
    _check_page_size(page_size)
    T, H, _ = q.shape
    heads = k_cache.shape[1]
    KL = num_modes * block_size
    if num_modes < 1 or block_size < 1 or T % KL or H % heads:
        raise ValueError(f"q {tuple(q.shape)} is not bs * {num_modes} * {block_size} rows of a multiple of {heads} heads")
    _rows3(q, None, "q")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (T, H) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous float32 [{T}, {H}], got {lse.dtype} {tuple(lse.shape)}")
    bs = T // KL
    device = _same_device(q, lse, k_cache, k_scale, page_table, req_pool_indices, ctx_lens, weights, err_flag)
    kp, kss, ksh, ksp = _cache_args(k_cache, k_scale, "k", page_size)
    rows, lens = _index(req_pool_indices, bs, "req_pool_indices"), _index(ctx_lens, bs, "ctx_lens")
    mfd_hip.call_on(device, "mfd_kv8_weights", q.data_ptr(), q.stride(0), q.stride(1), lse.data_ptr(), kp, kss, ksh, ksp,
          k_scale.shape[0], *_table_args(page_table), page_size, rows.data_ptr(), lens.data_ptr(), bs, num_modes,
          block_size, H, heads, HEAD_DIM, float(scaling), float(decay), *_weights_args(weights, heads),
          mfd_hip.ptr(err_flag))


def evict_select(*, weights: torch.Tensor, req_pool_indices: torch.Tensor, ctx_lens: torch.Tensor, budget: int,
                 sink: int = 4, recent: int = 32, keep_out: Optional[torch.Tensor] = None,
                 new_lens_out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                 err_flag: Optional[torch.Tensor] = None):
    """The tokens to keep of each request: all of one that has at most ``budget``; else its first ``sink``, its last
    ``recent``, and of the rest those whose weights, summed over the KV heads (in float64, rounded once to float32), are
    largest (ties: the lowest position; NaN below everything). Returns (keep [bs, budget] int32: positions ascending, -1
    behind them; new_lens [bs] int64). bs is ctx_lens' length."""
    bs = ctx_lens.numel()
    heads = weights.shape[1]
    device = _same_device(weights, req_pool_indices, ctx_lens, keep_out, new_lens_out, workspace, err_flag)
    wargs = _weights_args(weights, heads)
    keep = torch.empty((bs, budget), dtype=torch.int32, device=device) if keep_out is None else keep_out
    new_lens = torch.empty(bs, dtype=torch.int64, device=device) if new_lens_out is None else new_lens_out
    if keep.dtype != torch.int32 or tuple(keep.shape) != (bs, budget) or not keep.is_contiguous() or \
            new_lens.dtype != torch.int64 or tuple(new_lens.shape) != (bs,) or not new_lens.is_contiguous():
        raise ValueError(f"keep_out must be contiguous int32 [{bs}, {budget}] and new_lens_out int64 [{bs}]")
    need = mfd_hip.lib().mfd_evict_select_workspace_bytes(bs, weights.shape[2])
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
        raise ValueError(f"a contiguous workspace of {need} bytes is needed")
    rows, lens = _index(req_pool_indices, bs, "req_pool_indices"), _index(ctx_lens, bs, "ctx_lens")
    mfd_hip.call_on(device, "mfd_evict_select", *wargs, heads, rows.data_ptr(), lens.data_ptr(), bs, int(budget), int(sink),
          int(recent), keep.data_ptr(), new_lens.data_ptr(), workspace.data_ptr() if need else None, need,
          mfd_hip.ptr(err_flag))
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
    _check_page_size(page_size)
    bs, budget = keep.shape
    heads = k_cache.shape[1]
    if keep.dtype != torch.int32 or not keep.is_contiguous():
        raise ValueError(f"keep must be contiguous int32 [bs, budget], got {keep.dtype}")
    device = _same_device(keep, new_lens, ctx_lens, k_cache, v_cache, k_scale, v_scale, src_table, dst_table,
                          req_pool_indices, weights, err_flag)
    kp, kss, ksh, ksp = _cache_args(k_cache, k_scale, "k", page_size)
    vp, vss, vsh, vsp = _cache_args(v_cache, v_scale, "v", page_size)
    if k_scale.shape != v_scale.shape:
        raise ValueError("the K and V caches have different sizes")
    wargs = _weights_args(weights, heads) if weights is not None else (None, 0, 0, 0, 0)
    new, lens = _index(new_lens, bs, "new_lens"), _index(ctx_lens, bs, "ctx_lens")
    rows = _index(req_pool_indices, bs, "req_pool_indices")
    mfd_hip.call_on(device, "mfd_evict_compact_kv8", keep.data_ptr(), budget, new.data_ptr(), lens.data_ptr(), kp, vp, kss, ksh, vss,
          vsh, ksp, vsp, k_scale.shape[0], *_table_args(src_table), *_table_args(dst_table), page_size, rows.data_ptr(),
          *wargs, bs, heads, HEAD_DIM, mfd_hip.ptr(err_flag))


# ------------------------------------------------------------------------------------------------------------ pool


class Kv8Pool:
    """The drafter's KV pool in 8 bits, in the form paged_mode_attention.PagedModeAttention takes as its ``kv_pool``
    (``get_kv_buffer(layer)``, and ``get_kv_scale(layer)`` beside it). All layers share the page tables; which pages belong
    to whom is the caller's allocator's business."""

    def __init__(self, *, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, device="cuda"):
        _check_page_size(page_size)
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
