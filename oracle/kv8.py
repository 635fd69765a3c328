"""CPU oracle of the 8-bit draft KV cache. TEST INFRASTRUCTURE ONLY.

Plain float64 numpy from the definitions: a cache is kept as the values its codes stand for (float64, NaN where a code is
NaN) and its scales; pages are walked one by one. Layouts as in kv8_cache: cache [slots, Hkv, D], scale [pages, Hkv], token t
of a request in table row `row` at slot row[t // page] * page + t % page.
"""

from __future__ import annotations

import numpy as np

F64 = np.float64
MIN_EXP, MAX_EXP = -40, 40


def page_scale(amax):
    """The smallest power of two s in the cache's range with amax / s <= 448, by trying them upwards."""
    s = 2.0 ** MIN_EXP
    while s < 2.0 ** MAX_EXP and amax > 448 * s:
        s *= 2
    return s


def e4m3(x):
    """float64 values rounded to e4m3 (nearest, ties to even; beyond 448 to 448; NaN stays): three mantissa bits, the
    smallest normal 2^-6, subnormals in steps of 2^-9."""
    x = np.asarray(x, dtype=F64)
    a = np.minimum(np.abs(x), 448.0)
    with np.errstate(invalid="ignore"):
        _, e = np.frexp(np.maximum(a, 2.0 ** -6))
        step = np.ldexp(1.0, e - 4)  # a = m 2^e, m in [0.5, 1): the leading bit is 2^(e - 1)
        return np.copysign(np.rint(a / step) * step, x)


def _finite_amax(x):
    a = np.abs(x)
    return float(np.max(np.where(np.isfinite(a), a, 0.0), initial=0.0))


def store(x, cache, scale, table, rows, start_lens, cu_tokens, page):
    """x [N, Hkv, D] into (cache values, scale), in place."""
    for b in range(len(start_lens)):
        new = x[cu_tokens[b]:cu_tokens[b + 1]]
        start, end = int(start_lens[b]), int(start_lens[b]) + len(new)
        for p in range(start // page, -(-end // page)):
            pg = int(table[rows[b], p])
            lo, hi = max(start, p * page), min(end, (p + 1) * page)
            part = new[lo - start:hi - start]
            before = lo - p * page
            for h in range(x.shape[1]):
                s = page_scale(_finite_amax(part[:, h]))
                if before:
                    old = scale[pg, h]
                    s = max(s, old)
                    older = slice(pg * page, pg * page + before)
                    cache[older, h] = e4m3(cache[older, h] * old / s)
                cache[pg * page + before:pg * page + hi - p * page, h] = e4m3(part[:, h] / s)
                scale[pg, h] = s


def tokens(cache, scale, row, n, page):
    """Values [n, Hkv, D] of a request's first n tokens."""
    t = np.arange(n)
    pages = row[t // page].astype(np.int64) if n else np.zeros(0, np.int64)
    return cache[pages * page + t % page] * scale[pages][:, :, None]


def attention(q, k_new, v_new, k_ctx, v_ctx, num_modes, block_size, scaling, causal=False):
    """One request: q [KL, H, D], k_new / v_new [KL, Hkv, D] or None, k_ctx / v_ctx [n, Hkv, D]. Returns (out [KL, H, D],
    lse [KL, H], mass [KL, H, D] = sum p |v|, size [KL, H] = the largest scaling sum |q_d k_d|): the last two are what the
    rounding bounds are made of."""
    KL, H, D = q.shape
    G = H // k_ctx.shape[1]
    out, mass = np.zeros((KL, H, D)), np.zeros((KL, H, D))
    lse, size = np.full((KL, H), -np.inf), np.zeros((KL, H))
    mode = np.arange(KL) // block_size
    for h in range(H):
        k, v = k_ctx[:, h // G], v_ctx[:, h // G]
        mask = np.zeros((KL, len(k)))
        if k_new is not None:
            k, v = np.concatenate([k, k_new[:, h // G]]), np.concatenate([v, v_new[:, h // G]])
            blk = np.where(mode[:, None] != mode[None], -np.inf, 0.0)
            if causal:
                blk = np.where(np.arange(KL)[None] > np.arange(KL)[:, None], -np.inf, blk)
            mask = np.concatenate([mask, blk], axis=1)
        if not len(k):
            continue
        s = q[:, h] @ k.T * scaling + mask
        size[:, h] = (np.abs(q[:, h]) @ np.abs(k).T * scaling).max(axis=1)
        m = s.max(axis=1, keepdims=True)
        p = np.exp(s - m)
        total = p.sum(axis=1, keepdims=True)
        p = p / total
        lse[:, h] = (m + np.log(total))[:, 0]
        out[:, h] = p @ v
        mass[:, h] = p @ np.abs(v)
    return out, lse, mass, size


def weights(q, lse, k_ctx, scaling):
    """Attention weight [Hkv, n] that one request's tokens received: q [KL, H, D], lse [KL, H], k_ctx [n, Hkv, D]."""
    KL, H, _ = q.shape
    n, Hkv = k_ctx.shape[:2]
    w = np.zeros((Hkv, n))
    for h in range(H):
        seen = np.isfinite(lse[:, h])
        s = q[seen, h] @ k_ctx[:, h // (H // Hkv)].T * scaling
        w[h // (H // Hkv)] += np.exp(s - lse[seen, h][:, None]).sum(axis=0)
    return w


def select(w, n, budget, sink, recent):
    """Kept positions of one request, ascending: w [Hkv, n] float32."""
    if n <= budget:
        return list(range(n))
    score = w[:, :n].astype(F64).sum(axis=0).astype(np.float32)
    always = [t for t in range(n) if t < sink or t >= n - recent]
    rest = [t for t in range(n) if not (t < sink or t >= n - recent)]
    key = lambda t: (1, 0.0, t) if np.isnan(score[t]) else (0, -float(score[t]), t)
    return sorted(always + sorted(rest, key=key)[:budget - len(always)])


def compact(cache, scale, src_row, dst_row, kept, page):
    """Kept tokens of one request from src_row's pages into dst_row's, in place."""
    values = tokens(cache, scale, src_row, (max(kept) + 1) if kept else 0, page)[kept]
    for p in range(0, len(kept), page):
        pg = int(dst_row[p // page])
        part = values[p:p + page]
        for h in range(cache.shape[1]):
            s = page_scale(_finite_amax(part[:, h]))
            cache[pg * page:pg * page + len(part), h] = e4m3(part[:, h] / s)
            scale[pg, h] = s
