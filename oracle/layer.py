"""Plain 64-bit forms of the decoder-layer operators (numpy, no GPU) -- TEST INFRASTRUCTURE ONLY, like the rest of this
package.  Written from the definitions in include/tornado_b200.h, one loop per sentence of them."""
from __future__ import annotations

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}


def nearest(x, mantissa, lowest):
    """x rounded to `mantissa` bits behind the leading one, steps of 2**lowest at least, ties to even."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 1 - mantissa, lowest).astype(np.float64))
    return np.round(x / step) * step


def round_fp8(x, fmt):
    """Saturating conversion to the fp8 format's values."""
    x = np.clip(x, -TOP[fmt], TOP[fmt])
    return nearest(x, 3, -9) if fmt == "e4m3" else nearest(x, 2, -16)


def rmsnorm_quant(x, residual, weight, eps, fmt, group):
    """(y / scale before rounding, scales, h) in float64; x [rows][cols], residual like x or None."""
    h = x.astype(np.float64) + (0.0 if residual is None else residual.astype(np.float64))
    rows, cols = h.shape
    with np.errstate(all="ignore"):
        y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * weight.astype(np.float64)
    g = group or cols
    n = -(-cols // g)
    ratio, scales = np.zeros_like(y), np.zeros((rows, n))
    for b in range(n):
        part = y[:, b * g:(b + 1) * g]
        top = np.abs(part).max(1)
        scale = np.where(top == 0, 1.0, top / TOP[fmt])
        scale = np.where(np.isfinite(top), np.maximum(scale, 2.0 ** -126), top)
        scales[:, b] = scale
        with np.errstate(all="ignore"):
            ratio[:, b * g:(b + 1) * g] = np.where(np.isfinite(top)[:, None], part / scale[:, None], 0.0)
    return ratio, scales, h


def paged_plan(cached, new, page, width, max_tokens, free, table):
    """The step's layout, request by request and token by token."""
    requests = len(cached)
    table = np.array(table, np.int32).reshape(requests, width).copy()
    positions, slots = np.full(max_tokens, -1, np.int32), np.full(max_tokens, -1, np.int64)
    cu, kv = np.zeros(requests + 1, np.int32), np.zeros(requests, np.int32)
    used = asked = needed = 0
    for r in range(requests):
        c, n = max(0, int(cached[r])), max(0, int(new[r]))
        asked += n
        n = min(n, max(0, width * page - c), max_tokens - used)
        kv[r] = c + n
        if n:
            for i in range(-(-c // page), -(-(c + n) // page)):
                table[r, i] = free[needed] if needed < len(free) else -1
                needed += 1
        for i in range(n):
            p = c + i
            positions[used + i] = p
            entry = int(table[r, p // page])
            slots[used + i] = entry * page + p % page if entry >= 0 else -1
        used += n
        cu[r + 1] = used
    counts = np.array([used, min(asked, 2 ** 31 - 1), min(needed, len(free)), needed], np.int32)
    return table, cu, kv, positions, slots, counts


def rope(x, cos, sin, positions, interleaved):
    """x [tokens][heads][dim] float64 turned by its positions' angles; cos, sin [rows][rot / 2]."""
    out, half = x.astype(np.float64).copy(), cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos.astype(np.float64)[positions, i][:, None], sin.astype(np.float64)[positions, i][:, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def rope_append(q, k, v, cos, sin, positions, interleaved, slots, q_out, k_cache, v_cache):
    """Arrays as float64; q, k, v [tokens][heads][dim], caches [pages][heads][page][dim]; returns what the outputs hold."""
    q_out, k_cache, v_cache = q_out.copy(), k_cache.copy(), v_cache.copy()
    pages, _, page, _ = k_cache.shape
    rows = [t for t in range(len(positions)) if positions[t] >= 0 and (positions[t] < len(cos) or cos.shape[1] == 0)]
    at = positions[rows]
    if q.shape[1]:
        q_out[rows] = rope(q[rows], cos, sin, at, interleaved)
    turned = rope(k[rows], cos, sin, at, interleaved)
    for n, t in enumerate(rows):
        if 0 <= slots[t] < pages * page:
            k_cache[slots[t] // page, :, slots[t] % page] = turned[n]
            v_cache[slots[t] // page, :, slots[t] % page] = v[t]
    return q_out, k_cache, v_cache


def paged_attention(q, cu, kv_lens, table, k_cache, v_cache, scale, window, out):
    """q, out [tokens][heads][dim] float64, caches [pages][kv heads][page][dim]; rows that no request has stay."""
    out = out.copy()
    tokens, heads, _ = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    group, width = heads // kv_heads, table.shape[1]
    for r in range(len(kv_lens)):
        b = min(max(int(cu[r]), 0), tokens)
        e = min(max(int(cu[r + 1]), b), tokens)
        for t in range(b, e):
            p = int(kv_lens[r]) - (e - b) + (t - b)
            keys = np.arange(max(0, p - window + 1) if window else 0, min(p + 1, width * page))
            entries = table[r, keys // page]
            ok = (entries >= 0) & (entries < pages)
            keys, entries = keys[ok], entries[ok]
            for h in range(heads):
                k, v = k_cache[entries, h // group, keys % page], v_cache[entries, h // group, keys % page]
                with np.errstate(all="ignore"):
                    s = (k @ q[t, h]) * scale
                    if not len(s) or s.max() == -np.inf:
                        out[t, h] = 0
                        continue
                    w = np.exp(s - s.max())
                    out[t, h] = (w / w.sum()) @ v
    return out
