"""Float64 oracle for the smaller KV cache: MXFP4 rows, decode with attention
weights, a prompt's weights, eviction (test infrastructure, never product code).

None of these has a counterpart in the reference; each is written from its
definition and pinned in tests/test_small_cache_cpu.py by brute force.
"""
from __future__ import annotations

import numpy as np

#: What the eight magnitudes of a 4-bit code stand for.
FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_encode(x):
    """Codes [..., D/2] and scales [..., D/32] (uint8) of rows [..., D]."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, 0.0)
    top = np.abs(g).max(-1)
    m, e = np.frexp(top)  # top = m 2^e, 1/2 <= m < 1
    e = np.where(top > 0, e - 1 + (m >= 0.875) - 2, -126)
    scale = np.clip(e + 127, 1, 254)
    y = np.abs(np.ldexp(g, (127 - scale)[..., None]))
    # nearest, ties to the even code: the code steps up past each midpoint, or at
    # it where the code below is odd
    middle = (FP4[:-1] + FP4[1:]) / 2
    code = sum(((y > c) | ((y == c) & (i % 2 == 1))).astype(np.uint8) for i, c in enumerate(middle))
    code = code | (np.signbit(g).astype(np.uint8) << 3)
    code = np.where(finite[..., None], code, 0).astype(np.uint8).reshape(x.shape)
    scale = np.where(finite, scale, 255).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def mxfp4_decode(codes, scales):
    """The values, in float64, that codes [..., D/2] and scales [..., D/32] stand for."""
    code = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)
    value = np.where(code >= 8, -1.0, 1.0) * FP4[code % 8]
    factor = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return value * np.repeat(factor, 32, axis=-1)


def rows_of(cache, table, n, head, num_blocks=None):
    """Rows [n, ...] of one head along a block table, and which of them are on a page of the pool."""
    bs = cache.shape[2]
    pages = np.asarray(table)[np.arange(n) // bs]
    fine = (pages >= 0) & (pages < cache.shape[0])
    return cache[np.where(fine, pages, 0), head, np.arange(n) % bs], fine


def decode(q, k, v, tables, lens, scale):
    """q [B, H, D] over caches of values [blocks, Hkv, bs, D] in float64: the output, each token's weight summed
    over its kv head's query heads (a list of [Hkv, n]), and what the tolerances need: per output element the
    weighted sum of |v|, and per sequence and query head sum |q||k| scale at its largest."""
    B, H, D = q.shape
    hkv = k.shape[1]
    group = H // hkv
    out, spread = np.zeros((B, H, D)), np.zeros((B, H, D))
    weights, reach = [], np.zeros((B, H))
    for b in range(B):
        n = max(int(lens[b]), 0)
        w = np.zeros((hkv, n))
        for h in range(H if n else 0):
            kk, fine = rows_of(k, tables[b], n, h // group)
            vv, _ = rows_of(v, tables[b], n, h // group)
            if not fine.any():
                continue
            s = np.full(n, -np.inf)
            with np.errstate(invalid="ignore"):
                s[fine] = kk[fine] @ q[b, h] * scale
            if np.all(s == -np.inf):
                continue
            p = np.exp(s - s.max())
            p /= p.sum()
            with np.errstate(invalid="ignore"):
                out[b, h] = p[fine] @ vv[fine]
                spread[b, h] = p[fine] @ np.abs(vv[fine])
                reach[b, h] = np.nanmax(np.where(np.isfinite(kk[fine]), np.abs(kk[fine]), 0) @ np.abs(q[b, h])) * \
                    abs(scale)
            w[h // group] += np.where(fine, p, 0.0)
        weights.append(w)
    return out, weights, spread, reach


def prompt(q, k, cu, length, last=None, scale=None):
    """Weights [B, Hkv, length] of packed prompts q [T, H, D], k [T, Hkv, D], and the largest sum |q||k| scale."""
    H, D = q.shape[1:]
    hkv = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, reach = np.zeros((len(cu) - 1, hkv, length)), 0.0
    for b in range(len(cu) - 1):
        q1, k1 = q[cu[b]:cu[b + 1]], k[cu[b]:cu[b + 1]]
        n = len(q1)
        first = max(0, n - (n if last is None else last))
        for h in range(H if n else 0):
            s = q1[first:, h] @ k1[:, h // (H // hkv)].T * scale
            size = np.abs(np.where(np.isfinite(k1), k1, 0)[:, h // (H // hkv)])
            reach = max(reach, float((np.abs(q1[first:, h]) @ size.T).max() * abs(scale)))
            s[np.arange(n)[None, :] > np.arange(first, n)[:, None]] = -np.inf
            p = np.exp(s - s.max(-1, keepdims=True))
            out[b, h // (H // hkv), :n] += (p / p.sum(-1, keepdims=True)).sum(0)
    return out, reach


def keep(weights, budget, recent):
    """Positions that one head keeps of n tokens of these weights, ascending."""
    n = len(weights)
    if n <= budget:
        return np.arange(n)
    old = sorted(range(n - recent), key=lambda i: (0 if np.isnan(weights[i]) else 1,
                                                   0.0 if np.isnan(weights[i]) else -float(weights[i]), i))
    return np.array(sorted(old[:budget - recent]) + list(range(n - recent, n)), dtype=np.int64)


def evict(caches, tables, lens, weights, budget, recent, new_tables=None):
    """caches: a list of [blocks, Hkv, bs, ...] arrays; returns new lengths, weights, kept and new caches."""
    B, hkv, length = weights.shape
    bs = caches[0].shape[2]
    capacity = min(length, tables.shape[1] * bs)
    after = [c.copy() for c in caches]
    kept = np.full((B, hkv, budget), -1, dtype=np.int32)
    new_weights = np.zeros_like(weights)
    new = np.array([min(max(min(int(n), capacity), 0), budget) for n in lens], dtype=np.int32)
    to = tables if new_tables is None else new_tables
    for b in range(B):
        n = max(min(int(lens[b]), capacity), 0)
        for h in range(hkv):
            rows = keep(weights[b, h, :n], budget, recent)
            kept[b, h, :len(rows)] = rows
            new_weights[b, h, :len(rows)] = weights[b, h, rows]
            for i, r in enumerate(rows):
                src, dst = tables[b, r // bs], to[b, i // bs]
                if 0 <= src < len(caches[0]) and 0 <= dst < len(caches[0]):
                    for c, x in zip(caches, after):
                        x[dst, h, i % bs] = c[src, h, r % bs]
    return new, new_weights, kept, after
