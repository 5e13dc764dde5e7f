"""64-bit oracle of the bounded cache's operators: rotary forms, attention that scores
its cache, eviction, and drawing tokens from given random numbers. Plain loops and
definitions; checks only."""

from __future__ import annotations

import numpy as np


def rotary(x, positions, inv_freq, interleaved=False, scale=1.0):
    """x [B, T, heads, D], positions [B, T] or [T]: (turned x, bound on fp32 arithmetic's
    error: cos / sin, products and sums rounded to fp32, three half steps of 2^-24 of
    |x1| + |x2|, and the like once more for a rounded `scale`)."""
    x = np.asarray(x, np.float64)
    B, T, _, _ = x.shape
    p = np.broadcast_to(np.asarray(positions, np.float64), (B, T))
    a = p[:, :, None, None] * np.asarray(inv_freq, np.float64)
    P = a.shape[-1]
    one = np.arange(0, 2 * P, 2) if interleaved else np.arange(P)
    two = one + (1 if interleaved else P)
    y, bound = x.copy(), np.zeros_like(x)
    c, s = scale * np.cos(a), scale * np.sin(a)
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    bound[..., one] = bound[..., two] = 4 * 2.0 ** -24 * abs(scale) * (abs(x[..., one]) + abs(x[..., two]))
    return y, bound


def attention_scored(q, k_codes, k_scales, v_codes, v_scales, lengths, scale=None):
    """q [B, Tq, H, D] over caches [B, KVH, T_cap, ...]; row t sees the first
    lengths[b] - Tq + t + 1 slots. Returns (out, added scores [B, KVH, T_cap], bound of
    out, bound of the scores): a base-2 score is a fp32 sum of D products (error D 2^-24
    of the sum of their sizes), scaled and rounded a few times; its weight is off by that
    much times ln 2 relative, twice (numerator and sum); sums over n slots add n 2^-24,
    exp2, its argument's rounding and the division under 2^-20."""
    q = np.asarray(q, np.float64)
    B, Tq, H, D = q.shape
    KVH, cap = k_codes.shape[1:3]
    G = H // KVH
    scale = D ** -0.5 if scale is None else scale
    out, ob = np.zeros(q.shape), np.zeros(q.shape)
    add, ab = np.zeros((B, KVH, cap)), np.zeros((B, KVH, cap))
    for b in range(B):
        for t in range(Tq):
            n = min(int(lengths[b]), cap) - Tq + t + 1
            if n <= 0:
                continue
            for h in range(H):
                kv = h // G
                K = k_codes[b, kv, :n].astype(np.float64) * np.asarray(k_scales[b, kv, :n], np.float64)[:, None]
                V = v_codes[b, kv, :n].astype(np.float64) * np.asarray(v_scales[b, kv, :n], np.float64)[:, None]
                s = K @ q[b, t, h] * scale
                size = abs(K) @ abs(q[b, t, h]) * abs(scale)
                w = np.exp(s - s.max())
                w /= w.sum()
                rel = 2 * (D + 8) * 2.0 ** -24 * size.max() + (n + 64) * 2.0 ** -24 + 2.0 ** -20
                out[b, t, h] = w @ V
                ob[b, t, h] = rel * (w @ abs(V))
                add[b, kv, :n] += w
                ab[b, kv, :n] += rel * w
    return out, add, ob, ab


def evict(arrays, scores, positions, lengths, seen, budget, recent):
    """Cut each (sequence, head) of `arrays` (each [B, KVH, T_cap, ...], scores and
    positions among them) to `budget` slots: slots of the newest tokens by their index,
    then the others by score; returns (new arrays, new lengths)."""
    arrays = [a.copy() for a in arrays]
    out = []
    for b in range(scores.shape[0]):
        n = int(lengths[b])
        out.append(min(n, budget))
        if n <= budget:
            continue
        for h in range(scores.shape[1]):
            sc = scores[b, h, :n].astype(np.float64)
            sc[np.isnan(sc)] = -np.inf
            new = positions[b, h, :n].astype(np.int64) >= int(seen[b]) - recent
            order = sorted(range(n), key=lambda i: (not new[i], 0.0 if new[i] else -sc[i], i))
            kept = np.zeros(n, bool)
            kept[order[:budget]] = True
            holes = [i for i in range(budget) if not kept[i]]
            donors = [i for i in range(budget, n) if kept[i]]
            assert len(holes) == len(donors)
            for a in arrays:
                a[b, h, holes] = a[b, h, donors]
    return arrays, np.asarray(out, np.int32)


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability, its neighbours in the order where u lies within the
    weights' rounding of a border) of one row of logits."""
    x = np.asarray(row, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if x.size == 0 or x.max() == -np.inf:
        return -1, -np.inf, ()
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 0.0, ()
    x = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / temperature))
    w[x == -np.inf] = 0.0
    n = x.size
    if 0 < top_k < n:
        n = int((x >= x[top_k - 1]).sum())
    w = w[:n]
    if top_p < 1:
        n = int((np.cumsum(w) - w <= top_p * w.sum() * (1 + 1e-15)).sum()) if top_p > 0 else 1
        w = w[:max(n, 1)]
    w = w[:max(int((w >= min_p).sum()), 1)]
    run = np.cumsum(w)
    target = min(max(u, 0.0), 1.0) * run[-1]
    at = min(int(np.searchsorted(run, target, side="right")), int(np.nonzero(w)[0][-1]))
    slack = x.size * 2.0 ** -40
    near = [order[i] for i in (at - 1, at + 1) if 0 <= i < w.size and
            min(abs(run[at] - target), abs(run[at] - w[at] - target)) < slack and 0 < target < run[-1]]
    return int(order[at]), float(np.log(w[at] / run[-1])), tuple(int(i) for i in near)
