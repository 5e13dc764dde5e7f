"""64-bit oracle of the 4-bit cache's operators and of normed, turned heads: plain formulas
with bounds on what the kernels' fp32 steps may lose; checks only."""

from __future__ import annotations

import numpy as np

from . import bounded

U = 2.0 ** -24


def inv_rms(x, eps):
    """1 / sqrt(mean(x^2) + eps) over the last dim, and the relative error of it in fp32: the
    sum of D squares loses D + 8 half steps at most, the root halves that, mean, sum, root
    and quotient round once each."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    return 1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / D + eps), ((D + 8) / 2 + 4) * U


def qk_norm_rotary(x, w, positions, inv_freq, eps=1e-6, interleaved=False, scale=1.0):
    """x [B, T, heads, D]: (normed and turned, bound on fp32 arithmetic's error): two more
    roundings for x r w, and the turn's own."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    r, rel = inv_rms(x, eps)
    n = x * r * w
    y, b = bounded.rotary(n, positions, inv_freq, interleaved, scale)
    lost, _ = turn_sizes(abs(n) * (rel + 2 * U), inv_freq, interleaved, scale)
    return y, b * (1 + rel) + lost


def turn_sizes(e, inv_freq, interleaved, scale):
    """What errors e of the dims of a head come to once it turns: both of a pair's, scaled."""
    P = len(inv_freq)
    one = np.arange(0, 2 * P, 2) if interleaved else np.arange(P)
    two = one + (1 if interleaved else P)
    out = e.copy()
    out[..., one] = out[..., two] = abs(scale) * (e[..., one] + e[..., two])
    return out, one


def qk_norm_rotary_backward(x, w, gy, positions, inv_freq, eps=1e-6, interleaved=False, scale=1.0):
    """(dx, dw, bound of dx, bound of dw) for the output's gradient gy."""
    x, w, gy = (np.asarray(t, np.float64) for t in (x, w, gy))
    D = x.shape[-1]
    r, rel = inv_rms(x, eps)
    n = x * r
    g, eg = bounded.rotary(gy, -np.asarray(positions, np.int64), inv_freq, interleaved, scale)
    gw = g * w
    dot = (gw * n).mean(-1, keepdims=True)
    dx = r * (gw - n * dot)
    egw = eg * abs(w) + U * abs(gw)
    # the sum of D products: D + 8 half steps of their sizes, and what its terms are off
    edot = ((egw * abs(n) + abs(gw * n) * (rel + U)).mean(-1, keepdims=True)
            + (D + 10) * U * abs(gw * n).mean(-1, keepdims=True))
    edx = r * (egw + abs(n) * edot + abs(n * dot) * (rel + 2 * U)) + r * (abs(gw) + abs(n * dot)) * (rel + 3 * U)
    axes = tuple(range(x.ndim - 1))
    terms = np.prod([x.shape[a] for a in axes])
    dw = (g * n).sum(axes)
    edw = (eg * abs(n) + abs(g * n) * (rel + 2 * U)).sum(axes) + (terms + 16) * U * abs(g * n).sum(axes)
    return dx, dw, edx, edw


def quantize(x, group):
    """x [..., D] in 64 bits: (codes [..., D] int, s and m [..., D / group] as the fp16 that is
    held, and each code's distance from the nearest border, in steps)."""
    x = np.asarray(x, np.float64)
    y = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    lo, hi = y.min(-1), y.max(-1)
    with np.errstate(invalid="ignore", over="ignore"):
        m = np.clip(lo.astype(np.float32), -65504, 65504).astype(np.float16)
        s = np.minimum(((hi - lo) / 15).astype(np.float32), np.float32(65504)).astype(np.float16)
        step = np.where(s > 0, s, 1).astype(np.float64)[..., None]
        at = (y - m.astype(np.float64)[..., None]) / step
        codes = np.where(s[..., None] > 0, np.clip(np.rint(at), 0, 15), 0)
    bad = ~np.isfinite(y).all(-1)
    m, s = np.where(bad, np.float16(np.nan), m), np.where(bad, np.float16(np.nan), s)
    codes = np.where(bad[..., None], 0, codes).astype(np.int64)
    return codes.reshape(x.shape), s, m, abs(at - np.floor(at) - 0.5).reshape(x.shape)


def pack(codes):
    """Codes [..., D], two a byte, the even one in the low half."""
    c = np.asarray(codes).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def values(packed, params):
    """(values [..., D], their sizes s code + |m|) of packed codes and params [..., D / g, 2]."""
    packed, params = np.asarray(packed), np.asarray(params, np.float64)
    c = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], 2 * packed.shape[-1]).astype(np.float64)
    g = c.shape[-1] // params.shape[-2]
    s, m = (np.repeat(params[..., i], g, -1) for i in (0, 1))
    return m + s * c, s * c + abs(m)


def attention(q, k_codes, k_params, v_codes, v_params, lengths, scale=None, weights_rounded=2.0 ** -22,
              factors_rounded=2.0 ** -22):
    """q [B, Tq, H, D]; row t sees the first lengths[b] - Tq + t + 1 slots. (out, bound): a
    score sums D products of q with s c and with m, each a fp32 sum (D + 24 half steps of
    the sizes, which do not cancel where the values do) of q's two halves (2^-22 of q); its
    weight is off by that times ln 2, twice (numerator and sum); sums over n slots add
    n + 64 half steps, exp2, its argument's rounding and the division under 2^-20, and a
    weight's own rounding before it meets the codes `weights_rounded`."""
    q = np.asarray(q, np.float64)
    B, Tq, H, D = q.shape
    KVH = k_codes.shape[1]
    G = H // KVH
    scale = D ** -0.5 if scale is None else scale
    out, ob = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        for kv in range(KVH):
            most = max(0, min(int(lengths[b]), k_codes.shape[2]))
            (Ka, Ksa), (Va, Vsa) = (values(c[b, kv, :most], p[b, kv, :most]) for c, p in ((k_codes, k_params), (v_codes, v_params)))
            for t in range(Tq):
                n = most - Tq + t + 1
                if n <= 0:
                    continue
                K, Ks, V, Vs = Ka[:n], Ksa[:n], Va[:n], Vsa[:n]
                for h in range(kv * G, (kv + 1) * G):
                    s = K @ q[b, t, h] * scale
                    size = (Ks @ abs(q[b, t, h]) * abs(scale)).max()
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    rel = 2 * ((D + 24) * U + factors_rounded) * size + (n + 64) * U + 2.0 ** -20 + weights_rounded
                    out[b, t, h] = w @ V
                    ob[b, t, h] = rel * (w @ Vs)
    return out, ob
