"""Scored decode attention where every score is exact but for its scaling: each query has one
nonzero dim, so a product is one term of at most 23 bits, and the bound is that of the softmax
and of the sums alone. It is tight enough to tell weights (or queries) held in fp16 alone from
the high and low parts that the kernel carries; the CPU restates both to show it."""

import numpy as np
import pytest
import torch

from siliconfer_amd.kernels.attention import attention_decode_scored

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 14, 2, 64, 24, 0), (2, 8, 2, 128, 70, 0), (1, 9, 3, 72, 33, 2), (1, 8, 4, 256, 64, 3), (3, 4, 1, 64, 70, 3)]


def case(shape, dtype, seed=0):
    Tq, H, KVH, D, n, n_splits = shape
    r = np.random.default_rng(seed + D + n)
    bits = {"f32": 16, "f16": 11, "bf16": 8}[dtype]
    q = np.zeros((1, Tq, H, D), np.float32)
    for t in range(Tq):
        for h in range(H):  # 1 .. 2 in `bits` bits
            q[0, t, h, r.integers(D)] = r.choice([-1, 1]) * (1 + r.integers(1 << (bits - 1)) * 2.0 ** (1 - bits))
    cap = n + 3
    k, v = (r.integers(-127, 128, (1, KVH, cap, D)).astype(np.int8) for _ in range(2))
    ks = np.full((1, KVH, cap), 2.0 ** -7, np.float32)
    vs = r.uniform(0.005, 0.02, (1, KVH, cap)).astype(np.float16).astype(np.float32)
    return q, k, ks, v, vs, n, n_splits


def reference(q, k, ks, v, vs, n, round_p=None, round_q=None):
    """(out, weights summed a slot, bounds of both). A base-2 score is at most 2.9 and its scaling takes four
    roundings (the factor's constant, the factor, the slot's, the product), its difference to the maximum, at most
    5.8, one: 17.4 2^-24, ln 2 times that of the weight, and exp2's last place (2 2^-24): 14 2^-24. The sum is off by
    as much and a rounding a slot; products with V by two a slot (high and low part) and 16 for the scale, the
    parts' 2^-22 and the waves', splits' and tiles' factors."""
    B, Tq, H, D = q.shape
    KVH = k.shape[1]
    out, ob = np.zeros(q.shape), np.zeros(q.shape)
    add, ab = np.zeros(k.shape[:3]), np.zeros(k.shape[:3])
    for t in range(Tq):
        m = n - Tq + t + 1
        for h in range(H):
            kv = h // (H // KVH)
            x = q[0, t, h] if round_q is None else round_q(q[0, t, h])
            s = (k[0, kv, :m].astype(np.float64) * ks[0, kv, :m, None]) @ x.astype(np.float64)
            w = np.exp(s - s.max())
            V = v[0, kv, :m].astype(np.float64) * vs[0, kv, :m, None]
            p = w * vs[0, kv, :m]
            if round_p is not None:
                p = round_p(p)
            out[0, t, h] = (p @ v[0, kv, :m].astype(np.float64)) / w.sum()
            w /= w.sum()
            ob[0, t, h] = (2 * 14 + 3 * m + 16) * 2.0 ** -24 * (w @ abs(V))
            add[0, kv, :m] += w
            ab[0, kv, :m] += (2 * 14 + m + 16) * 2.0 ** -24 * w
    return out, add, ob, ab


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_within_the_softmax_s_own_rounding(dev, shape, dtype):
    q, k, ks, v, vs, n, n_splits = case(shape, dtype)
    t = [torch.from_numpy(a).to(dev) for a in (k, ks, v, vs)]
    scores = torch.zeros(k.shape[:3], device=dev)
    out = attention_decode_scored(torch.from_numpy(q).to(dev, DT[dtype]), *t, scores, lengths=n, scale=1.0,
                                  n_splits=n_splits)
    ref, add, ob, ab = reference(q, k, ks, v, vs, n)
    err = abs(out.double().cpu().numpy() - ref)
    assert (err <= ob + 2.0 ** -24 * abs(ref)).all(), float((err / ob).max())
    err = abs(scores.double().cpu().numpy() - add)
    assert (err <= ab + shape[0] * shape[1] * 2.0 ** -24 * add + 1e-30).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_the_bound_tells_fp16_alone(shape):
    """The same in fp16 alone, weights or 16-bit queries, lies well outside (on the CPU)."""
    q, *rest = case(shape, "f32")
    ref, add, ob, ab = reference(q, *rest[:-1])
    half = lambda x: x.astype(np.float16).astype(np.float64)
    scaled = lambda p: half(p * (2.0 ** 13 / p.max())) * (p.max() / 2.0 ** 13)
    out, _, _, _ = reference(q, *rest[:-1], round_p=scaled)
    assert (abs(out - ref) > ob).mean() > 0.3 and (abs(out - ref) / ob).max() > 4
    out, low, _, _ = reference(q, *rest[:-1], round_q=half)
    assert (abs(out - ref) > ob).mean() > 0.3 and (abs(low - add) / np.maximum(ab, 1e-30)).max() > 4
