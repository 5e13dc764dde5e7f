"""Decode attention that scores its cache (sf_attn_decode_scored_i8kv) against the
64-bit oracle, within the oracle's bound on fp32 arithmetic plus half a step of the
output's type; scores add one fp32 rounding (2^-24 of the score)."""

import numpy as np
import pytest
import torch

from oracle import attention as A
from oracle import bounded
from siliconfer_amd.kernels.attention import attention_decode_scored

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def cache(rng, B, KVH, cap, D, scale_dtype=np.float16):
    out = []
    for _ in range(2):
        c, s = A.quantize_kv(rng.normal(0, 1, (B, KVH, cap, D)).astype(np.float32))
        out += [c, s[..., 0].astype(scale_dtype)]
    return out  # k codes, k scales, v codes, v scales


def run(dev, q, kv, scores, lengths, **kw):
    t = [torch.as_tensor(a).to(dev) for a in kv]
    sc = torch.as_tensor(scores).to(dev)
    le = lengths if isinstance(lengths, int) else torch.as_tensor(np.asarray(lengths, np.int32)).to(dev)
    out = attention_decode_scored(q.to(dev), *t, sc, lengths=le, **kw)
    return out, sc.cpu().numpy()


def check(dev, q, kv, lengths, out_dtype=torch.float32, **kw):
    B, Tq, H, D = q.shape
    KVH, cap = kv[0].shape[1:3]
    rng = np.random.default_rng(99)
    before = rng.random((B, KVH, cap)).astype(np.float32) * 0.01
    out, after = run(dev, q, kv, before, lengths, out_dtype=out_dtype, **kw)
    ns = [lengths] * B if isinstance(lengths, int) else lengths
    ref, add, ob, ab = bounded.attention_scored(q.double().numpy(), *kv, ns, kw.get("scale"))
    g = out.double().cpu().numpy()
    tol = ob + torch.finfo(out_dtype).eps / 2 * (abs(ref) + ob) + (2.0 ** -25 if out_dtype == torch.float16 else 1e-37)
    assert (abs(g - ref) <= tol).all(), float((abs(g - ref) / tol).max())
    want = before.astype(np.float64) + add
    stol = ab + 2.0 ** -24 * (abs(want) + ab) + 1e-37
    assert (abs(after - want) <= stol).all(), float((abs(after - want) / stol).max())
    for b, n in enumerate(ns):
        assert np.array_equal(after[b, :, max(n, 0):], before[b, :, max(n, 0):])
    return g


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 127, 500, 1501])
def test_lengths(dev, dtype, T):
    rng = np.random.default_rng(T)
    q = torch.from_numpy(rng.normal(0, 1.5, (1, 1, 14, 64)).astype(np.float32)).to(DT[dtype])
    check(dev, q, cache(rng, 1, 2, T + T % 3, 64), T)


@pytest.mark.parametrize("H,KVH,D", [(4, 4, 8), (6, 2, 16), (9, 3, 80), (12, 1, 96), (8, 2, 128), (32, 8, 128),
                                     (16, 4, 256), (40, 2, 128), (17, 1, 72), (33, 1, 24), (5, 5, 200), (2, 1, 64)])
@pytest.mark.parametrize("Tq", [1, 3])
def test_geometries(dev, H, KVH, D, Tq):
    rng = np.random.default_rng(H * D + Tq)
    q = torch.from_numpy(rng.normal(0, 1, (2, Tq, H, D)).astype(np.float32))
    check(dev, q.bfloat16() if D == 128 else q, cache(rng, 2, KVH, 203, D, np.float32 if H % 2 else np.float16),
          [203, 75], out_dtype=torch.bfloat16 if D == 128 else torch.float32)


@pytest.mark.parametrize("n_splits", [1, 2, 3, 7, 64, 128, 500])
def test_splits(dev, n_splits):
    rng = np.random.default_rng(4)
    q = torch.from_numpy(rng.normal(0, 1, (2, 1, 14, 64)).astype(np.float32)).half()
    check(dev, q, cache(rng, 2, 2, 700, 64), [700, 260], n_splits=n_splits)


def test_ragged_empty_and_past_the_capacity(dev):
    """Sequences of zero slots, of fewer slots than query rows, and lengths past the
    capacity, which are cut to it."""
    rng = np.random.default_rng(5)
    q = torch.from_numpy(rng.normal(0, 1, (5, 4, 14, 64)).astype(np.float32))
    kv = cache(rng, 5, 2, 90, 64)
    g = check(dev, q, kv, [0, 2, 90, 4, 1])
    assert (g[0] == 0).all() and (g[1, :2] == 0).all() and (g[4, :3] == 0).all()
    before = np.zeros((5, 2, 90), np.float32)
    a, sa = run(dev, q, kv, before, [90, 2, 2 ** 31 - 1, -3, 50])
    b, sb = run(dev, q, kv, before, [90, 2, 90, 0, 50])
    assert torch.equal(a, b) and np.array_equal(sa, sb)


@pytest.mark.parametrize("Tq", [2, 8, 16, 32])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows(dev, Tq, dtype):
    rng = np.random.default_rng(Tq)
    q = torch.from_numpy(rng.normal(0, 1, (2, Tq, 14, 64)).astype(np.float32)).to(DT[dtype])
    check(dev, q, cache(rng, 2, 2, 333, 64), [333, 40])


def test_add_max_length_and_three_dims(dev):
    rng = np.random.default_rng(8)
    q = torch.from_numpy(rng.normal(0, 1, (2, 14, 64)).astype(np.float32))
    kv = cache(rng, 2, 2, 400, 64)
    z = np.zeros((2, 2, 400), np.float32)
    a, sa = run(dev, q, kv, z, [150, 99], add=1, n_splits=4)
    b, sb = run(dev, q[:, None], kv, z, [151, 100], max_length=160, n_splits=4)
    assert a.shape == (2, 14, 64) and torch.equal(a, b[:, 0]) and np.array_equal(sa, sb)
    c, sc = run(dev, q, kv, z, 150, add=1, n_splits=4)
    d, sd = run(dev, q, kv, z, [151, 151], n_splits=4)
    assert torch.equal(c, d) and np.array_equal(sc, sd)


def test_stale_slots_do_not_reach_the_result(dev):
    """NaN and infinite scales, and any codes, at and past a sequence's length."""
    rng = np.random.default_rng(9)
    q = torch.from_numpy(rng.normal(0, 1, (2, 2, 14, 64)).astype(np.float32))
    kv = cache(rng, 2, 2, 128, 64)
    z = np.zeros((2, 2, 128), np.float32)
    a, sa = run(dev, q, kv, z, [77, 50])
    for i, bad in ((1, np.nan), (3, np.inf)):
        kv[i][0, :, 77:] = bad
        kv[i][1, :, 50:] = bad
    kv[0][:, :, 77:] = -128
    b, sb = run(dev, q, kv, z, [77, 50])
    assert torch.equal(a, b) and np.array_equal(sa, sb)


@pytest.mark.parametrize("qs,ks,vs", [(3e4, 1e-6, 1e20), (1e-20, 1e18, 1e-20), (1e5, 1e-7, 1.0), (1.0, 1.0, 1e35)])
def test_magnitudes(dev, qs, ks, vs):
    """fp32 queries and scales far outside fp16's range."""
    rng = np.random.default_rng(11)
    q = torch.from_numpy((rng.normal(0, 1, (1, 1, 8, 128)) * qs).astype(np.float32))
    kv = cache(rng, 1, 2, 600, 128, np.float32)
    kv[1] *= np.float32(ks)
    kv[3] *= np.float32(vs)
    kv[3][0, 0, ::7] *= np.float32(1e-3)
    check(dev, q, kv, 600)


def test_one_slot_takes_all_the_weight(dev):
    """A key far above the others: its weight is 1, the others' underflow to 0."""
    rng = np.random.default_rng(12)
    kv = cache(rng, 1, 1, 300, 64)
    kv[0][0, 0, 123] = 127
    kv[1][0, 0, 123] = 60.0
    q = torch.ones(1, 1, 4, 64)
    z = np.zeros((1, 1, 300), np.float32)
    out, sc = run(dev, q, kv, z, 300)
    assert sc[0, 0, 123] == 4.0 and sc.sum() == 4.0
    v = kv[2][0, 0, 123].astype(np.float32) * kv[3][0, 0, 123].astype(np.float32)
    assert np.allclose(out.cpu().numpy()[0, 0], v, rtol=2 ** -22, atol=0)


def test_repeats_are_equal_and_scores_accumulate(dev):
    rng = np.random.default_rng(13)
    q = torch.from_numpy(rng.normal(0, 1, (4, 1, 32, 128)).astype(np.float32)).bfloat16()
    kv = cache(rng, 4, 8, 900, 128)
    z = np.zeros((4, 8, 900), np.float32)
    a, sa = run(dev, q, kv, z, [900, 1, 500, 899])
    for _ in range(5):
        b, sb = run(dev, q, kv, z, [900, 1, 500, 899])
        assert torch.equal(a, b) and np.array_equal(sa, sb)
    _, twice = run(dev, q, kv, sa, [900, 1, 500, 899])
    assert np.array_equal(twice, sa + sa)


def test_graph_replays(dev):
    """Recorded once with lengths on the device, replayed as they grow, beside eager calls."""
    rng = np.random.default_rng(14)
    kv = [torch.as_tensor(a).to(dev) for a in cache(rng, 1, 2, 700, 64)]
    q = torch.from_numpy(rng.normal(0, 1, (1, 14, 64)).astype(np.float32)).to(dev)
    le = torch.tensor([600], dtype=torch.int32, device=dev)
    sc = torch.zeros(1, 2, 700, device=dev)
    eager = lambda s: attention_decode_scored(q, *kv, s, lengths=le)
    eager(sc.clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = eager(sc)
    want_sc = torch.zeros_like(sc)
    for _ in range(4):
        want = eager(want_sc)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(sc, want_sc)
        le.add_(13)
