"""Eviction by accumulated weight (sf_kv_evict) against the oracle: nothing is computed,
so every buffer is equal, the slots past the new length included."""

import numpy as np
import pytest
import torch

from oracle import bounded
from siliconfer_amd.kernels.eviction import evict

pytestmark = pytest.mark.gpu


def make(rng, B, KVH, cap, D, scale_dtype=np.float16, levels=None):
    codes = [rng.integers(-127, 128, (B, KVH, cap, D)).astype(np.int8) for _ in range(2)]
    scales = [rng.random((B, KVH, cap)).astype(scale_dtype) for _ in range(2)]
    scores = rng.exponential(1, (B, KVH, cap)).astype(np.float32)
    if levels:
        scores = np.floor(scores * levels).astype(np.float32)
    positions = np.stack([[rng.permutation(3 * cap)[:cap] for _ in range(KVH)] for _ in range(B)]).astype(np.int32)
    return [codes[0], scales[0], codes[1], scales[1], scores, positions]


def check(dev, arrays, lengths, seen, budget, recent):
    scores, positions = arrays[4], arrays[5]
    B = scores.shape[0]
    t = [torch.as_tensor(a).to(dev) for a in arrays]
    arg = lambda v: v if isinstance(v, int) else torch.as_tensor(np.asarray(v, np.int32)).to(dev)
    new = evict(*t, arg(lengths), arg(seen), budget, recent)
    each = lambda v: [v] * B if isinstance(v, int) else v
    want, want_len = bounded.evict(arrays, scores, positions, each(lengths), each(seen), budget, recent)
    assert np.array_equal(new.cpu().numpy(), want_len)
    for g, w, n in zip(t, want, ("k codes", "k scales", "v codes", "v scales", "scores", "positions")):
        assert np.array_equal(g.cpu().numpy().view(np.uint8), w.view(np.uint8)), n
    return want


@pytest.mark.parametrize("n", [2, 3, 63, 64, 65, 1000, 1024, 1025, 5000])
@pytest.mark.parametrize("share", [0.01, 0.5, 0.98])
def test_lengths(dev, n, share):
    rng = np.random.default_rng(n)
    budget = max(1, int(n * share))
    check(dev, make(rng, 1, 2, n + 5, 64), n, 3 * n, budget, budget // 3)


@pytest.mark.parametrize("D,scale_dtype", [(8, np.float32), (16, np.float16), (24, np.float16), (128, np.float16),
                                           (256, np.float32), (200, np.float32)])
def test_head_dims(dev, D, scale_dtype):
    rng = np.random.default_rng(D)
    check(dev, make(rng, 2, 3, 300, D, scale_dtype), [300, 211], [900, 700], 100, 20)


def test_ragged(dev):
    """Sequences past, at and below the budget, empty ones, lengths past the capacity."""
    rng = np.random.default_rng(1)
    a = make(rng, 6, 2, 500, 64)
    check(dev, a, [500, 200, 199, 0, 201, 333], [1500, 1500, 1, 0, 1200, 10 ** 9], 200, 50)
    t = [torch.as_tensor(x).to(dev) for x in a]
    u = [x.clone() for x in t]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    x = evict(*t, i32([2 ** 31 - 1, 500, -4, 1, 2, 3]), 1500, 200, 10)
    y = evict(*u, i32([500, 500, 0, 1, 2, 3]), 1500, 200, 10)
    assert torch.equal(x, y) and x.tolist() == [200, 200, 0, 1, 2, 3]
    assert all(torch.equal(p, q) for p, q in zip(t, u))


@pytest.mark.parametrize("levels", [1, 3, 50])
def test_ties_go_to_the_lower_slot(dev, levels):
    rng = np.random.default_rng(levels)
    check(dev, make(rng, 2, 2, 3000, 8, levels=levels), 3000, 9000, 777, 0)


def test_all_equal_and_special_scores(dev):
    rng = np.random.default_rng(2)
    a = make(rng, 1, 4, 400, 16)
    a[4][0, 0] = 0.0
    a[4][0, 0, ::2] = -0.0
    a[4][0, 1, ::3] = np.nan
    a[4][0, 1, 1::3] = -np.inf
    a[4][0, 2, ::3] = np.inf
    a[4][0, 3] = -a[4][0, 3]
    for budget in (1, 100, 137, 399):
        check(dev, a, 400, 0, budget, 0)


def test_recent_tokens_stay(dev):
    """The newest tokens outrank every score, +inf included; more of them than the
    budget (positions given twice) still leave exactly the budget."""
    rng = np.random.default_rng(3)
    a = make(rng, 1, 2, 300, 16)
    a[4][0, :, ::5] = np.inf
    w = check(dev, a, 300, 900, 64, 64)
    new = {int(p) for p in a[5][0, 0, :300] if p >= 900 - 64}
    assert new <= {int(p) for p in w[5][0, 0, :64]}
    a[5][:] = 7
    check(dev, a, 300, 8, 64, 10)


@pytest.mark.parametrize("n", [32768, 40000, 100003])
def test_long(dev, n):
    rng = np.random.default_rng(n)
    check(dev, make(rng, 1, 1, n, 8), n, 3 * n, n // 3, 1000)


def test_offsets_past_32_bits(dev):
    """Codes of 2.3 GB: the last sequence's rows lie past 2^31 bytes."""
    B, KVH, cap, D = 9, 1, 1 << 20, 256
    codes = [torch.zeros(B, KVH, cap, D, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.zeros(B, KVH, cap, dtype=torch.float16, device=dev) for _ in range(2)]
    scores = torch.zeros(B, KVH, cap, device=dev)
    positions = torch.zeros(B, KVH, cap, dtype=torch.int32, device=dev)
    scores[:, 0, cap - 2] = 2.0
    scores[:, 0, :3] = 1.0
    for c in codes:
        c[:, 0, cap - 2] = torch.arange(1, B + 1, dtype=torch.int8, device=dev)[:, None]
    new = evict(codes[0], scales[0], codes[1], scales[1], scores, positions, cap, 10, 3, 0)
    assert new.tolist() == [3] * B
    for c in codes:
        assert (c[:, 0, 2] == torch.arange(1, B + 1, dtype=torch.int8, device=dev)[:, None]).all()
    assert scores[:, 0, :3].tolist() == [[1.0, 1.0, 2.0]] * B


def test_graph_replays(dev):
    rng = np.random.default_rng(6)
    arrays = make(rng, 2, 2, 600, 64)
    start = [torch.as_tensor(a).to(dev) for a in arrays]
    t = [a.clone() for a in start]
    le = torch.tensor([600, 400], dtype=torch.int32, device=dev)
    seen = torch.tensor([1800, 1800], dtype=torch.int32, device=dev)
    evict(*[a.clone() for a in start], le, seen, 128, 32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        new = evict(*t, le, seen, 128, 32)
    for n in ([600, 400], [512, 100], [129, 599]):
        le.copy_(torch.tensor(n, dtype=torch.int32))
        for a, s in zip(t, start):
            a.copy_(s)
        g.replay()
        u = [s.clone() for s in start]
        want = evict(*u, le, seen, 128, 32)
        torch.cuda.synchronize()
        assert torch.equal(new, want) and all(torch.equal(a, b) for a, b in zip(t, u))
