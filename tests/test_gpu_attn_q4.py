"""Attention over a 4-bit cache against the 64-bit oracle and its bound, plus half a step of the
output's type: one row a sequence to many, every group, ragged and empty sequences, splits."""

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.kv_q4 import attention_q4kv

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def cache(B, KVH, cap, D, group, dev, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        c, s, m, _ = O.quantize((spread * torch.randn(B, KVH, cap, D, generator=g)).double().numpy(), group)
        out += [torch.from_numpy(O.pack(c)).to(dev), torch.from_numpy(np.stack([s, m], -1)).to(dev)]
    return out


def check(got, q, bufs, lengths, scale=None, many=False):
    """A bf16 output comes from q and weights in fp16 (2^-12 of each, 2^-11 where they are cut). many:
    the kernel of many rows may have taken the call, which takes K and V in fp16 too."""
    kc, kp, vc, vp = (t.cpu().numpy() for t in bufs)
    bf16 = got.dtype == torch.bfloat16
    rounded = (3 if many else 1) * 2.0 ** -11 if bf16 else 2.0 ** -22  # (of the weights and V, before they are summed)
    q4 = q if q.dim() == 4 else q[:, None]
    want, bound = O.attention(q4.double().cpu().numpy(), kc, kp.astype(np.float64), vc, vp.astype(np.float64), lengths, scale,
                              rounded, (2.0 ** -10 if many else 2.0 ** -11) if bf16 else 2.0 ** -22)
    g = got.double().cpu().numpy().reshape(want.shape)
    tol = bound + torch.finfo(got.dtype).eps / 2 * (abs(want) + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    top = 65520.0 if got.dtype == torch.float16 else np.inf  # fp16 rounds to infinity from there on
    past = abs(want) - tol > top
    assert (g[past] == np.sign(want[past]) * np.inf).all()
    near = ~past & ((abs(want) + tol < top) | np.isfinite(g))
    assert (near | past | (abs(want) + tol >= top)).all()
    assert (abs(g - want)[near] <= tol[near]).all(), float((abs(g - want)[near] / np.maximum(tol[near], 1e-300)).max())


GEOMETRIES = [(14, 2, 64, 64), (14, 2, 64, 32), (8, 2, 128, 64), (4, 1, 128, 128), (3, 3, 128, 32), (4, 2, 80, 80),
              (6, 3, 96, 32), (2, 1, 256, 64), (4, 2, 256, 256), (40, 2, 128, 64), (5, 1, 16, 16), (2, 1, 192, 64),
              (1, 1, 48, 48), (3, 1, 112, 112), (16, 1, 64, 64), (2, 1, 160, 32), (2, 1, 256, 128), (2, 1, 256, 32)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,KVH,D,group", GEOMETRIES)
def test_rows(dev, dtype, H, KVH, D, group):
    B, cap = 3, 200
    bufs = cache(B, KVH, cap, D, group, dev, seed=D + group)
    g = torch.Generator().manual_seed(H)
    lengths = torch.tensor([200, 67, 0], dtype=torch.int32, device=dev)
    for Tq in (1, 3, 17):
        q = (2 * torch.randn(B, Tq, H, D, generator=g)).to(DT[dtype]).to(dev)
        for out in (torch.float32, DT[dtype]):
            for n_splits in (None, 1, 3):
                y = attention_q4kv(q, *bufs, lengths=lengths, n_splits=n_splits, out_dtype=out)
                assert y.shape == q.shape and y.dtype is out
                check(y, q, bufs, lengths.tolist())
    y = attention_q4kv(q[:, 0].contiguous(), *bufs, lengths=64, scale=0.05)
    check(y, q[:, 0], bufs, [64] * B, 0.05)


@pytest.mark.parametrize("D,group,H,KVH", [(64, 64, 14, 2), (128, 64, 8, 2), (80, 80, 2, 1), (128, 32, 4, 4)])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 257, 1000])
def test_lengths(dev, n, D, group, H, KVH):
    """Lengths around the tiles' ends, as an int and from the device, rows before the cache's start."""
    bufs = cache(1, KVH, 1003, D, group, dev, seed=n)
    g = torch.Generator().manual_seed(n)
    for Tq in (1, 5):
        q = torch.randn(1, Tq, H, D, generator=g).to(dev)
        a = attention_q4kv(q, *bufs, lengths=n)
        check(a, q, bufs, [n])
        dev_len = torch.tensor([n - 2], dtype=torch.int32, device=dev)
        b = attention_q4kv(q, *bufs, lengths=dev_len, add=2, n_splits=2)
        check(b, q, bufs, [n])
        c = attention_q4kv(q, *bufs, lengths=torch.tensor([5000], dtype=torch.int32, device=dev), max_length=n)
        check(c, q, bufs, [n])
        if Tq > n:
            assert (a[:, :Tq - n] == 0).all()


@pytest.mark.parametrize("rows", [16, 40, 100, 333])
@pytest.mark.parametrize("H,KVH,D,group", [(14, 2, 64, 64), (4, 1, 128, 64), (2, 2, 128, 128), (2, 1, 128, 32), (2, 1, 64, 32),
                                           (2, 1, 96, 96), (1, 1, 256, 64)])
def test_prompts(dev, rows, H, KVH, D, group):
    """A prompt's rows, whole or behind a prefix, ragged, longer than a sequence."""
    bufs = cache(2, KVH, 400, D, group, dev, seed=rows)
    g = torch.Generator().manual_seed(rows)
    lengths = torch.tensor([rows + 30, rows - 11], dtype=torch.int32, device=dev)
    for dtype in DT.values():
        q = (1.5 * torch.randn(2, rows, H, D, generator=g)).to(dtype).to(dev)
        for out in {torch.float32, dtype}:
            check(attention_q4kv(q, *bufs, lengths=lengths, out_dtype=out), q, bufs, lengths.tolist())


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("rows", [150, 261])
def test_many_rows(dev, rows, D, group):
    """Enough rows, heads and sequences for the workgroups of 128 columns: every group and type,
    ragged, rows before a sequence's start, an empty sequence, scales of every sign."""
    B, H, KVH, cap = 4, 32 if D == 64 else 16, 16 if D == 64 else 8, 300
    bufs = cache(B, KVH, cap, D, group, dev, seed=rows)
    g = torch.Generator().manual_seed(rows)
    lengths = torch.tensor([rows, 0, 39, 300], dtype=torch.int32, device=dev)
    for dtype in DT.values():
        q = (1.5 * torch.randn(B, rows, H, D, generator=g)).to(dtype).to(dev)
        for out, scale in ((torch.float32, None), (dtype, -0.07), (torch.bfloat16, 0.0)):
            y = attention_q4kv(q, *bufs, lengths=lengths, out_dtype=out, scale=scale)
            check(y, q, bufs, lengths.tolist(), scale, many=True)
            assert (y[1] == 0).all() and (y[2, :max(0, rows - 39)] == 0).all()


@pytest.mark.parametrize("out", list(DT))
def test_many_rows_with_large_and_missing_values(dev, out):
    """K and V past fp16's range once put together, and parameters of NaN: before, within and
    past what a column sees."""
    B, H, KVH, D, rows, n = 1, 64, 32, 128, 260, 330
    bufs = cache(B, KVH, 400, D, 64, dev, seed=1)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(B, rows, H, D, generator=g).to(dev)
    want = attention_q4kv(q, *bufs, lengths=n, out_dtype=DT[out])
    dirty = [t.clone() for t in bufs]
    for t in (1, 3):
        dirty[t][:, :, n:] = float("nan")
    assert torch.equal(attention_q4kv(q, *dirty, lengths=n, out_dtype=DT[out]), want)
    dirty[3][:, 3, 200, 1] = float("nan")  # of V's second group: the rows from 130 on, dims from 64 on
    dirty[1][:, 5, 300, 0] = float("nan")  # of K: the rows from 230 on
    y = attention_q4kv(q, *dirty, lengths=n, out_dtype=DT[out])
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[:, 130:, 6:8, 64:] = True
    bad[:, 230:, 10:12] = True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], want[~bad])
    large = [t.clone() for t in bufs]
    large[3][:, :, 100:120, 0] *= 20000.0   # V up to some 80000: sums of the columns that see it
    large[3][:, 1] *= 30000.0
    large[1][:, 2, 40:50, 0] *= 12000.0     # K likewise: these slots take all the weight, or none
    large[1].clamp_(-65504, 65504)
    large[3].clamp_(-65504, 65504)
    few = slice(0, 8)  # (of the first kv heads: enough for the oracle)
    y = attention_q4kv(q, *large, lengths=n, out_dtype=DT[out])
    check(y[:, :, few].contiguous(), q[:, :, few], [t[:, :4] for t in large], [n], None, many=True)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (80, 80)])
def test_what_a_row_does_not_see(dev, rows, D, group):
    """Parameters of NaN past a row's own slot, and codes there, change nothing; a NaN that a row
    sees is that row's alone."""
    bufs = cache(1, 1, 200, D, group, dev)
    q = torch.randn(1, rows, 2, D, generator=torch.Generator().manual_seed(1)).to(dev)
    want = attention_q4kv(q, *bufs, lengths=150)
    dirty = [t.clone() for t in bufs]
    for t in dirty:
        t[:, :, 150:] = float("nan") if t.is_floating_point() else 255
    assert torch.equal(attention_q4kv(q, *dirty, lengths=150), want)
    if rows > 1:  # a slot that only the rows from 40 on see
        at = 150 - rows + 40
        for t in (1, 3):
            dirty[t][:, :, at] = float("nan")
        y = attention_q4kv(q, *dirty, lengths=150)
        assert torch.equal(y[:, :40], want[:, :40]) and y[:, 40:].isnan().all()


@pytest.mark.parametrize("rows", [1, 33])
def test_sharp_flat_and_far_scales(dev, rows):
    """Weights that all fall on one slot, or on all alike; V scales far apart between slots, the
    large ones where no weight is; a common scale of 1e-4 and of 1e4."""
    D, group, n = 128, 64, 300
    bufs = cache(1, 2, n, D, group, dev, seed=3)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(1, rows, 4, D, generator=g).to(dev)
    for mul in (0.0, 30.0, 1e-30):
        check(attention_q4kv(q * mul, *bufs, lengths=n), q * mul, bufs, [n])
    far = [t.clone() for t in bufs]
    far[3][:, :, ::2] *= 2.0 ** -12  # every second slot's values are tiny, and only they are seen
    far[1][:, :, 1::2] = 0
    far[1][:, :, 1::2, :, 1] = -100.0
    ones = torch.ones_like(q)
    check(attention_q4kv(ones, *far, lengths=n, scale=1.0), ones, far, [n], 1.0)
    for mul in (1e-4, 1e4):
        scaled = [bufs[0], bufs[1], bufs[2], (bufs[3].float() * mul).half()]
        check(attention_q4kv(q, *scaled, lengths=n), q, scaled, [n])


def held(x, group, dev):
    c, s, m, _ = O.quantize(x, group)
    return [torch.from_numpy(O.pack(c)).to(dev), torch.from_numpy(np.stack([s, m], -1)).to(dev)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (80, 80)])
@pytest.mark.parametrize("rows", [1, 3, 9])
def test_constant_groups_under_rising_scores(dev, rows, D, group, dtype):
    """V whose groups hold one value each (scales of 0), keys whose scores rise from slot to slot by
    less than what moves a softmax's reference: every weight past the first tile's is over 1."""
    B, H, KVH, n = 2, 4, 2, 700
    g = np.random.default_rng(rows)
    k = np.zeros((B, KVH, n, D)) + (np.arange(n) / 100)[:, None]
    v = np.repeat(g.standard_normal((B, KVH, n, D // group)), group, -1)
    bufs = held(k, group, dev) + held(v, group, dev)
    assert (bufs[3][..., 0] == 0).all()
    q = torch.full((B, rows, H, D), D ** -0.5).to(DT[dtype]).to(dev)
    for n_splits in (1, 2, None):
        check(attention_q4kv(q, *bufs, lengths=n, n_splits=n_splits, out_dtype=DT[dtype]), q, bufs, [n] * B)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (80, 80)])
@pytest.mark.parametrize("rows", [1, 3, 9])
def test_small_values_that_outweigh_large_ones(dev, rows, D, group, dtype):
    """Large V, then at scores that leave it no weight V of a billionth, zeros, and V of a
    hundredth, few slots each in one wave's tiles."""
    B, H, KVH, n = 1, 4, 2, 1030
    g = np.random.default_rng(rows)
    at = np.arange(n)
    level = np.where(at < 64, 0.0, np.where((at >= 256) & (at < 261), 40.0, np.where(at < 512, -40.0, np.where(at < 1024, -20.0, 60.0))))
    size = np.where(at < 64, 50000.0, np.where(at < 512, 3e-5, np.where(at < 1024, 0.0, 300.0)))
    k = np.zeros((B, KVH, n, D)) + level[:, None]
    v = g.uniform(-1, 1, (B, KVH, n, D)) * size[:, None]
    bufs = held(k, group, dev) + held(v, group, dev)
    q = torch.full((B, rows, H, D), D ** -0.5).to(DT[dtype]).to(dev)
    for length in (261 + rows, 800, n):
        for n_splits in (1, 2, None):
            y = attention_q4kv(q, *bufs, lengths=length, n_splits=n_splits, out_dtype=DT[dtype])
            check(y, q, bufs, [length] * B)


@pytest.mark.parametrize("D", [64, 128])
def test_resident_workgroups(dev, D):
    """More workgroups than CUs, up to two a CU: the first ones' columns in the other order, and for
    a bf16 output four waves each."""
    B, H, KVH, rows, cap = 2, 64, 32, 300, 333
    bufs = cache(B, KVH, cap, D, 64, dev, seed=D)
    q = (1.5 * torch.randn(B, rows, H, D, generator=torch.Generator().manual_seed(D))).to(dev)
    lengths = torch.tensor([333, 290], dtype=torch.int32, device=dev)
    for dtype in DT.values():
        x = q.to(dtype)
        y = attention_q4kv(x, *bufs, lengths=lengths, out_dtype=dtype)
        for heads in (slice(0, 2), slice(30, 32)):  # (enough for the oracle)
            rows_of = slice(2 * heads.start, 2 * heads.stop)
            check(y[:, :, rows_of].contiguous(), x[:, :, rows_of], [t[:, heads] for t in bufs], [333, 290], many=True)



def test_long_cache(dev):
    """70000 slots through many splits; the slots far behind weigh what they should."""
    D, KVH, n = 64, 1, 70001
    g = torch.Generator(device=dev).manual_seed(1)
    bufs = []
    for _ in range(2):
        bufs += [torch.randint(0, 256, (1, KVH, n, D // 2), generator=g, device=dev, dtype=torch.uint8),
                 torch.rand(1, KVH, n, 1, 2, generator=g, device=dev).half() * 0.25]
    q = torch.randn(1, 2, D, generator=g, device=dev)
    for n_splits in (None, 1, 128):
        check(attention_q4kv(q, *bufs, lengths=n, n_splits=n_splits), q, bufs, [n])


def test_streams_and_graphs(dev):
    """Two graphs, and eager calls on a side stream between their replays, keep out of each other's
    workspaces; replays follow the device lengths."""
    g = torch.Generator().manual_seed(5)
    bufs = cache(2, 2, 700, 128, 64, dev)
    q = torch.randn(2, 1, 8, 128, generator=g).to(dev)
    lengths = torch.tensor([600, 40], dtype=torch.int32, device=dev)
    graphs, outs = [], []
    attention_q4kv(q, *bufs, lengths=lengths)
    for n_splits in (4, 9):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attention_q4kv(q, *bufs, lengths=lengths, n_splits=n_splits))
        graphs.append(graph)
    s = torch.cuda.Stream()
    for i in range(3):
        lengths.copy_(torch.tensor([600 - i, 40 + 3 * i], dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0].replay()
        graphs[1].replay()
        eager = attention_q4kv(q, *bufs, lengths=lengths, n_splits=4)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager)
        assert torch.equal(outs[1], attention_q4kv(q, *bufs, lengths=lengths, n_splits=9))
        check(outs[1], q, bufs, lengths.tolist())


def test_out_and_refusals(dev):
    bufs = cache(1, 2, 64, 64, 32, dev)
    q = torch.randn(1, 3, 4, 64, device=dev)
    out = torch.empty(1, 3, 4, 64, device=dev, dtype=torch.bfloat16)
    assert attention_q4kv(q, *bufs, lengths=9, out=out) is out
    check(out, q, bufs, [9])
    for bad, text in ((dict(lengths=65), "65 slots"), (dict(lengths=9, add=60), "slots"), (dict(lengths=torch.zeros(1, dtype=torch.int32, device=dev), max_length=65), "invalid"),
                      (dict(lengths=torch.zeros(2, dtype=torch.int32, device=dev)), "lengths"), (dict(lengths=9, add=1 << 31), "32 bits"),
                      (dict(lengths=2, add=-3), "invalid"), (dict(lengths=9, out=out[:, :1]), "out must be")):
        with pytest.raises(SFError, match=text):
            attention_q4kv(q, *bufs, **bad)
    with pytest.raises(SFError, match="does not match q"):
        attention_q4kv(q[..., :32].contiguous(), *bufs, lengths=9)
    with pytest.raises(SFError, match="not a multiple"):
        attention_q4kv(q[:, :, :3].contiguous(), *bufs, lengths=9)
    with pytest.raises(SFError, match="contiguous"):
        attention_q4kv(q.transpose(1, 2), *bufs, lengths=9)
    with pytest.raises(SFError, match="k/v codes must be"):
        attention_q4kv(q, bufs[0].char(), *bufs[1:], lengths=9)
    with pytest.raises(SFError, match="dtype"):
        attention_q4kv(q.int(), *bufs, lengths=9)
