"""Drawing tokens from given numbers (sf_sample) against the 64-bit oracle: tokens are
equal, except where u lies within the weights' rounding of a border between two
(the oracle names the neighbour); log probabilities to fp32's rounding and the
weights' (2^-23 of the value and 2^-23 absolute)."""

import numpy as np
import pytest
import torch

from oracle import bounded
from siliconfer_amd.kernels.sampling import sample

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(dev, logits, u, **kw):
    d = {k: torch.as_tensor(v).to(dev) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    tok, lp = sample(logits.to(dev), torch.as_tensor(np.asarray(u, np.float32)).to(dev), logprobs=True, **d)
    tok, lp = tok.cpu().numpy(), lp.cpu().numpy()
    rows = logits.float().numpy()
    for b in range(rows.shape[0]):
        one = {k: (v[b].item() if isinstance(v, np.ndarray) else float(np.float32(v)) if k != "top_k" else v)
               for k, v in kw.items()}
        want, wlp, near = bounded.sample(rows[b], float(np.float32(u[b])), **one)
        assert tok[b] == want or tok[b] in near, (b, tok[b], want, near, one)
        if tok[b] == want:
            assert lp[b] == wlp or abs(lp[b] - wlp) <= 2.0 ** -23 * (1 + abs(wlp)), (b, lp[b], wlp)
    return tok


def rows(rng, B, V, dtype="f32", peaked=True):
    x = rng.normal(0, 2.5, (B, V))
    if peaked:
        x -= 1.3 * np.log1p(rng.permuted(np.broadcast_to(np.arange(V), (B, V)), axis=1)) - 10
    return torch.from_numpy(x.astype(np.float32)).to(DT[dtype])


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
            dict(temperature=1.3, top_k=50, top_p=0.95, min_p=0.02), dict(top_k=5, min_p=1.0),
            dict(temperature=0.0), dict(temperature=1e-4), dict(temperature=100.0, top_p=0.5), dict(top_p=1e-6)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: ",".join(f"{a}={b}" for a, b in k.items()) or "plain")
@pytest.mark.parametrize("V", [32000, 1001])
def test_settings(dev, dtype, kw, V):
    rng = np.random.default_rng(V)
    for peaked in (True, False):
        check(dev, rows(rng, 6, V, dtype, peaked), np.append(rng.random(4), [0.0, 1 - 2 ** -24]), **kw)


@pytest.mark.parametrize("V", [1, 2, 3, 7, 63, 64, 65, 255, 1023, 1024, 1025, 4097, 50257, 151936, 200003])
def test_vocabularies(dev, V):
    rng = np.random.default_rng(V)
    check(dev, rows(rng, 3, V), rng.random(3), temperature=0.9, top_p=0.97)
    check(dev, rows(rng, 3, V, "bf16", False), rng.random(3), top_k=min(V, 500))


def test_a_row_s_own_settings(dev):
    rng = np.random.default_rng(1)
    B = 64
    check(dev, rows(rng, B, 5000), rng.random(B),
          temperature=np.where(np.arange(B) % 5 == 0, 0, rng.random(B) * 2).astype(np.float32),
          top_k=rng.integers(-1, 200, B).astype(np.int32), top_p=rng.uniform(0.3, 1.2, B).astype(np.float32),
          min_p=(rng.random(B) * 0.1 * (np.arange(B) % 2)).astype(np.float32))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5), dict(top_k=1000, top_p=0.4)],
                         ids=str)
def test_ties(dev, kw):
    """All logits equal, and a few distinct values: ties in order of the index, the
    k-th's ties all kept, borders hit exactly."""
    u = np.arange(8) / 8.0
    for V in (1, 4, 8, 4096, 151936):
        check(dev, torch.zeros(8, V), u, **kw)
        check(dev, torch.from_numpy((np.random.default_rng(V).integers(0, 3, (8, V)) * 2.0).astype(np.float32)), u, **kw)


def test_special_logits(dev):
    """-inf, +inf and NaN; rows with nothing to draw."""
    rng = np.random.default_rng(2)
    inf, nan = float("inf"), float("nan")
    x = rows(rng, 8, 3000)
    x[0] = -inf
    x[1] = nan
    x[2, ::2] = nan
    x[3, 5:] = -inf
    x[4, 17] = inf
    x[5, [9, 40, 2999]] = inf
    x[6] = torch.where(torch.rand(3000, generator=torch.Generator().manual_seed(0)) < 0.5, x[6], torch.tensor(-inf))
    x[7, :2999] = -inf
    for kw in (dict(), dict(top_k=10, top_p=0.9), dict(temperature=0.0), dict(temperature=1e30), dict(min_p=0.1)):
        tok = check(dev, x, [0.3, 0.1, 0.6, 0.9, 0.5, 0.7, 0.2, 0.99], **kw)
        assert tok[0] == -1 and tok[1] == -1 and tok[7] == 2999


def test_numbers_outside_the_unit_interval(dev):
    x = rows(np.random.default_rng(3), 1, 500).repeat(4, 1)
    u = torch.tensor([-1.0, 2.0, float("nan"), float("inf")], device=dev)
    tok = sample(x.to(dev), u).tolist()
    order = torch.argsort(x[0], descending=True, stable=True).tolist()
    assert tok == [order[0], order[-1], order[0], order[-1]]


def test_strided_rows_and_out(dev):
    rng = np.random.default_rng(4)
    wide = rows(rng, 5, 1300).to(dev)
    u = torch.from_numpy(rng.random(5).astype(np.float32)).to(dev)
    out = torch.empty(5, dtype=torch.int32, device=dev)
    got = sample(wide[:, 3:1004], u, top_p=0.9, out=out)
    assert got is out and torch.equal(got, sample(wide[:, 3:1004].contiguous(), u, top_p=0.9))
    half = wide.half()[:, 1:1002]
    assert torch.equal(sample(half, u), sample(half.contiguous(), u))
    assert torch.equal(sample(wide[2:3, :1000].expand(5, 1000), u, top_k=20), sample(wide[2:3, :1000].repeat(5, 1), u, top_k=20))


def test_frequencies_follow_the_weights(dev):
    """Evenly spaced numbers meet every token as often as its weight says."""
    x = torch.tensor([[1.0, 3.0, 2.0, 0.0, -1.0]], device=dev).expand(100000, 5)
    u = (torch.arange(100000, device=dev) + 0.5) / 100000
    n = torch.bincount(sample(x, u.float(), temperature=0.8).long(), minlength=5).double() / 100000
    p = torch.softmax(x[0].double() / 0.8, -1)
    assert (n - p).abs().max() <= 2e-5 + 2 ** -24


def test_repeats_are_equal(dev):
    rng = np.random.default_rng(5)
    x = rows(rng, 16, 151936, "bf16", False).to(dev)
    u = torch.from_numpy(rng.random(16).astype(np.float32)).to(dev)
    first = sample(x, u, temperature=1.2, top_k=3000, top_p=0.9, logprobs=True)
    for _ in range(10):
        again = sample(x, u, temperature=1.2, top_k=3000, top_p=0.9, logprobs=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_graph_replays(dev):
    rng = np.random.default_rng(6)
    x = rows(rng, 4, 20000).to(dev)
    u = torch.from_numpy(rng.random(4).astype(np.float32)).to(dev)
    sample(x, u, top_p=0.9)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok = sample(x, u, top_p=0.9)
    for i in range(4):
        x.copy_(rows(rng, 4, 20000, peaked=bool(i % 2)))
        u.copy_(torch.from_numpy(rng.random(4).astype(np.float32)))
        g.replay()
        want = sample(x, u, top_p=0.9)
        torch.cuda.synchronize()
        assert torch.equal(tok, want)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=9001), dict(top_p=0.6), dict(min_p=0.95), dict(temperature=8.0),
                                dict(temperature=30.0, top_k=12345, top_p=0.7, min_p=0.9)], ids=str)
def test_crowded_bins(dev, kw):
    """Thousands of tokens within an eighth of a nat: spread over many keys, around zero
    (where the keys' ranges are widest), around a power of two, a few values with many
    ties each among single ones, and large values that the temperature brings together."""
    rng = np.random.default_rng(5)
    V = 40000
    x = np.stack([rng.normal(0, 1, V), rng.uniform(-0.06, 0.06, V), 4 + rng.uniform(-0.05, 0.05, V),
                  np.where(rng.random(V) < 0.5, 1 + rng.integers(0, 5, V) * 2.0 ** -9, rng.normal(1, 0.02, V)),
                  rng.normal(0, 1e-40, V), -1000 + rng.normal(0, 0.3, V)]).astype(np.float32)
    for u in (0.0, 0.37, 0.5, 0.93, 1 - 2 ** -24):
        check(dev, torch.from_numpy(x), np.full(6, u), **kw)


@pytest.mark.parametrize("T", [0.6, 1.0, 1.37])
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.999), dict(top_k=50000), dict(min_p=1e-9)], ids=str)
def test_the_last_token_of_a_crowded_bin(dev, T, kw):
    """Rows over several chunks whose maxima lie in different bins, thousands of tokens in the last
    bin (a floor of equal logits, or spread within it), and numbers at and past the end of [0, 1)."""
    rng = np.random.default_rng(7)
    V = 60000
    x = np.concatenate([rng.normal(-9, 0.02, (6, V)), rng.choice([-9.0, -8.97, -9.03], (2, V)), np.full((2, V), -9.0)])
    for r in range(10):
        at = rng.choice(V, 40, replace=False)
        x[r, at] = rng.uniform(-7, 6, 40)
    x = (x * T).astype(np.float32)
    for u in (1.0, 2.0, 1 - 2.0 ** -24, 0.9999):
        check(dev, torch.from_numpy(x), np.full(10, u), temperature=T, **kw)
