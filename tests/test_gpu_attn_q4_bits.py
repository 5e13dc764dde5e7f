"""What attention over a 4-bit cache keeps of its operands' bits, against the 64-bit oracle: values
of one sign, scores whose parts cancel, small values beside large ones."""

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd import _lib
from siliconfer_amd.kernels.kv_q4 import attention_q4kv
from test_gpu_attn_q4 import DT, cache

pytestmark = pytest.mark.gpu


def of_codes(codes, s, m, group, dev):
    """A cache's (codes, params) of codes [B, KVH, n, D] and, a group, s and m [B, KVH, n, D / group]."""
    params = np.stack(np.broadcast_arrays(s, m), -1).astype(np.float16)
    assert params.shape[:3] == codes.shape[:3] and params.shape[3] * group == codes.shape[3]
    return [torch.from_numpy(O.pack(codes)).to(dev), torch.from_numpy(params).to(dev)]


def by_many_rows(q, bufs, length, out):
    """Whether the kernel of many rows takes a call (few rows in one split need no workspace)."""
    B, rows, H, D = q.shape
    code = [_lib.dt(torch.empty(0, dtype=t)) for t in (q.dtype, DT[out])]
    KVH, group = bufs[0].shape[1], D // bufs[1].shape[3]
    return _lib.load().sf_attn_q4_workspace_bytes(B, rows, H, KVH, length, D, group, *code, 1) > 0


def close(got, q, bufs, lengths, rounded, factors, more=(), scale=None):
    """|got - oracle| within its bound for weights (and V) off by `rounded` and scores' factors by
    `factors`, half a step of got's type, and the bounds that `more` V's (codes, params) have."""
    host = lambda bufs: [t.cpu().numpy().astype(np.float64 if t.is_floating_point() else np.uint8) for t in bufs]
    k, x = host(bufs[:2]), q.double().cpu().numpy()
    want, bound = O.attention(x, *k, *host(bufs[2:]), lengths, scale, rounded, factors)
    for v in more:
        bound = bound + O.attention(x, *k, *host(v), lengths, scale, rounded, factors)[1]
    g = got.double().cpu().numpy()
    tol = bound + torch.finfo(got.dtype).eps / 2 * (abs(want) + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    assert (abs(g - want) <= tol).all(), float((abs(g - want) / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,KVH,D,group", [(4, 2, 64, 64), (4, 1, 64, 32), (8, 2, 128, 32), (4, 2, 80, 80)])
@pytest.mark.parametrize("rows", [1, 3, 9, 20])
def test_values_of_one_sign(dev, rows, H, KVH, D, group, dtype):
    """Codes of 0 stand for the minimum alone. For a bf16 output the codes stand beside the weights as
    they are, so that a dim of zeros is exactly 0. Others hold weights to 2^-22 beside a code less 8,
    and 8 s in fp32 with the minimum: they are off by the bound of values of 8 s besides."""
    B, bf16 = 2, dtype == "bf16"
    g = np.random.default_rng(rows)
    for n in (2, 64, 700):
        codes = g.integers(0, 16, (B, KVH, n, D))
        codes[..., ::3] = 0
        s = g.uniform(0.5, 1.5, (B, KVH, n, D // group)).astype(np.float16)
        k = cache(B, KVH, n, D, group, dev, seed=n)[:2]
        eights = of_codes(np.full_like(codes, 8), s, np.zeros_like(s), group, dev)
        q = torch.randn(B, rows, H, D, generator=torch.Generator().manual_seed(n)).to(DT[dtype]).to(dev)
        for part in (0.0, 1 / 32):
            bufs = k + of_codes(codes, s, (s * part).astype(np.float16), group, dev)
            for n_splits in (1, 2):
                y = attention_q4kv(q, *bufs, lengths=n, n_splits=n_splits, out_dtype=DT[dtype])
                close(y, q, bufs, [n] * B, 2.0 ** -22, 2.0 ** -22, () if bf16 else (eights,))
                if part == 0 and bf16:
                    assert (y[..., ::3] == 0).all()


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("H,KVH,D,group,rows", [(4, 2, 64, 32, 1), (8, 2, 128, 64, 3), (4, 1, 96, 32, 9), (36, 18, 64, 32, 260),
                                                (36, 18, 128, 64, 260)])
def test_scores_whose_parts_cancel(dev, rows, H, KVH, D, group, out):
    """fp32 queries of two large dims, over keys of t and 2 - t there: their scores are apart by what
    fp16 cannot hold of the queries, whatever type the output has. V is t too."""
    B, n = 2, 300
    g = np.random.default_rng(D)
    codes = np.zeros((B, KVH, n, D), np.int64)
    codes[..., 0] = g.integers(1, 16, (B, KVH, n))
    codes[..., D // 2] = 16 - codes[..., 0]
    s = np.full((B, KVH, n, D // group), 0.125)
    bufs = 2 * of_codes(codes, s, np.zeros_like(s), group, dev)
    q = torch.zeros(B, rows, H, D)
    q[..., 0] = 1000 + torch.rand(B, rows, H, generator=torch.Generator().manual_seed(rows))
    q[..., D // 2] = 1000 + torch.rand(B, rows, H, generator=torch.Generator().manual_seed(rows + 1))
    q = q.to(dev)
    assert by_many_rows(q, bufs, n, out) is (rows == 260)
    y = attention_q4kv(q, *bufs, lengths=n, scale=1.0, out_dtype=DT[out])
    # (V and weights: both in two parts; V's codes less 8, as above)
    eights = of_codes(np.full_like(codes, 8), s, np.zeros_like(s), group, dev)
    close(y, q, bufs, [n] * B, 2.0 ** -21, 2.0 ** -22, (eights,), 1.0)


def test_weights_of_a_prompt_are_rounded(dev):
    """bf16 queries and outputs, many rows: slot 0 holds 1 and weighs about what all others, which hold
    -1, weigh together. K and V are exact in fp16, so that a row is off by its weights' rounding, 2^-11
    at most of the others', and by its own."""
    H, KVH, D, rows, n = 32, 16, 128, 260, 300
    k, v = (np.zeros((1, KVH, n, D, 1)) for _ in range(2))
    k[:, :, 1:, 0], v[:, :, :], v[:, :, 0] = 1, -1, 1  # (codes of dim 0 below: 0 for slot 0, else 1, of -1 each)
    codes = k[..., 0].astype(np.int64)
    s, zero = np.full((1, KVH, n, 2), -1.0), np.zeros((1, KVH, n, 2))
    bufs = of_codes(codes, s, zero, 64, dev) + of_codes(np.zeros_like(codes), zero, v[..., :2, 0], 64, dev)
    others = torch.arange(n - rows, n, dtype=torch.float64)
    q = torch.zeros(1, rows, H, D, dtype=torch.float64)
    q[..., 0] = (others.log()[None, :, None] + torch.randn(1, rows, H, generator=torch.Generator().manual_seed(0)) / 32)
    q = q.to(dev, torch.bfloat16)
    assert by_many_rows(q, bufs, n, "bf16")
    y = attention_q4kv(q, *bufs, lengths=n, scale=1.0, out_dtype=torch.bfloat16).double().cpu()
    w = others[:, None] * torch.exp(-q[0, :, :, 0].double().cpu())  # of the others together, slot 0 weighing 1
    want = (1 - w) / (1 + w)
    # fp32: a score's products with 1.44 and 2^f, the sums of 300 weights
    tol = w / (1 + w) * 2.0 ** -11 * (want + 1 + 2.0 ** -10) + want.abs() * 2.0 ** -8 + 400 * 2.0 ** -24
    assert ((y[0] - want[..., None]).abs() <= tol[..., None]).all(), ((y[0] - want[..., None]).abs() / tol[..., None]).max().item()


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("H,KVH,D,group", [(32, 16, 64, 32), (16, 8, 128, 64), (36, 18, 64, 32), (36, 18, 128, 64)])
def test_small_values_beside_large_ones_of_a_prompt(dev, H, KVH, D, group, out):
    """Many rows over tiles whose first group holds values up to 20000 and whose others a thousandth: in K
    (the queries are 0 beside the large ones, and large beside the small) and in V. Then some of V's
    large ones past fp16's range: the other groups keep theirs all the same."""
    B, n, rows = 2, 300, 260
    g = np.random.default_rng(D)
    codes = [g.integers(0, 16, (B, KVH, n, D)) for _ in range(2)]
    s = g.uniform(0.5, 1.5, (B, KVH, n, D // group)) * 1e-4
    m = -7.5 * s
    s[..., 0], m[..., 0] = 2700, -20000
    bufs = of_codes(codes[0], s, m, group, dev) + of_codes(codes[1], s, m, group, dev)
    gen = torch.Generator().manual_seed(D)
    q = 3000 * torch.randn(B, rows, H, D, generator=gen)
    q[..., :group] = 0
    q = q.to(DT[out]).to(dev)
    whole = out != "bf16"  # (a bf16 output: weights and V in fp16, and K where rows are many)
    how = (2.0 ** -21, 2.0 ** -22) if whole else (2.0 ** -10, 2.0 ** -11)
    eights = of_codes(np.full_like(codes[1], 8), s, np.zeros_like(s), group, dev)  # (where codes are taken less 8)
    y = attention_q4kv(q, *bufs, lengths=n, out_dtype=DT[out])
    close(y, q, bufs, [n] * B, *how, more=(eights,) if whole else ())
    far = [t.clone() for t in bufs]
    far[3][:, :, ::7, 0, 0] = 60000  # up to 880000 in the first group
    z = attention_q4kv(q, *far, lengths=n, out_dtype=DT[out])
    # (few rows' weights share one factor: 2^-38 of the largest weight times scale is their last place, here
    # 60000 2^-38 beside scales of 1e-4)
    many = by_many_rows(q, bufs, n, out)
    assert many is (not whole or KVH == 18)
    if many:
        assert torch.equal(z[..., group:], y[..., group:])
    else:
        assert ((z - y)[..., group:].abs() <= n * 8 * 60000 * 2.0 ** -38).all()


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("rows", [1, 5, 260])
def test_an_output_at_any_address(dev, rows, out):
    """A contiguous `out` that starts off 16 bytes holds what an aligned one holds, and nothing around
    it is written."""
    bufs = cache(1, 36, 300, 128, 64, dev)
    q = torch.randn(1, rows, 72, 128, generator=torch.Generator().manual_seed(0)).to(dev, DT[out])
    assert by_many_rows(q, bufs, 300, out) is (rows == 260)
    want = attention_q4kv(q, *bufs, lengths=300, out_dtype=DT[out])
    for off in (1, 2, 4, 7, 8):
        flat = torch.full((want.numel() + 16,), 7.0, dtype=DT[out], device=dev)
        y = flat[off:off + want.numel()].view(want.shape)
        assert attention_q4kv(q, *bufs, lengths=300, out=y) is y
        assert torch.equal(y, want) and (flat[:off] == 7).all() and (flat[off + want.numel():] == 7).all()
