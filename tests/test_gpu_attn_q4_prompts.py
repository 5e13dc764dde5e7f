"""Prompts over a 4-bit cache in two parts a factor, at sizes that the kernel of many rows takes: every
group, ragged and empty sequences, parameters that are not finite or past fp16's range."""

import pytest
import torch

from siliconfer_amd.kernels.kv_q4 import attention_q4kv
from test_gpu_attn_q4 import DT, cache, check
from test_gpu_attn_q4_bits import by_many_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("rows", [150, 261])
def test_two_parts(dev, rows, D, group):
    """fp32 queries with every output, 16-bit ones with fp32 and fp16: ragged, rows before a sequence's
    start, an empty sequence, scales of every sign."""
    B, H, KVH, cap = 4, 32, 16, 300
    bufs = cache(B, KVH, cap, D, group, dev, seed=rows)
    x = 1.5 * torch.randn(B, rows, H, D, generator=torch.Generator().manual_seed(rows))
    lengths = torch.tensor([rows, 0, 39, 300], dtype=torch.int32, device=dev)
    for dtype, out, scale in (("f32", "f32", None), ("f32", "bf16", -0.07), ("f16", "f16", None), ("bf16", "f32", 0.0)):
        q = x.to(DT[dtype]).to(dev)
        assert by_many_rows(q, bufs, cap, out)
        y = attention_q4kv(q, *bufs, lengths=lengths, out_dtype=DT[out], scale=scale)
        few = slice(12, 16)  # (enough heads for the oracle: kv heads 6 and 7)
        check(y[:, :, few].contiguous(), q[:, :, few], [t[:, 6:8] for t in bufs], lengths.tolist(), scale)
        assert (y[1] == 0).all() and (y[2, :max(0, rows - 39)] == 0).all()


@pytest.mark.parametrize("out", ["f32", "f16"])
@pytest.mark.parametrize("D", [64, 128])
def test_missing_and_large_values(dev, D, out):
    """Parameters of NaN before, within and past what a column sees; K and V past fp16's range."""
    B, H, KVH, rows, n = 1, 72, 36, 260, 330
    bufs = cache(B, KVH, 400, D, 32, dev, seed=1)
    q = torch.randn(B, rows, H, D, generator=torch.Generator().manual_seed(1)).to(dev, DT[out])
    assert by_many_rows(q, bufs, n, out)
    want = attention_q4kv(q, *bufs, lengths=n, out_dtype=DT[out])
    check(want[:, :, :4].contiguous(), q[:, :, :4], [t[:, :2] for t in bufs], [n])
    dirty = [t.clone() for t in bufs]
    for t in (1, 3):
        dirty[t][:, :, n:] = float("nan")
    assert torch.equal(attention_q4kv(q, *dirty, lengths=n, out_dtype=DT[out]), want)
    dirty[3][:, 3, 200, 1] = float("nan")  # of V's second group: the rows from 130 on, 32 dims
    dirty[1][:, 5, 300, 0] = float("nan")  # of K: the rows from 230 on
    y = attention_q4kv(q, *dirty, lengths=n, out_dtype=DT[out])
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[:, 130:, 6:8, 32:64] = True
    bad[:, 230:, 10:12] = True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], want[~bad])
    large = [t.clone() for t in bufs]
    large[3][:, :, 100:120, 0] *= 20000.0  # V up to some 80000: sums of the columns that see it
    large[1][:, 1, 40:50, 0] *= 12000.0    # K likewise: these slots take all the weight, or none
    large[1].clamp_(-65504, 65504)
    large[3].clamp_(-65504, 65504)
    y = attention_q4kv(q, *large, lengths=n, out_dtype=DT[out])
    check(y[:, :, :4].contiguous(), q[:, :, :4], [t[:, :2] for t in large], [n])
