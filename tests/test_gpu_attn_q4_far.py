"""Attention over a 4-bit cache whose parameters, counted by group, pass 2^31."""

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd.kernels.kv_q4 import attention_q4kv, dequantize_kv_q4
from test_gpu_attn_q4 import cache

pytestmark = pytest.mark.gpu


def test_more_than_2_31_groups(dev):
    """2^28 + 64 slots of 256 dims in groups of 32, K and V in the same 43 GB: a call over the first slots
    equals one over a small cache of them, and one over all of them weighs its last slots."""
    D, group, cap, few = 256, 32, (1 << 28) + 64, 150
    need = cap * (D // 2 + 4 * (D // group))
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < need + (8 << 30):
        pytest.skip(f"needs {need >> 30} GiB of device memory")
    codes = torch.zeros(1, 1, cap, D // 2, dtype=torch.uint8, device=dev)
    params = torch.zeros(1, 1, cap, D // group, 2, dtype=torch.float16, device=dev)
    small = cache(1, 1, few, D, group, dev, seed=1)[:2]
    for at in (0, cap - few):
        codes[:, :, at:at + few], params[:, :, at:at + few] = small
    q = torch.randn(1, 2, 3, D, generator=torch.Generator().manual_seed(2)).to(dev)
    for n in (1, 64, few):
        for n_splits in (1, 2):
            got = attention_q4kv(q, codes, params, codes, params, lengths=n, n_splits=n_splits)
            assert torch.equal(got, attention_q4kv(q, *small, *small, lengths=n, n_splits=n_splits))
    # every other slot scores 0 and holds 0: cap - 2 few of them weigh 1 each
    q[0, 0, 0], q[0, 1] = 0, 6 * q[0, 1]  # (rows that weigh them, and rows that weigh the last slots)
    got = attention_q4kv(q, codes, params, codes, params, lengths=cap)[0].double().cpu().numpy()
    v, size = (t[0, 0] for t in O.values(small[0].cpu().numpy(), small[1].cpu().double().numpy()))
    x = q[0].double().cpu().numpy()
    for t in range(2):
        last = few - 1 + t  # row 0 does not see the last slot
        K, V, Vs = (np.concatenate([a, a[:last]]) for a in (v, v, size))
        score = x[t] @ K.T / 16
        w = np.exp(score - np.maximum(score.max(-1, keepdims=True), 0))
        rest = (cap - 1 + t - len(K)) * np.exp(-np.maximum(score.max(-1), 0))
        total = w.sum(-1) + rest
        # a score's two bounds (as the oracle's), and 2^28 sums, 128 splits of four waves of 16 lanes each:
        # 2^28 / (128 * 4 * 4) additions a lane at most, then 2^12
        rel = 2 * ((D + 24) * O.U + 2.0 ** -22) * (abs(x[t]) @ np.concatenate([size, size]).T / 16).max(-1) + (2.0 ** 17 + 2.0 ** 12) * O.U + 2.0 ** -19
        assert (abs(got[t] - w @ V / total[:, None]) <= rel[:, None] * (w @ Vs) / total[:, None] + 2.0 ** -24 * abs(got[t])).all()
    assert torch.equal(dequantize_kv_q4(codes[:, :, -few:], params[:, :, -few:]), dequantize_kv_q4(*small))
    del codes, params
    torch.cuda.empty_cache()
