"""What the 4-bit cache and the heads' norm make of ties, constants, ranges and values that are no
numbers: values as keys, and an infinity in a head."""

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd.kernels.kv_q4 import dequantize_kv_q4, kv_append_q4, rotary_kv_append_q4
from siliconfer_amd.kernels.rotary import qk_norm_rotary

pytestmark = pytest.mark.gpu


def empty(KVH, cap, D, group, dev, codes, params):
    return [t for _ in range(2) for t in (torch.full((1, KVH, cap, D // 2), codes, dtype=torch.uint8, device=dev),
                                          torch.full((1, KVH, cap, D // group, 2), params, dtype=torch.float16, device=dev))]


def test_values_as_keys(dev):
    """V's codes and parameters are the oracle's where K holds other rows, and slots that were not
    written keep what was there."""
    x = torch.randn(1, 1, 7, 64, generator=torch.Generator().manual_seed(0)).to(dev)
    x[0, 0, 1, :31] = torch.arange(31, device=dev).float() * 0.5  # 0 .. 15: s = 1, every half a tie
    x[0, 0, 1, 31] = 0
    x[0, 0, 2] = 2.5
    x[0, 0, 3, 0], x[0, 0, 3, 1] = 1e30, -1e30
    x[0, 0, 4, 40] = float("nan")
    x[0, 0, 5, 3] = float("-inf")
    x[0, 0, 6] = 1e-12 * torch.arange(64, device=dev)
    k = torch.randn(1, 1, 7, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    for first, second in ((k, x), (x, k)):
        kc, kp, vc, vp = empty(1, 9, 64, 32, dev, 0xA5, 3.0)
        kv_append_q4(first, second, kc, kp, vc, vp, lengths=1)
        for c, p, y in ((kc, kp, first), (vc, vp, second)):
            codes, s, m, _ = O.quantize(y.double().cpu().numpy(), 32)
            assert torch.equal(c[:, :, 1:8].cpu(), torch.from_numpy(O.pack(codes)))
            assert np.array_equal(p[:, :, 1:8].cpu().numpy(), np.stack([s, m], -1), equal_nan=True)
            assert (c[:, :, ::8] == 0xA5).all() and (p[:, :, ::8] == 3).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinity_in_a_head(dev, dtype):
    """Its root mean square is infinite, so that the head's other dims come to 0 and the infinite one,
    and its partner in the turn, to NaN; cached, the groups of these two read back as NaN."""
    H, KVH, D, T = 2, 2, 64, 2
    x = torch.randn(1, T, H + 2 * KVH, D, generator=torch.Generator().manual_seed(2)).to(dev, dtype)
    clean = x.clone()
    x[0, 1, 0, 5] = x[0, 1, H, 5] = float("inf")  # of a q head and of a k head
    w = torch.ones(D, device=dev)
    pos, f = torch.tensor([3, 4], dtype=torch.int32, device=dev), torch.from_numpy(1e4 ** (-np.arange(32) / 32.0)).to(dev)
    for interleaved, partner in ((False, 37), (True, 4)):
        how = dict(interleaved=interleaved)
        for at in (0, H):
            y, want = (qk_norm_rotary(t[:, :, at:at + 2], None, pos, f, w, **how)[0] for t in (x, clean))
            none = torch.zeros(D, dtype=torch.bool, device=dev)
            none[[5, partner]] = True
            assert torch.equal(y[0, 1, 0].isnan(), none) and (y[0, 1, 0][~none] == 0).all()
            assert torch.equal(y[:, :, 1], want[:, :, 1]) and torch.equal(y[:, 0], want[:, 0])
        bufs = empty(KVH, 4, D, 32, dev, 0, 0.0)
        q = rotary_kv_append_q4(x.reshape(1, T, -1), pos, f, *bufs, n_heads=H, lengths=1, q_weight=w, k_weight=w, **how)
        assert torch.equal(q[0, 1, 0].isnan(), none) and (q[0, 1, 0][~none] == 0).all() and q[0, 1, 1].isfinite().all()
        k = dequantize_kv_q4(*bufs[:2])[0]
        for g in range(2):
            part = k[0, 2, 32 * g:32 * g + 32]
            assert part.isnan().all() if none[32 * g:32 * g + 32].any() else (part == 0).all()
        assert k[1].isfinite().all() and k[0, 1].isfinite().all() and dequantize_kv_q4(*bufs[2:]).isfinite().all()
