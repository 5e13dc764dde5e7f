"""An append that a 4-bit cache refuses leaves nothing behind."""

import pytest
import torch

from siliconfer_amd._lib import SFError
from siliconfer_amd.model import Q4KVCache, Rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_a_refused_append(dev):
    """Weights, outputs and turns that do not fit, at the first append and at one that would grow the
    buffers: no buffers are made, and those that were there stay."""
    H, KVH, D = 4, 2, 64
    r, wide = (Rotary(*rotary_frequencies(n, 1e4)) for n in (64, 128))
    qkv = torch.randn(2, 3, (H + 2 * KVH) * D, generator=torch.Generator().manual_seed(0)).to(dev)
    w = torch.ones(D, device=dev)
    bad = [dict(rotary=r, q_weight=w[:32]), dict(rotary=r, q_weight=w, k_weight=w.half()), dict(rotary=wide),
           dict(rotary=r, out_dtype=torch.int32), dict(rotary=r, q_weight=w.double())]
    cache = Q4KVCache(4)
    for kw in bad:
        with pytest.raises(SFError):
            cache.append_rotary(qkv, H, KVH, **kw)
        assert cache.buffers() == (None,) * 4 and cache.capacity == 4 and cache.length() == 0
    want = cache.append_rotary(qkv, H, KVH, r)
    before, copies = cache.buffers(), [t.clone() for t in cache.buffers()]
    for kw in bad:
        with pytest.raises(SFError):
            cache.append_rotary(qkv, H, KVH, **kw)
        assert all(a is b for a, b in zip(cache.buffers(), before)) and cache.capacity == 4 and cache.length() == 3
    assert all(torch.equal(a[:, :, :3], b[:, :, :3]) for a, b in zip(before, copies))
    assert torch.equal(Q4KVCache(4).append_rotary(qkv, H, KVH, r), want)
    cache.append_rotary(qkv, H, KVH, r)
    assert cache.length() == 6 and cache.capacity == 8
