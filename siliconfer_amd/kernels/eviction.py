"""Eviction from an int8 KV cache by accumulated attention weight.

`evict(...)` cuts every sequence's cache to `budget` slots a kv head: the slots of the
newest `recent` tokens stay, then those with the largest scores
(`attention_decode_scored` accumulates them). The kept slots behind the budget move
into the holes below it, in place; attention does not depend on the slots' order,
since keys are rotated before they are cached.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._lib import SFError

__all__ = ["evict"]


def evict(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
          scores: torch.Tensor, positions: torch.Tensor, lengths, seen, budget: int,
          recent: int = 0) -> torch.Tensor:
    """Cut the cache (codes [B, KVH, T_cap, D], scales, fp32 scores and int32
    positions [B, KVH, T_cap]) to its `budget` best slots and return the new lengths,
    int32 [B]: min(length, budget). `lengths` and `seen` (the tokens each sequence has
    had so far): int32 [B] on the device, or one int for all. Slots at and past the
    new length are left as they were."""
    if not (_lib.INT_MIN <= budget <= _lib.INT_MAX and _lib.INT_MIN <= recent <= _lib.INT_MAX):
        _lib.refuse_int(budget=budget, recent=recent)
    _lib.require_device(k_codes, "k_codes")
    if k_codes.dim() != 4:
        raise SFError("k_codes / v_codes must both be [B, n_kv_heads, T, head_dim]")
    B, KVH, T_cap, D = k_codes.shape
    _lib.check_cache(k_codes.device, k_codes, k_scales, v_codes, v_scales, positions, scores)
    dev_len, T = _lib.lengths_arg(lengths, B, k_codes.device)
    dev_seen, seen_host = _lib.lengths_arg(seen, B, k_codes.device, "seen")
    lib = _lib.load()
    out = torch.empty((B,), dtype=torch.int32, device=k_codes.device)
    with _lib.on_device(k_codes):
        st = _lib.stream(k_codes)
        ws = _lib.scratch(k_codes.device, st, lib.sf_kv_evict_workspace_bytes(
            B, KVH, budget, T_cap if dev_len else T))
        rc = lib.sf_kv_evict(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                             _lib.dt(k_scales), scores.data_ptr(), positions.data_ptr(), dev_len, T, dev_seen,
                             seen_host, budget, recent, out.data_ptr(), ws.data_ptr(), ws.numel(), B, KVH, T_cap,
                             D, st)
    if rc:
        _lib.check(rc, "sf_kv_evict")
    return out
