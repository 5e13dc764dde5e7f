"""Group-wise int8 KV cache on the device — the counterpart of the reference's
`siliconfer.model.kv_cache` (/root/reference/siliconfer/model/kv_cache.py:49-126).

Per (b, head, t) vector over head_dim: s = max|x| / 127 (1 if the vector is
zero), code = clip(rint(x / s), -128, 127), all in fp32 (kv_cache.py:59-63).
The reference grows its cache by concatenation every step and returns the
whole cache dequantized (kv_cache.py:99-105); here the codes go into a
preallocated buffer at the current length by one HIP kernel
(`sf_kv_quant_append`), and the fused decode attention reads them in place.
`update()` still returns the dequantized cache for callers that want the
reference's behaviour; `append()` skips that.

Scales are stored as fp16 by default (scale_dtype=torch.float32 keeps the
reference's fp32 scales).
"""

from __future__ import annotations

import torch

from .. import _lib
from .._lib import SFError


def _check_kv(k: torch.Tensor, v: torch.Tensor) -> None:
    for t, n in ((k, "k"), (v, "v")):
        _lib.require_device(t, n)
    if k.dim() != 4 or v.shape != k.shape:
        raise SFError("k and v must have the same shape")
    if k.dtype not in (torch.float16, torch.bfloat16, torch.float32) or v.dtype != k.dtype:
        raise SFError(f"unsupported KV dtype {k.dtype}")


def _append(k: torch.Tensor, v: torch.Tensor, qk, sk, qv, sv, t_off: int) -> None:
    _check_kv(k, v)
    B, KVH, Tn, D = k.shape
    T_cap = qk.shape[2]
    rc = _lib.load().sf_kv_quant_append(k.data_ptr(), v.data_ptr(), _lib.dt(k), qk.data_ptr(),
                                        sk.data_ptr(), qv.data_ptr(), sv.data_ptr(), _lib.dt(sk),
                                        B, KVH, Tn, t_off, T_cap, D, _lib.stream(k))
    _lib.check(rc, "sf_kv_quant_append")


def quantize_kv(x: torch.Tensor, scale_dtype: torch.dtype = torch.float32):
    """Symmetric int8 quantization, one scale per (b, head, token) vector.
    x [B, KVH, T, D] -> (codes int8 [B, KVH, T, D], scales [B, KVH, T, 1])."""
    x = x.contiguous()
    B, KVH, T, D = x.shape
    qk = torch.empty((B, KVH, T, D), dtype=torch.int8, device=x.device)
    sk = torch.empty((B, KVH, T), dtype=scale_dtype, device=x.device)
    # the append kernel quantizes K and V in one launch; quantize x as both
    qv = torch.empty_like(qk)
    sv = torch.empty_like(sk)
    _append(x, x, qk, sk, qv, sv, 0)
    return qk, sk.unsqueeze(-1)


def dequantize_kv(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float16):
    """Inverse of quantize_kv: q * scale, in `dtype`."""
    s = scale if scale.dim() == q.dim() else scale.unsqueeze(-1)
    return (q.float() * s.float()).to(dtype)


class QuantizedKVCache:
    """Per-layer int8 KV cache in preallocated device buffers.

    `capacity` is the maximum number of positions (grown by doubling if an
    update would overflow and `growable` is set). Buffers are allocated on the
    first update, when batch, heads, head_dim and device are known.
    """

    def __init__(self, capacity: int = 4096, scale_dtype: torch.dtype = torch.float16,
                 growable: bool = True) -> None:
        self.capacity = int(capacity)
        self.scale_dtype = scale_dtype
        self.growable = growable
        self._len = 0
        self._qk = self._sk = self._qv = self._sv = None

    # -- reference API ------------------------------------------------------
    def length(self) -> int:
        return self._len

    @property
    def q_k(self):
        return None if self._qk is None else self._qk[:, :, :self._len]

    @property
    def s_k(self):
        return None if self._sk is None else self._sk[:, :, :self._len].unsqueeze(-1)

    @property
    def q_v(self):
        return None if self._qv is None else self._qv[:, :, :self._len]

    @property
    def s_v(self):
        return None if self._sv is None else self._sv[:, :, :self._len].unsqueeze(-1)

    def update(self, k: torch.Tensor, v: torch.Tensor):
        """Quantize and append new (k, v) [B, KVH, T_new, D]; return the full
        dequantized cache in k's dtype (the reference's contract)."""
        self.append(k, v)
        return (dequantize_kv(self.q_k, self.s_k, k.dtype),
                dequantize_kv(self.q_v, self.s_v, k.dtype))

    def trim(self, n: int) -> None:
        """Keep the first n positions."""
        self._len = max(0, min(int(n), self._len))

    def nbytes(self) -> int:
        """Footprint of the valid prefix (codes + scales), as the reference reports it."""
        if self._qk is None:
            return 0
        B, KVH, _, D = self._qk.shape
        es = torch.empty((), dtype=self.scale_dtype).element_size()
        return 2 * B * KVH * self._len * (D + es)

    # -- device-resident fast path -------------------------------------------
    def reserve(self, B: int, KVH: int, D: int, need: int, device) -> None:
        """Make the buffers hold at least `need` positions of [B, KVH, *, D]
        (allocating them on first use) without appending anything."""
        self._ensure(torch.empty((B, KVH, 0, D), device=device), need)

    def set_length(self, n: int) -> None:
        """Mark the first n positions valid (a kernel wrote them in place)."""
        if self._qk is None or not 0 <= n <= self._qk.shape[2]:
            raise SFError(f"length {n} outside the cache's buffers")
        self._len = int(n)

    def _ensure(self, k: torch.Tensor, need: int) -> None:
        B, KVH, _, D = k.shape
        if self._qk is not None:
            if self._qk.shape[0] != B or self._qk.shape[1] != KVH or self._qk.shape[3] != D:
                raise SFError("KV cache shape changed between updates")
            if need <= self._qk.shape[2]:
                return
            if not self.growable:
                raise SFError(f"KV cache overflow: {need} > capacity {self._qk.shape[2]}")
        cap = max(self.capacity, 1)
        while cap < need:
            cap *= 2
        qk = torch.empty((B, KVH, cap, D), dtype=torch.int8, device=k.device)
        sk = torch.empty((B, KVH, cap), dtype=self.scale_dtype, device=k.device)
        qv, sv = torch.empty_like(qk), torch.empty_like(sk)
        if self._qk is not None and self._len:
            qk[:, :, :self._len].copy_(self._qk[:, :, :self._len])
            sk[:, :, :self._len].copy_(self._sk[:, :, :self._len])
            qv[:, :, :self._len].copy_(self._qv[:, :, :self._len])
            sv[:, :, :self._len].copy_(self._sv[:, :, :self._len])
        self._qk, self._sk, self._qv, self._sv = qk, sk, qv, sv
        self.capacity = cap

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantize new (k, v) straight into the buffers at the current length."""
        k = k.contiguous()
        v = v.contiguous()
        _check_kv(k, v)  # (before any buffer is made for them)
        self._ensure(k, self._len + k.shape[2])
        _append(k, v, self._qk, self._sk, self._qv, self._sv, self._len)
        self._len += k.shape[2]

    def buffers(self):
        """(k_codes, k_scales, v_codes, v_scales) full-capacity buffers."""
        return self._qk, self._sk, self._qv, self._sv


def make_quantized_cache(n_layers: int, capacity: int = 4096,
                         scale_dtype: torch.dtype = torch.float16) -> list[QuantizedKVCache]:
    """One fresh QuantizedKVCache per transformer layer."""
    return [QuantizedKVCache(capacity, scale_dtype) for _ in range(n_layers)]


class BoundedKVCache(QuantizedKVCache):
    """An int8 cache that keeps at most `budget` tokens a kv head: it counts the
    attention weight that every slot receives (`scores`) and, once it holds more than
    budget + slack, drops the slots with the least of it; those of the newest `recent`
    tokens (a quarter of the budget by default) stay. Each kv head keeps tokens of its
    own, in any order, with their `positions`; `length()` counts slots, `seen` the
    tokens that went through. Keys are cached turned to their positions. The buffers have
    budget + slack + 1 slots; for a longer prompt (or by `reserve`) they grow, until
    `release` or the first append after a cut that fits those again."""

    def __init__(self, budget: int, recent: int | None = None, slack: int = 64,
                 scale_dtype: torch.dtype = torch.float16) -> None:
        recent = budget // 4 if recent is None else recent
        if not (budget > 0 and 0 <= recent <= budget and slack >= 0):
            raise SFError(f"need budget > 0, 0 <= recent <= budget, slack >= 0 (got {budget}, {recent}, {slack})")
        super().__init__(budget + slack + 1, scale_dtype)
        self.budget, self.recent, self.slack = int(budget), int(recent), int(slack)
        self.seen = 0
        self.scores = self.positions = None
        self._cut = False  # shortened since the buffers were last asked to hold more than the bound

    def _ensure(self, k: torch.Tensor, need: int) -> None:
        if need > self.budget + self.slack + 1:
            self._cut = False
        elif self._cut:
            self.release()
        before = self._qk
        super()._ensure(k, need)
        if self._qk is before:
            return
        shape = self._qk.shape[:3]
        scores = torch.zeros(shape, dtype=torch.float32, device=self._qk.device)
        positions = torch.zeros(shape, dtype=torch.int32, device=self._qk.device)
        if self.scores is not None and self._len:
            scores[:, :, :self._len].copy_(self.scores[:, :, :self._len])
            positions[:, :, :self._len].copy_(self.positions[:, :, :self._len])
        self.scores, self.positions = scores, positions

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Append keys that are turned already, and values, [B, KVH, T, D]."""
        n, T = self._len, k.shape[2]
        super().append(k, v)
        self.scores[:, :, n:n + T] = 0
        self.positions[:, :, n:n + T] = torch.arange(self.seen, self.seen + T, dtype=torch.int32, device=k.device)
        self.seen += T

    def append_rotary(self, qkv: torch.Tensor, n_heads: int, n_kv_heads: int, rotary,
                      out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Append the next tokens' fused q|k|v rows [B, T, (H + 2 KVH) D], keys turned to
        their positions; returns the turned q [B, T, H, D]."""
        from ..kernels.rotary import rotary_kv_append
        _lib.require_device(qkv, "qkv")  # (all before any buffer is made for the rows)
        B, T, W = qkv.shape if qkv.dim() == 3 else (0, 0, 0)
        D = W // (n_heads + 2 * n_kv_heads) if n_heads > 0 and n_kv_heads > 0 and n_heads % n_kv_heads == 0 else 0
        if D == 0 or D % 8 or D > 256 or W != (n_heads + 2 * n_kv_heads) * D:
            raise SFError(f"qkv {list(qkv.shape)} does not hold {n_heads} and 2 x {n_kv_heads} heads of a multiple of 8 "
                          "dims up to 256")
        self.reserve(B, n_kv_heads, D, self._len + T, qkv.device)
        positions = torch.arange(self.seen, self.seen + T, dtype=torch.int32, device=qkv.device)
        q = rotary_kv_append(qkv, positions, rotary.on(qkv.device), *self.buffers(), n_heads=n_heads,
                             lengths=self._len, interleaved=rotary.interleaved, scale=rotary.scale,
                             slot_positions=self.positions, scores=self.scores, out_dtype=out_dtype)
        self._len += T
        self.seen += T
        return q

    def attend(self, q: torch.Tensor, scale: float | None = None) -> torch.Tensor:
        """Attention of the newest rows q [B, T, H, D] (T <= 32) over the cache, their
        weights added to the scores; fp32."""
        from ..kernels.attention import attention_decode_scored
        return attention_decode_scored(q, *self.buffers(), self.scores, lengths=self._len, scale=scale)

    def evict(self) -> None:
        """Cut the cache to its budget where it holds more than budget + slack."""
        from ..kernels.eviction import evict
        if self._len > self.budget + self.slack:
            evict(*self.buffers(), self.scores, self.positions, self._len, self.seen, self.budget, self.recent)
            self._len = self.budget
            self._cut = True

    def release(self) -> None:
        """Let buffers that grew for a prompt go back to budget + slack + 1 slots, if what is
        kept fits them."""
        base, n = self.budget + self.slack + 1, self._len
        if self._qk is None or self._qk.shape[2] <= base or n > base:
            return
        old = (*self.buffers(), self.scores, self.positions)
        new = [t.new_zeros((*t.shape[:2], base, *t.shape[3:])) for t in old]
        for a, b in zip(new, old):
            a[:, :, :n].copy_(b[:, :, :n])
        self._qk, self._sk, self._qv, self._sv, self.scores, self.positions = new
        self.capacity = base
        self._cut = False

    def nbytes(self) -> int:
        """Footprint of the valid slots: codes, scales, scores and positions."""
        rows = 0 if self._qk is None else self._qk.shape[0] * self._qk.shape[1] * self._len
        return super().nbytes() + 8 * rows

    def set_length(self, n: int) -> None:
        raise SFError("a bounded cache's slots are set by append and evict")

    def trim(self, n: int) -> None:
        """Keep the first n positions; once tokens were dropped all or none of them.
        The scores keep what the rows behind them added."""
        if self.seen != self._len and 0 < n < self.seen:
            raise SFError("a bounded cache that dropped tokens cannot be trimmed")
        super().trim(n)
        self.seen = min(self.seen, max(0, int(n)))
        self._cut = True
