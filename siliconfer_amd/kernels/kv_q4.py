"""A KV cache held in 4 bits: append, reading back, and attention over it.

Beside the int8 cache (one scale a token and head; the reference has that one only,
/root/reference/siliconfer/model/kv_cache.py:49-126), each group of `group` dims is held as
codes 0..15 with a scale s and a minimum m in fp16: x is m + s code, m = min x,
s = (max x - min x) / 15, the code rint((x - m) / s). A buffer pair is

  codes   uint8 [B, KVH, T_cap, D / 2], the even dim of two in the low half of a byte
  params  fp16 [B, KVH, T_cap, D / group, 2], (s, m) a group

with D a multiple of 16 up to 256 and group 32, 64, 128 (dividing D) or D itself. A minimum or a
scale past fp16's range is held at its end; a group with a value that is not finite reads back as NaN.
Keys are cached turned to their positions. Nothing here is differentiable.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .._lib import SFError
from .rotary import _pairs, _positions

__all__ = ["kv_append_q4", "rotary_kv_append_q4", "dequantize_kv_q4", "attention_q4kv"]

_STRIDES9 = ctypes.c_longlong * 9
_STRIDES6 = ctypes.c_longlong * 6


def _check(device: torch.device, k_codes, k_params, v_codes, v_params) -> tuple:
    """(B, KVH, T_cap, D, group) of a cache's buffers, all contiguous on `device`."""
    at, u8, f16 = device.index, torch.uint8, torch.float16
    cs, ps = k_codes.shape, k_params.shape
    if not (len(cs) == 4 and len(ps) == 5 and k_codes.get_device() == v_codes.get_device() == k_params.get_device()
            == v_params.get_device() == at and k_codes.dtype is u8 and v_codes.dtype is u8 and k_params.dtype is f16
            and v_params.dtype is f16 and v_codes.shape == cs and v_params.shape == ps and ps[:3] == cs[:3] and ps[4] == 2
            and ps[3] > 0 and 2 * cs[3] % ps[3] == 0 and k_codes.is_contiguous() and v_codes.is_contiguous()
            and k_params.is_contiguous() and v_params.is_contiguous()):
        raise SFError("k/v codes must be uint8 [B, n_kv_heads, T, head_dim / 2] and k/v params float16 [B, n_kv_heads, "
                      f"T, groups, 2], all contiguous on {device} (got {k_codes.dtype} {list(cs)}, {v_codes.dtype} "
                      f"{list(v_codes.shape)}, {k_params.dtype} {list(ps)}, {v_params.dtype} {list(v_params.shape)})")
    return cs[0], cs[1], cs[2], 2 * cs[3], 2 * cs[3] // ps[3]


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x [.., heads, .., D] as it is where rows of 8 dims can be loaded whole, else a copy."""
    s = x.stride()
    if s[3] == 1 and not (s[0] % 8 or s[1] % 8 or s[2] % 8) and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def kv_append_q4(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_params: torch.Tensor,
                 v_codes: torch.Tensor, v_params: torch.Tensor, *, lengths) -> None:
    """Append k (turned already) and v [B, KVH, T, D], any strides, at slots lengths[b] + t.
    `lengths`: int32 [B] on the device, or one int for every sequence; they are not changed.
    Device lengths are not checked against the capacity: a token past it is not stored."""
    if not k.is_cuda or not v.is_cuda or k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise SFError("k and v must be device tensors of the same shape [B, n_kv_heads, T, head_dim] and dtype")
    B, KVH, T, D = k.shape
    Bc, KVHc, T_cap, Dc, g = _check(k.device, k_codes, k_params, v_codes, v_params)
    if (Bc, KVHc, Dc) != (B, KVH, D):
        raise SFError(f"k / v {list(k.shape)} do not match a cache of {Bc} x {KVHc} heads of {Dc}")
    dev_len, start = _lib.lengths_arg(lengths, B, k.device)
    k, v = _aligned(k), _aligned(v)
    (kb, kh, kt, _), (vb, vh, vt, _) = k.stride(), v.stride()
    with _lib.on_device(k):
        rc = _lib.load().sf_kv_q4_append(
            None, k.data_ptr(), v.data_ptr(), _lib.dt(k), _STRIDES9(0, 0, 0, kb, kt, kh, vb, vt, vh), None, None, 0, 0.0,
            None, 0, 0, None, 0, 1.0, 0, None, 0, k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(),
            v_params.data_ptr(), g, dev_len, start, B, T, 0, KVH, D, T_cap, _lib.stream(k))
    if rc:
        _lib.check(rc, "sf_kv_q4_append")


def rotary_kv_append_q4(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, k_codes: torch.Tensor,
                        k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor, *, n_heads: int,
                        lengths, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                        eps: float = 1e-6, interleaved: bool = False, scale: float = 1.0,
                        out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Append the T tokens of fused rows qkv [B, T, (H + 2 KVH) D] to a 4-bit cache at slots
    lengths[b] + t and return the turned q [B, T, H, D]. q and k turn to their positions
    ([B, T] or [T]) as in `rotary`; with `q_weight` / `k_weight` ([D]) each of their heads is
    normed first, as in `qk_norm_rotary`. `lengths` as in `kv_append_q4`."""
    _lib.require_device(qkv, "qkv")
    if qkv.dim() != 3:
        raise SFError("qkv must be [B, T, width]")
    B, T, W = qkv.shape
    Bc, KVH, T_cap, D, g = _check(qkv.device, k_codes, k_params, v_codes, v_params)
    if Bc != B or n_heads <= 0 or W != (n_heads + 2 * KVH) * D:
        raise SFError(f"qkv {list(qkv.shape)} does not match {n_heads} heads and a cache of {Bc} x {KVH} heads of {D}")
    i64, per_seq = _positions(positions, B, T, qkv)
    pairs = _pairs(inv_freq, D, qkv)
    wdt = 0
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            if w.shape != (D,) or w.device != qkv.device or not w.is_contiguous():
                raise SFError(f"{name} must be a contiguous [{D}] on the rows' device")
            wdt = _lib.dt(w)
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise SFError("q_weight and k_weight must have one dtype")
    dev_len, start = _lib.lengths_arg(lengths, B, qkv.device)
    if qkv.data_ptr() % 16:
        qkv = qkv.clone()
    out = torch.empty((B, T, n_heads, D), dtype=out_dtype, device=qkv.device)
    at, row, size = qkv.data_ptr(), T * W, qkv.element_size()
    with _lib.on_device(qkv):
        rc = _lib.load().sf_kv_q4_append(
            at, at + n_heads * D * size, at + (n_heads + KVH) * D * size, _lib.dt(qkv),
            _STRIDES9(row, W, D, row, W, D, row, W, D), _lib.ptr(q_weight), _lib.ptr(k_weight), wdt, eps,
            positions.data_ptr(), i64, per_seq, inv_freq.data_ptr(), pairs, scale, interleaved, out.data_ptr(),
            _lib.dt(out), k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(), g, dev_len,
            start, B, T, n_heads, KVH, D, T_cap, _lib.stream(qkv))
    if rc:
        _lib.check(rc, "sf_kv_q4_append")
    return out


def dequantize_kv_q4(codes: torch.Tensor, params: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [B, KVH, T, D] that codes [B, KVH, T, D / 2] and params [B, KVH, T, D / group,
    2] stand for: a cache's buffers, or their slots from .. to (views [:, :, a:b])."""
    if not codes.is_cuda or params.get_device() != codes.get_device():
        raise SFError("codes and params must be on one device")
    cs, ps = codes.shape, params.shape
    if (codes.dtype is not torch.uint8 or params.dtype is not torch.float16 or len(cs) != 4 or len(ps) != 5
            or ps[:3] != cs[:3] or ps[4] != 2 or ps[3] == 0 or 2 * cs[3] % ps[3]):
        raise SFError("codes must be uint8 [B, n_kv_heads, T, head_dim / 2], params float16 [B, n_kv_heads, T, groups, 2]")
    if codes.stride(3) != 1 or params.stride(4) != 1 or params.stride(3) != 2:
        raise SFError("a token's codes and params must be contiguous")
    B, KVH, T, D = cs[0], cs[1], cs[2], 2 * cs[3]
    out = torch.empty((B, KVH, T, D), dtype=dtype, device=codes.device)
    with _lib.on_device(codes):
        rc = _lib.load().sf_kv_q4_dequant(codes.data_ptr(), params.data_ptr(), out.data_ptr(), _lib.dt(out), D // ps[3],
                                          _STRIDES6(*codes.stride()[:3], *params.stride()[:3]), B, KVH, T, D,
                                          _lib.stream(codes))
    if rc:
        _lib.check(rc, "sf_kv_q4_dequant")
    return out


@functools.lru_cache(maxsize=256)
def _attention_bytes(B: int, Tq: int, H: int, KVH: int, T_max: int, D: int, g: int, dt: int, out: int,
                     n: int) -> int:
    """sf_attn_q4_workspace_bytes of a shape."""
    return int(_lib.load().sf_attn_q4_workspace_bytes(B, Tq, H, KVH, T_max, D, g, dt, out, n))


def attention_q4kv(q: torch.Tensor, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
                   v_params: torch.Tensor, *, lengths, add: int = 0, max_length: int | None = None,
                   n_splits: int | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Attention of q [B, H, D], or of the Tq newest rows q [B, Tq, H, D], over the first
    lengths[b] + add slots of a 4-bit cache: softmax(scale q K^T) V in fp32 sums, one rounding
    to the output's dtype, factors held to 2^-22. (Where rows are many, and q has 16 bits, a bf16
    output is made of weights, K and V rounded to fp16: 2^-11 of each, and of a weight by K's
    rounding up to 2^-11 of scale sum |q K|.) Row t of Tq sees the slots up to its own, lengths[b] + add - Tq + t;
    a row that sees none gives zeros. `lengths`: int32 [B] on the device, or one int. Device
    lengths are cut to `max_length` (the capacity where it is not given). `n_splits`: among how
    many workgroups a sequence's slots are shared out where rows are few (its own choice by
    default)."""
    n = n_splits or 0
    if not (_lib.INT_MIN <= add <= _lib.INT_MAX and _lib.INT_MIN <= n <= _lib.INT_MAX
            and _lib.INT_MIN <= (max_length or 0) <= _lib.INT_MAX):
        _lib.refuse_int(add=add, n_splits=n, max_length=max_length)
    three = q.dim() == 3
    if not three and q.dim() != 4:
        raise SFError("q must be [B, n_heads, head_dim] or [B, rows, n_heads, head_dim]")
    _lib.require_device(q, "q")
    B, H, D = q.shape[0], q.shape[-2], q.shape[-1]
    Tq = 1 if three else q.shape[1]
    Bc, KVH, T_cap, Dc, g = _check(q.device, k_codes, k_params, v_codes, v_params)
    if Bc != B or Dc != D:
        raise SFError("cache shape does not match q")
    dev_len, T = _lib.lengths_arg(lengths, B, q.device)
    T += add
    T_max = T_cap if max_length is None else max_length
    if dev_len is None:
        if T > T_max:
            raise SFError(f"{T} slots of a cache of {T_max}")
        T_max = T
    if q.data_ptr() % 16:
        q = q.clone()
    if out is None:
        out = torch.empty_like(q, dtype=out_dtype)
    elif out.shape != q.shape or out.device != q.device or not out.is_contiguous():
        raise SFError("out must be contiguous, of q's shape and on its device")
    elif out.data_ptr() % 16:
        return out.copy_(attention_q4kv(q, k_codes, k_params, v_codes, v_params, lengths=lengths, add=add,
                                        max_length=max_length, n_splits=n_splits, scale=scale, out_dtype=out.dtype))
    lib = _lib.load()
    with _lib.on_device(q):
        st = _lib.stream(q)
        need = _attention_bytes(B, Tq, H, KVH, T_max, D, g, _lib.dt(q), _lib.dt(out), n)
        ws = _lib.scratch(q.device, st, need) if need else None
        rc = lib.sf_attn_q4kv(
            q.data_ptr(), _lib.dt(q), k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(), g,
            out.data_ptr(), _lib.dt(out), None if ws is None else ws.data_ptr(), need, B, Tq, H, KVH, dev_len, T, T_max,
            T_cap, D, D ** -0.5 if scale is None else scale, n, st)
    if rc:
        _lib.check(rc, "sf_attn_q4kv")
    return out
