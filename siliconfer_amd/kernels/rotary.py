"""Rotary positions given row by row: both pair layouts, part of the head, scaled
frequencies (the reference's RoPE is rotate-half over the whole head at one
offset, /root/reference/siliconfer/model/layers.py:58-66).

`rotary(q, k, positions, inv_freq)` turns q [B, T, H, D] and k [B, T, KVH, D] (k may
be None); any strides with contiguous dims. `qk_norm_rotary` norms each head by its root
mean square first, for models with a norm of queries and keys. `rotary_kv_append` turns
the q and k heads of fused q|k|v rows and quantizes k and v into the slots of an int8
cache, whose slots need not be the positions. `inv_freq` is the float64 angle a position of each
pair, on the device: `siliconfer_amd.model.rope.rotary_frequencies` makes it and the
`scale` that goes with it.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import SFError

__all__ = ["rotary", "qk_norm_rotary", "rotary_kv_append"]

_STRIDES = ctypes.c_longlong * 12
_STRIDES_BACK = ctypes.c_longlong * 18
_INT = (torch.int32, torch.int64)


def _positions(positions: torch.Tensor, B: int, T: int, x: torch.Tensor) -> tuple[bool, bool]:
    """(int64?, one row of positions a sequence?) of positions [B, T] or [T]."""
    dt, shape = positions.dtype, positions.shape
    if dt not in _INT or not positions.is_contiguous() or positions.get_device() != x.get_device():
        raise SFError("positions must be contiguous int32 or int64 on the rows' device")
    if shape != (B, T) and shape != (T,):
        raise SFError(f"positions must be [{B}, {T}] or [{T}] (got {list(shape)})")
    return dt is torch.int64, len(shape) == 2


def _pairs(inv_freq: torch.Tensor, D: int, x: torch.Tensor) -> int:
    if (inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous()
            or inv_freq.get_device() != x.get_device()):
        raise SFError("inv_freq must be a contiguous 1-D float64 tensor on the rows' device")
    n = inv_freq.shape[0]
    if not 0 < 2 * n <= D:
        raise SFError(f"{n} rotated pairs in a head of {D}")
    return n


def _rows(x: torch.Tensor, name: str) -> None:
    if not x.is_cuda:
        raise SFError(f"{name} must be a device tensor (got {x.device})")
    if x.dim() != 4:
        raise SFError(f"{name} must be [B, T, heads, head_dim]")
    if x.stride(3) != 1 and x.shape[3] != 1:
        raise SFError(f"{name}: a head's dims must be contiguous")


def _no_tangents(*tensors) -> None:
    """Raise for a tensor with a forward-mode tangent, which a kernel would drop."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise SFError("no forward-mode derivatives here: a tensor has a tangent")


def _forward_mode() -> bool:
    # (_current_level: asking each tensor costs a microsecond a call)
    return getattr(forward_ad, "_current_level", 0) >= 0


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
           interleaved: bool = False, scale: float = 1.0, out_q: torch.Tensor | None = None,
           out_k: torch.Tensor | None = None):
    """(q turned, k turned) at positions [B, T] or [T], in q's dtype. `out_q` /
    `out_k` may be the inputs themselves; other outputs must not overlap them, and
    inputs that need a gradient take none. Differentiable in q and k (in reverse mode)."""
    if _forward_mode():
        _no_tangents(q, k)
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        if out_q is not None or out_k is not None:
            raise SFError("rotary: inputs that need a gradient take no out_q / out_k")
        return _Turn.apply(q, k, positions, inv_freq, interleaved, scale)
    _rows(q, "q")
    B, T, H, D = q.shape
    KVH = 0
    if out_q is None:
        out_q = torch.empty_like(q, memory_format=torch.contiguous_format)
    plain = q.is_contiguous() and out_q.is_contiguous()
    if out_q.shape != q.shape or out_q.dtype != q.dtype or out_q.device != q.device:
        raise SFError("out_q must have q's shape, dtype and device")
    if k is not None:
        _rows(k, "k")
        KVH = k.shape[2]
        if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D or k.dtype != q.dtype or k.device != q.device:
            raise SFError("k must match q in batch, rows, head_dim, dtype and device")
        if out_k is None:
            out_k = torch.empty_like(k, memory_format=torch.contiguous_format)
        elif out_k.shape != k.shape or out_k.dtype != k.dtype or out_k.device != k.device:
            raise SFError("out_k must have k's shape, dtype and device")
        plain = plain and k.is_contiguous() and out_k.is_contiguous()
    elif out_k is not None:
        raise SFError("out_k without k")
    i64, per_seq = _positions(positions, B, T, q)
    pairs = _pairs(inv_freq, D, q)
    strides = None
    if not plain:
        for o in (out_q, out_k):
            if o is not None and any(st == 0 and n > 1 for st, n in zip(o.stride(), o.shape)):
                raise SFError("an output's rows must not share memory")
        _rows(out_q, "out_q")
        s = list(q.stride()[:3]) + list(out_q.stride()[:3])
        if k is not None:
            _rows(out_k, "out_k")
            s += list(k.stride()[:3]) + list(out_k.stride()[:3])
        strides = _STRIDES(*s)
    with _lib.on_device(q):
        rc = _lib.load().sf_rotary(q.data_ptr(), out_q.data_ptr(), None if k is None else k.data_ptr(),
                                   None if k is None else out_k.data_ptr(), _lib.dt(q), positions.data_ptr(), i64,
                                   per_seq, inv_freq.data_ptr(), pairs, scale, interleaved, B, T, H, KVH, D,
                                   strides, _lib.stream(q))
    if rc:
        _lib.check(rc, "sf_rotary")
    return out_q, out_k


class _Turn(torch.autograd.Function):
    """A turn by an angle is orthogonal but for its scale: the gradient is turned back by
    the same kernel, at the opposite positions. (Both run with gradients off.)"""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = dict(interleaved=interleaved, scale=scale)
        return rotary(q, k, positions, inv_freq, **ctx.how)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        positions, inv_freq = ctx.saved_tensors
        gq, gk = (g if g is None or g.stride(3) == 1 else g.contiguous() for g in (gq, gk))
        return (*rotary(gq, gk, -positions, inv_freq, **ctx.how), None, None, None, None)


def _side(x: torch.Tensor, w: torch.Tensor, out, name: str):
    """The output of one side's heads: `out`, checked, or a new tensor."""
    D = x.shape[3]
    if w.shape != (D,) or w.get_device() != x.get_device() or not w.is_contiguous():
        raise SFError(f"{name}_weight must be a contiguous [{D}] on {name}'s device (got {list(w.shape)} on {w.device})")
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise SFError(f"out_{name} must have {name}'s shape, dtype and device")
    _rows(out, f"out_{name}")
    if any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape)):
        raise SFError("an output's rows must not share memory")
    return out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
                   q_weight: torch.Tensor, k_weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                   interleaved: bool = False, scale: float = 1.0, out_q: torch.Tensor | None = None,
                   out_k: torch.Tensor | None = None):
    """(q, k), every head x of D dims normed, x / sqrt(mean(x^2) + eps) * weight ([D], one for
    q's heads and one for k's), then turned as `rotary` turns it, in one pass in fp32 and one
    rounding to q's dtype. D <= 256. `out_q` / `out_k` may be the inputs themselves; other
    outputs must not overlap them, and inputs that need a gradient take none. Differentiable
    in q, k and the weights (once, in reverse mode)."""
    if _forward_mode():
        _no_tangents(q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        if out_q is not None or out_k is not None:
            raise SFError("qk_norm_rotary: inputs that need a gradient take no out_q / out_k")
        return _NormTurn.apply(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, scale)
    _rows(q, "q")
    B, T, H, D = q.shape
    out_q = _side(q, q_weight, out_q, "q")
    plain, KVH = q.is_contiguous() and out_q.is_contiguous(), 0
    if k is not None:
        _rows(k, "k")
        KVH = k.shape[2]
        if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D or k.dtype != q.dtype or k.device != q.device:
            raise SFError("k must match q in batch, rows, head_dim, dtype and device")
        if k_weight is None or k_weight.dtype != q_weight.dtype:
            raise SFError("k needs a k_weight of q_weight's dtype")
        out_k = _side(k, k_weight, out_k, "k")
        plain = plain and k.is_contiguous() and out_k.is_contiguous()
    elif out_k is not None or k_weight is not None:
        raise SFError("out_k / k_weight without k")
    i64, per_seq = _positions(positions, B, T, q)
    pairs = _pairs(inv_freq, D, q)
    strides = None
    if not plain:
        strides = _STRIDES(*(t.stride(i) for t in (q, out_q, k, out_k) if t is not None for i in range(3)))
    with _lib.on_device(q):
        rc = _lib.load().sf_qk_norm_rotary(
            q.data_ptr(), out_q.data_ptr(), None if k is None else k.data_ptr(), None if k is None else out_k.data_ptr(),
            _lib.dt(q), q_weight.data_ptr(), None if k is None else k_weight.data_ptr(), _lib.dt(q_weight), eps,
            positions.data_ptr(), i64, per_seq, inv_freq.data_ptr(), pairs, scale, interleaved, B, T, H, KVH, D, strides,
            _lib.stream(q))
    if rc:
        _lib.check(rc, "sf_qk_norm_rotary")
    return out_q, out_k


@functools.lru_cache(maxsize=256)
def _norm_bytes(B: int, T: int, H: int, KVH: int, D: int) -> int:
    """sf_qk_norm_backward_workspace_bytes of a shape."""
    return int(_lib.load().sf_qk_norm_backward_workspace_bytes(B, T, H, KVH, D))


def _norm_turn_back(ctx, gq, gk):
    """The gradients of `_NormTurn`'s inputs."""
    q, k, positions, inv_freq, q_weight, k_weight = ctx.saved_tensors
    eps, interleaved, scale = ctx.how
    B, T, H, D = q.shape
    KVH = 0 if k is None else k.shape[2]
    if gq.stride(3) != 1:
        gq = gq.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dwq = torch.empty_like(q_weight)
    dk = dwk = None
    plain = q.is_contiguous() and gq.is_contiguous()
    if k is not None:
        if gk.stride(3) != 1:
            gk = gk.contiguous()
        dk = torch.empty_like(k, memory_format=torch.contiguous_format)
        dwk = torch.empty_like(dwq) if KVH else torch.zeros_like(dwq)
        plain = plain and k.is_contiguous() and gk.is_contiguous()
    if B * T == 0:
        dwq.zero_()
        if dwk is not None:
            dwk.zero_()
    else:
        strides = None
        if not plain:
            strides = _STRIDES_BACK(*(t.stride(i) for t in (q, gq, dq, k, gk, dk) if t is not None for i in range(3)))
        ptr = _lib.ptr
        with _lib.on_device(q):
            lib, st = _lib.load(), _lib.stream(q)
            ws = _lib.scratch(q.device, st, _norm_bytes(B, T, H, KVH, D))
            rc = lib.sf_qk_norm_rotary_backward(
                q.data_ptr(), gq.data_ptr(), dq.data_ptr(), ptr(k), ptr(gk if KVH else None), ptr(dk), _lib.dt(q),
                q_weight.data_ptr(), ptr(k_weight), _lib.dt(q_weight), dwq.data_ptr(), ptr(dwk), eps,
                positions.data_ptr(), positions.dtype is torch.int64, positions.dim() == 2, inv_freq.data_ptr(),
                inv_freq.shape[0], scale, interleaved, B, T, H, KVH, D, strides, ws.data_ptr(), ws.numel(), st)
        if rc:
            _lib.check(rc, "sf_qk_norm_rotary_backward")
    return dq, dk, None, None, dwq, dwk, None, None, None


# (where a graph of the gradients is asked for: it refuses to be differentiated)
_norm_turn_back_once = torch.autograd.function.once_differentiable(_norm_turn_back)


class _NormTurn(torch.autograd.Function):
    """`qk_norm_rotary` with its gradients, by one kernel that norms the saved rows again."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, scale):
        ctx.save_for_backward(q, k, positions, inv_freq, q_weight, k_weight)
        ctx.how = eps, interleaved, scale
        return qk_norm_rotary(q, k, positions, inv_freq, q_weight, k_weight, eps=eps, interleaved=interleaved,
                              scale=scale)

    @staticmethod
    def backward(ctx, gq, gk):
        # (once_differentiable's own checks cost 10 us a call)
        return (_norm_turn_back_once if torch.is_grad_enabled() else _norm_turn_back)(ctx, gq, gk)


def rotary_kv_append(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                     k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                     v_scales: torch.Tensor, *, n_heads: int, lengths, interleaved: bool = False,
                     scale: float = 1.0, slot_positions: torch.Tensor | None = None,
                     scores: torch.Tensor | None = None,
                     out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Append the T tokens of fused rows qkv [B, T, (H + 2 KVH) D] to the int8 cache
    (codes [B, KVH, T_cap, D], scales [B, KVH, T_cap]) at slots lengths[b] + t, keys
    turned to their positions, and return the turned q [B, T, H, D]. `lengths`: int32
    [B] on the device, or one int for every sequence; they are not changed. Device
    lengths are not checked against the capacity: a token past it is not stored."""
    _lib.require_device(qkv, "qkv")
    if qkv.dim() != 3 or k_codes.dim() != 4:
        raise SFError("qkv must be [B, T, width], k_codes / v_codes both [B, n_kv_heads, T, head_dim]")
    B, T, W = qkv.shape
    KVH, T_cap, D = k_codes.shape[1:]
    if k_codes.shape[0] != B or W != (n_heads + 2 * KVH) * D:
        raise SFError(f"qkv of width {W} does not match {n_heads} heads and a cache of {list(k_codes.shape)}")
    _lib.check_cache(qkv.device, k_codes, k_scales, v_codes, v_scales, slot_positions, scores)
    i64, per_seq = _positions(positions, B, T, qkv)
    pairs = _pairs(inv_freq, D, qkv)
    dev_len, start = _lib.lengths_arg(lengths, B, qkv.device)
    out = torch.empty((B, T, n_heads, D), dtype=out_dtype, device=qkv.device)
    with _lib.on_device(qkv):
        rc = _lib.load().sf_rotary_kv_append(
            qkv.data_ptr(), _lib.dt(qkv), positions.data_ptr(), i64, per_seq, inv_freq.data_ptr(), pairs, scale,
            interleaved, out.data_ptr(), _lib.dt(out), k_codes.data_ptr(), k_scales.data_ptr(),
            v_codes.data_ptr(), v_scales.data_ptr(), _lib.dt(k_scales),
            None if slot_positions is None else slot_positions.data_ptr(),
            None if scores is None else scores.data_ptr(), dev_len, start, B, T, n_heads, KVH, D, T_cap,
            _lib.stream(qkv))
    if rc:
        _lib.check(rc, "sf_rotary_kv_append")
    return out
