"""Drawing a token a row on the device, from random numbers that the caller gives.

The rules are `engine.generate.sample_token`'s (the reference's temperature, top-k and
top-p, /root/reference/siliconfer/engine/generate.py:24-67) and min-p, with the draw
taken in descending order of the logits: the token is the first whose running weight
exceeds u times the weight that the filters leave. Nothing returns to the host.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._lib import SFError

__all__ = ["sample"]


def _setting(v, name: str, B: int, dtype: torch.dtype, device) -> tuple[float, int | None]:
    """(value for every row, device pointer of a value a row or None)."""
    if not isinstance(v, torch.Tensor):
        return v, None
    if v.dtype != dtype or v.shape != (B,) or v.device != device or not v.is_contiguous():
        raise SFError(f"{name}: a number, or a contiguous {dtype} tensor [{B}] on the logits' device")
    return (0 if dtype is torch.int32 else 1.0), v.data_ptr()


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *,
           logprobs: bool = False, out: torch.Tensor | None = None,
           at: torch.Tensor | None = None, at_add: int = 0, hist: torch.Tensor | None = None):
    """int32 tokens [B] drawn from logits [B, V] (fp32, fp16 or bf16; a row's logits
    contiguous) with the numbers u, fp32 [B] in [0, 1); with `logprobs` (tokens, the log
    of each token's share of the weight kept, fp32 [B]). Each setting is one number, or
    a tensor [B] of every row's own (fp32; int32 for top_k): temperature <= 0 takes the
    largest logit, top_k 0, top_p 1 and min_p 0 keep every token. A row with no logit
    above -inf gives -1. For steps replayed from a graph, `at`, int32 [1] on the device,
    counts the steps: u then holds every step's numbers (fp32 [n], n >= B), row b takes
    u[at + at_add + b], and its token also goes to the same place of `hist`, int32 [n]."""
    k = 0 if isinstance(top_k, torch.Tensor) else top_k
    if not (_lib.INT_MIN <= at_add <= _lib.INT_MAX and _lib.INT_MIN <= k <= _lib.INT_MAX):
        _lib.refuse_int(top_k=top_k, at_add=at_add)
    if not logits.is_cuda:
        raise SFError(f"logits must be a device tensor (got {logits.device})")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise SFError("logits must be [B, V] with contiguous rows")
    B, V = logits.shape
    dev = logits.device
    n = u.shape[0] if u.dim() == 1 else -1
    if u.dtype is not torch.float32 or (n != B if at is None else n < B) or u.device != dev or not u.is_contiguous():
        raise SFError(f"u must be a contiguous float32 tensor [{B}] on the logits' device")
    if at is not None and (at.dtype is not torch.int32 or at.numel() != 1 or at.device != dev):
        raise SFError("at must be one int32 on the logits' device")
    if hist is not None and (at is None or hist.dtype is not torch.int32 or hist.shape != u.shape
                             or hist.device != dev or not hist.is_contiguous()):
        raise SFError("hist goes with at: a contiguous int32 tensor as long as u on the logits' device")
    t, tp = _setting(temperature, "temperature", B, torch.float32, dev)
    k, kp = _setting(top_k, "top_k", B, torch.int32, dev)
    p, pp = _setting(top_p, "top_p", B, torch.float32, dev)
    m, mp = _setting(min_p, "min_p", B, torch.float32, dev)
    if out is None:
        out = torch.empty((B,), dtype=torch.int32, device=dev)
    elif out.dtype is not torch.int32 or out.shape != (B,) or out.device != dev or not out.is_contiguous():
        raise SFError(f"out must be a contiguous int32 tensor [{B}] on the logits' device")
    lp = torch.empty((B,), dtype=torch.float32, device=dev) if logprobs else None
    lib = _lib.load()
    with _lib.on_device(logits):
        st = _lib.stream(logits)
        need = lib.sf_sample_workspace_bytes(B, V)
        ws = _lib.scratch(dev, st, need) if need else None
        rc = lib.sf_sample(logits.data_ptr(), _lib.dt(logits), logits.stride(0), B, V, u.data_ptr(), t, k, p, m, tp,
                           kp, pp, mp, out.data_ptr(), None if lp is None else lp.data_ptr(),
                           None if at is None else at.data_ptr(), at_add, n,
                           None if hist is None else hist.data_ptr(),
                           None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), st)
    if rc:
        _lib.check(rc, "sf_sample")
    return (out, lp) if logprobs else out
