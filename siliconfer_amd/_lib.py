"""ctypes binding of libsiliconfer_hip.so (the C ABI in include/siliconfer_hip.h).

torch is imported first so that the library binds to the HIP runtime torch has
already loaded (both are libamdhip64.so.7); device pointers and streams then
come straight from torch tensors.

There is no CPU fallback anywhere in siliconfer_amd: every compute call goes
through this library and raises if it cannot be loaded or no gfx950 device is
present.
"""

from __future__ import annotations

import contextlib
import ctypes
import os
import threading

import torch

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libsiliconfer_hip.so")

SF_F32, SF_F16, SF_BF16 = 0, 1, 2
SF_PRE_RMSNORM, SF_PRE_SILU_MUL = 1, 2
SF_GROUP_CONCAT, SF_GROUP_SWIGLU = 0, 1
SF_CHAIN_IN_X0, SF_CHAIN_IN_PREV, SF_CHAIN_IN_SWIGLU = 0, 1, 2
SF_CHAIN_MAX_PHASES = 8
_DT = {torch.float32: SF_F32, torch.float16: SF_F16, torch.bfloat16: SF_BF16}

_c_i, _c_f, _c_sz, _c_p = ctypes.c_int, ctypes.c_float, ctypes.c_size_t, ctypes.c_void_p

# name -> (restype, argtypes); mirrors include/siliconfer_hip.h
_SIGS = {
    "sf_last_error": (ctypes.c_char_p, []),
    "sf_abi_version": (_c_i, []),
    "sf_device_arch_ok": (_c_i, [_c_i]),
    "sf_q4_blob_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i]),
    "sf_q4_repack": (_c_i, [_c_p, _c_p, _c_p, _c_i, _c_i, _c_i, _c_p, _c_sz, _c_p]),
    "sf_q4_unpack": (_c_i, [_c_p, _c_i, _c_i, _c_i, _c_i, _c_p, _c_p, _c_p, _c_p]),
    "sf_q4_gemv": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_p, _c_p, _c_i,
                          _c_i, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_q4_gemv_supported": (_c_i, [_c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_q4_gemv_fused": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_f, _c_i, _c_p, _c_i, _c_p, _c_p,
                                _c_i, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_q4_gemv_fused_rows_supported": (_c_i, [_c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_q4_gemv_fused_rows": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_f, _c_i, _c_p, _c_i, _c_p, _c_p, _c_i,
                                     _c_i, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_q4_gemv_fused_rope_supported": (_c_i, [_c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_q4_gemv_fused_rope": (_c_i, [_c_p, _c_p, _c_p, _c_f, _c_i, _c_p, _c_i, _c_p, _c_p, _c_i, _c_p,
                                     _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_i, _c_i, _c_i, _c_i,
                                     _c_p, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_q4_gemm_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i]),
    "sf_q4_gemm": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_p, _c_p, _c_i,
                          _c_i, _c_i, _c_i, _c_i, _c_i, _c_p, _c_sz, _c_p]),
    "sf_q4_matmul_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_q4_rows_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_q4_matmul": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_p, _c_p, _c_i,
                            _c_i, _c_i, _c_i, _c_i, _c_i, _c_p, _c_sz, _c_p]),
    "sf_q4_matmul_group_supported": (_c_i, [_c_i, _c_i, _c_p, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_q4_matmul_group": (_c_i, [_c_i, _c_i, _c_p, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_i,
                                  _c_i, _c_i, _c_i, _c_p, _c_sz, _c_p]),
    "sf_q4_gemm_splits": (_c_i, [_c_i, _c_i, _c_i, _c_i]),
    "sf_q4_gemm_partials": (_c_i, [_c_p, _c_p, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_p, _c_sz,
                                   _c_p]),
    "sf_kv_quant_append": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i,
                                  _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_attn_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i]),
    "sf_attn_default_splits": (_c_i, [_c_i, _c_i, _c_i]),
    "sf_attn_default_splits_d": (_c_i, [_c_i, _c_i, _c_i, _c_i]),
    "sf_attn_decode_i8kv": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i,
                                   _c_p, _c_sz, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_f,
                                   _c_i, _c_p]),
    "sf_attn_noalloc_max_bytes": (_c_sz, []),
    "sf_attn_decode_i8kv_noalloc": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i,
                                           _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_f, _c_i, _c_p]),
    "sf_attn_decode_i8kv_dev": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i,
                                       _c_p, _c_sz, _c_i, _c_i, _c_i, _c_p, _c_i, _c_i, _c_i,
                                       _c_i, _c_f, _c_i, _c_p]),
    "sf_attn_decode_i8kv_partials_dev": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_sz,
                                                _c_i, _c_i, _c_i, _c_p, _c_i, _c_i, _c_i, _c_i, _c_f,
                                                _c_i, _c_p]),
    "sf_q4_gemv_attn_merge_supported": (_c_i, [_c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_q4_gemv_attn_merge": (_c_i, [_c_p, _c_p, _c_sz, _c_i, _c_i, _c_i, _c_i, _c_p, _c_i, _c_p, _c_p,
                                     _c_i, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_attn_prefill_i8kv": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i,
                                    _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_f, _c_p]),
    "sf_attn_prefill_i8kv_dev": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_p,
                                        _c_sz, _c_i, _c_i, _c_i, _c_p, _c_i, _c_i, _c_i, _c_f,
                                        _c_i, _c_p]),
    "sf_embed": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_i, _c_p]),
    "sf_rmsnorm": (_c_i, [_c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_i, _c_f, _c_p]),
    "sf_rmsnorm_partials": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_p, _c_i, _c_i, _c_i, _c_f,
                                   _c_p]),
    "sf_rope_kv_append": (_c_i, [_c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_p, _c_p, _c_p, _c_p,
                                 _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_p, _c_i, _c_p]),
    "sf_rope_kv_append_partials": (_c_i, [_c_p, _c_i, _c_p, _c_i, _c_p, _c_p, _c_i, _c_p, _c_i,
                                          _c_p, _c_p, _c_p, _c_p, _c_i, _c_i, _c_i, _c_i, _c_i,
                                          _c_i, _c_p, _c_i, _c_p]),
    "sf_silu_mul": (_c_i, [_c_p, _c_p, _c_i, _c_i, _c_i, _c_p]),
    "sf_lm_head_workspace_bytes": (_c_sz, [_c_i]),
    "sf_lm_head_argmax": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_p, _c_p, _c_p, _c_p,
                                 _c_sz, _c_p]),
    "sf_lm_head_argmax_rmsnorm": (_c_i, [_c_p, _c_p, _c_p, _c_f, _c_i, _c_p, _c_i, _c_i, _c_p,
                                         _c_p, _c_p, _c_p, _c_sz, _c_p]),
    "sf_lm_head_rows_workspace_bytes": (_c_sz, [_c_i, _c_i]),
    "sf_lm_head_argmax_rows": (_c_i, [_c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_i, _c_p, _c_p, _c_sz,
                                      _c_p]),
    "sf_rotary": (_c_i, [_c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_p, _c_i, _c_f, _c_i, _c_i,
                         _c_i, _c_i, _c_i, _c_i, _c_p, _c_p]),
    "sf_qk_norm_rotary": (_c_i, [_c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_i, _c_f, _c_p, _c_i, _c_i, _c_p, _c_i,
                                 _c_f, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_p, _c_p]),
    "sf_qk_norm_backward_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_qk_norm_rotary_backward": (_c_i, [_c_p, _c_p, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_i, _c_p, _c_p,
                                          _c_f, _c_p, _c_i, _c_i, _c_p, _c_i, _c_f, _c_i, _c_i, _c_i, _c_i, _c_i,
                                          _c_i, _c_p, _c_p, _c_sz, _c_p]),
    "sf_rotary_kv_append": (_c_i, [_c_p, _c_i, _c_p, _c_i, _c_i, _c_p, _c_i, _c_f, _c_i, _c_p, _c_i, _c_p,
                                   _c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_p, _c_i, _c_i, _c_i, _c_i, _c_i,
                                   _c_i, _c_i, _c_p]),
    "sf_attn_scored_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_attn_decode_scored_i8kv": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_i, _c_p,
                                          _c_sz, _c_i, _c_i, _c_i, _c_i, _c_p, _c_i, _c_i, _c_i, _c_i,
                                          _c_f, _c_i, _c_p]),
    "sf_kv_q4_append": (_c_i, [_c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_p, _c_i, _c_f, _c_p, _c_i, _c_i, _c_p, _c_i,
                               _c_f, _c_i, _c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_i, _c_i,
                               _c_i, _c_i, _c_i, _c_p]),
    "sf_kv_q4_dequant": (_c_i, [_c_p, _c_p, _c_p, _c_i, _c_i, _c_p, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_attn_q4_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i, _c_i]),
    "sf_attn_q4kv": (_c_i, [_c_p, _c_i, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_p, _c_sz, _c_i, _c_i, _c_i, _c_i,
                            _c_p, _c_i, _c_i, _c_i, _c_i, _c_f, _c_i, _c_p]),
    "sf_kv_evict_workspace_bytes": (_c_sz, [_c_i, _c_i, _c_i, _c_i]),
    "sf_kv_evict": (_c_i, [_c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_p, _c_i, _c_p, _c_i, _c_i, _c_i,
                           _c_p, _c_p, _c_sz, _c_i, _c_i, _c_i, _c_i, _c_p]),
    "sf_sample_workspace_bytes": (_c_sz, [_c_i, _c_i]),
    "sf_sample": (_c_i, [_c_p, _c_i, ctypes.c_longlong, _c_i, _c_i, _c_p, _c_f, _c_i, _c_f, _c_f, _c_p,
                         _c_p, _c_p, _c_p, _c_p, _c_p, _c_p, _c_i, _c_i, _c_p, _c_p, _c_sz, _c_p]),
    "sf_q4_chain_workspace_bytes": (_c_sz, [_c_p, _c_i]),
    "sf_q4_chain": (_c_i, [_c_p, _c_p, _c_p, _c_p, _c_p, _c_i, _c_p, _c_p, _c_p, _c_sz, _c_i, _c_i,
                           _c_p]),
    "sf_q4_chain_error": (_c_i, [_c_p, _c_p, _c_p]),
    "sf_floor_empty": (_c_i, [_c_p]),
    "sf_floor_read": (_c_i, [_c_p, _c_sz, _c_p, _c_p]),
}

_lock = threading.Lock()
_lib = None
_arch_ok: dict[int, bool] = {}


class SFError(RuntimeError):
    """A libsiliconfer_hip call failed (the reference raises RuntimeError too)."""


def load() -> ctypes.CDLL:
    """Load the library once; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise SFError(f"{LIB_PATH} is not built: run `python -m siliconfer_amd.build`")
            lib = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in _SIGS.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def exported_symbols() -> list[str]:
    return sorted(_SIGS)


def last_error() -> str:
    return load().sf_last_error().decode(errors="replace")


def check(rc: int, what: str) -> None:
    if rc != 0:
        raise SFError(f"{what}: {last_error()} (code {rc})")


def hip_available() -> bool:
    """True when the library loads and the current device is a gfx950 GPU."""
    try:
        lib = load()
    except SFError:
        return False
    if not torch.cuda.is_available():
        return False
    dev = torch.cuda.current_device()
    if dev not in _arch_ok:
        _arch_ok[dev] = lib.sf_device_arch_ok(dev) == 1
    return _arch_ok[dev]


def require_device(t: torch.Tensor, name: str) -> None:
    if t.is_cuda and t.is_contiguous():
        return
    if not t.is_cuda:
        raise SFError(f"{name} must be a device tensor (got {t.device})")
    raise SFError(f"{name} must be contiguous")


def dt(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise SFError(f"unsupported dtype {t.dtype}") from None


def stream(t: torch.Tensor | None = None) -> int:
    """The current stream's handle on t's device (else the current device)."""
    if t is not None and not t.is_cuda:
        raise ValueError(f"Expected a device tensor, got {t.device}")
    # the raw handle: torch.cuda.current_stream builds a Stream object around it,
    # most of the 13.1 us of host time that one small Q4Linear call took (8.4 now)
    return torch._C._cuda_getCurrentRawStream(t.get_device() if t is not None
                                              else torch.cuda.current_device())


def on_device(t: torch.Tensor):
    """A context in which t's device is the current one (launches go there)."""
    return _NOTHING if torch._C._cuda_getDevice() == t.get_device() else torch.cuda.device(t.device)


_NOTHING = contextlib.nullcontext()


class _Scratch(threading.local):
    def __init__(self) -> None:
        self.held: dict = {}


_scratch = _Scratch()
SCRATCH_HELD = 64 << 20  # bytes that a thread keeps a stream; more goes back to torch's allocator after its call


def scratch(device: torch.device, stream_handle: int, nbytes: int) -> torch.Tensor:
    """Workspace of one call: kept a (host thread, device, stream) and grown on demand. A
    thread's calls on a stream run one after the other; two threads' launches on it may
    interleave, since a call gives up the interpreter's lock. While a graph is recorded a
    tensor of the graph's own, so that no two graphs share one; past SCRATCH_HELD one of the call's own."""
    if nbytes > SCRATCH_HELD or torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
    held, key = _scratch.held, (device, stream_handle)
    ws = held.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = held[key] = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
    return ws


INT_MIN, INT_MAX = -0x80000000, 0x7fffffff


def refuse_int(**numbers):
    """Raise for numbers of which a C int cannot hold one (ctypes would cut it to its low half)."""
    raise SFError(", ".join(f"{k} {v}" for k, v in numbers.items()) + ": numbers must fit 32 bits")


def lengths_arg(lengths, B: int, device: torch.device, name: str = "lengths") -> tuple[int | None, int]:
    """(device pointer or None, host value) of lengths given as int32 [B] or one int."""
    if not isinstance(lengths, torch.Tensor):
        n = int(lengths)
        if not 0 <= n < 1 << 31:
            raise SFError(f"{name} {n} outside 0 .. 2^31 - 1")
        return None, n
    if (lengths.dtype is not torch.int32 or lengths.shape != (B,) or lengths.device != device
            or not lengths.is_contiguous()):
        raise SFError(f"{name} must be an int, or a contiguous int32 tensor [{B}] on the cache's device")
    return lengths.data_ptr(), 0


def check_cache(device: torch.device, k_codes, k_scales, v_codes, v_scales, positions=None,
                scores=None) -> None:
    """The buffers of an int8 cache: codes [B, KVH, T_cap, D], the others [B, KVH, T_cap],
    all contiguous on `device`."""
    at, rows, i8, dt = device.index, k_codes.shape[:-1], torch.int8, k_scales.dtype
    if not (k_codes.get_device() == v_codes.get_device() == k_scales.get_device() == v_scales.get_device() == at
            and k_codes.dtype is i8 and v_codes.dtype is i8 and v_scales.dtype is dt
            and (dt is torch.float16 or dt is torch.float32) and v_codes.shape == k_codes.shape
            and k_scales.shape == rows and v_scales.shape == rows and k_codes.is_contiguous()
            and v_codes.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()):
        _explain_cache(device, k_codes, k_scales, v_codes, v_scales)
    if positions is not None:
        _check_buffer(positions, "slot positions", rows, device)
        if positions.dtype is not torch.int32:
            raise SFError("slot positions must be int32")
    if scores is not None:
        _check_buffer(scores, "scores", rows, device)
        if scores.dtype is not torch.float32:
            raise SFError("scores must be float32")


def _explain_cache(device: torch.device, k_codes, k_scales, v_codes, v_scales) -> None:
    if k_codes.dtype is not torch.int8 or v_codes.dtype is not torch.int8:
        raise SFError("KV codes must be int8")
    if k_scales.dtype is not v_scales.dtype or k_scales.dtype not in (torch.float16, torch.float32):
        raise SFError("k/v scales must both be float16 or both float32")
    if k_codes.dim() != 4 or v_codes.shape != k_codes.shape:
        raise SFError("k_codes / v_codes must both be [B, n_kv_heads, T, head_dim]")
    rows = k_codes.shape[:3]
    _check_buffer(k_codes, "k_codes", None, device)
    _check_buffer(v_codes, "v_codes", None, device)
    _check_buffer(k_scales, "k_scales", rows, device)
    _check_buffer(v_scales, "v_scales", rows, device)


def _check_buffer(t: torch.Tensor, name: str, rows, device: torch.device) -> None:
    if not t.is_contiguous() or t.device != device:
        raise SFError(f"{name} must be contiguous on {device}")
    if rows is not None and t.shape != rows:
        raise SFError(f"{name} must be {list(rows)} (got {list(t.shape)})")


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()
