"""Rotary frequencies in 64 bits and their long-context scalings, for
`kernels.rotary` (the reference has the plain and the llama3 form in fp32,
/root/reference/siliconfer/model/layers.py:24-55).

Scaling types, by the names and fields of a HuggingFace `rope_scaling` entry:
  default  theta^(-2 i / r)
  linear   positions divided by `factor`
  dynamic  theta grown so that the slowest pair spans `factor` times the trained
           length, from the length that is asked for on
  llama3   slow pairs divided by `factor`, fast ones kept, a ramp between
  yarn     the ramp in numbers of turns over the trained length (beta_fast,
           beta_slow), and cos / sin times 0.1 ln(factor) + 1 (attention_factor in its
           place where given; mscale, mscale_all_dim and truncate false are refused)
A field that is null counts as absent.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from .._lib import SFError
from .config import ModelConfig

__all__ = ["rotary_frequencies", "Rotary"]


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None,
                       trained: int | None = None, length: int | None = None) -> tuple[np.ndarray, float]:
    """(float64 angles a position of the rotary_dim / 2 pairs, the factor on cos and
    sin). `trained`: the length the model was trained at, where `scaling` does not name
    it (`original_max_position_embeddings`); `length`: the longest position + 1 that
    "dynamic" is to reach."""
    if rotary_dim <= 0 or rotary_dim % 2 or not theta > 0:
        raise SFError(f"need an even rotary_dim and theta > 0 (got {rotary_dim}, {theta})")
    i = np.arange(0, rotary_dim, 2, dtype=np.float64)
    f = float(theta) ** (-i / rotary_dim)
    sc = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = sc.get("rope_type", sc.get("type", "")) or "default"
    if kind == "default":
        return f, 1.0
    factor = float(sc.get("factor", 1.0))
    if not factor > 0:
        raise SFError(f"rope scaling factor {factor}")
    trained = sc.get("original_max_position_embeddings", trained)
    if kind == "linear":
        return f / factor, 1.0
    if trained is None:
        raise SFError(f"rope scaling {kind!r} needs the trained length")
    trained = float(trained)
    if kind == "dynamic":
        if rotary_dim < 4:
            raise SFError("rope scaling 'dynamic' needs at least two pairs")
        over = max(float(length or trained), trained)
        base = float(theta) * (factor * over / trained - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
        return base ** (-i / rotary_dim), 1.0
    if kind == "llama3":
        lo, hi = float(sc.get("low_freq_factor", 1.0)), float(sc.get("high_freq_factor", 4.0))
        turns = trained * f / (2 * math.pi)  # over the trained length
        keep = np.clip((turns - lo) / (hi - lo), 0, 1) if hi != lo else (turns >= hi).astype(np.float64)
        return f / factor * (1 - keep) + f * keep, 1.0
    if kind == "yarn":
        other = [k for k in ("mscale", "mscale_all_dim") if k in sc] + ["truncate"] * (not sc.get("truncate", True))
        if other:  # they would change the factor, or the ramp's ends
            raise SFError(f"rope scaling 'yarn' with {', '.join(other)}")
        at = lambda turns: rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo = max(math.floor(at(float(sc.get("beta_fast", 32.0)))), 0)
        hi = min(math.ceil(at(float(sc.get("beta_slow", 1.0)))), rotary_dim - 1)
        ramp = np.clip((np.arange(rotary_dim // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        scale = sc.get("attention_factor")
        scale = float(scale) if scale is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
        return f / factor * ramp + f * (1 - ramp), scale
    raise SFError(f"rope scaling type {kind!r}")


class Rotary:
    """How a model turns its heads: the pair layout, the rotated part of the head, and
    the frequencies with their factor (kept on each device that asks)."""

    def __init__(self, inv_freq, scale: float = 1.0, interleaved: bool = False) -> None:
        self.inv_freq = np.ascontiguousarray(inv_freq, dtype=np.float64)
        if self.inv_freq.ndim != 1 or self.inv_freq.size == 0:
            raise SFError("inv_freq must be a non-empty 1-D array")
        self.scale, self.interleaved = float(scale), bool(interleaved)
        self._on: dict = {}

    @classmethod
    def from_config(cls, config: ModelConfig, rotary_dim: int | None = None, interleaved: bool = False,
                    scaling: dict | None = None, length: int | None = None) -> "Rotary":
        """Of a model's head_dim, theta and rope_scaling (or `scaling` in its place). An entry
        that names no trained length goes by max_position_embeddings, llama3 by 8192 as in
        `config.rope_freqs`."""
        if scaling is None and config.rope_scaling is not None:
            scaling = config.rope_scaling.entry()
            if config.rope_scaling.type == "llama3":
                scaling["original_max_position_embeddings"] = config.rope_scaling.original_max_position_embeddings
        r = config.head_dim if rotary_dim is None else rotary_dim
        if r > config.head_dim:
            raise SFError(f"rotary_dim {r} exceeds the head's {config.head_dim}")
        return cls(*rotary_frequencies(r, config.rope_theta, scaling, config.max_position_embeddings or None, length),
                   interleaved)

    def on(self, device) -> torch.Tensor:
        """The frequencies on `device`, copied there when it first asks."""
        f = self._on.get(device)
        if f is None:
            d = torch.device(device)
            if d.type == "cuda":
                d = torch.device("cuda", torch.cuda.current_device() if d.index is None else d.index)
                if d not in self._on and torch._C._cuda_isCurrentStreamCapturing():
                    raise SFError("Rotary.on(device): once before a graph is recorded (it copies from the host)")
            f = self._on.get(d)
            if f is None:
                f = self._on[d] = torch.from_numpy(self.inv_freq).to(d)
        return f
