"""Model-side call surface: Q4Linear, the int8 and 4-bit KV caches and the transformer
layer modules."""

from .kv_cache import BoundedKVCache, Q4KVCache, QuantizedKVCache, dequantize_kv, make_quantized_cache, quantize_kv
from .layers import MLP, Attention, RMSNorm, TransformerBlock, apply_rope, compute_rope_freqs
from .q4_linear import Q4Linear
from .rope import Rotary, rotary_frequencies

__all__ = ["Q4Linear", "QuantizedKVCache", "BoundedKVCache", "Q4KVCache", "quantize_kv", "dequantize_kv",
           "make_quantized_cache", "RMSNorm", "Attention", "MLP", "TransformerBlock", "apply_rope", "compute_rope_freqs",
           "Rotary", "rotary_frequencies"]
