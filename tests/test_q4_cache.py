"""The 4-bit cache's own rules without a GPU: buffers, growth, lengths, refusals; norms of heads in a
layer's module tree."""

import numpy as np
import pytest
import torch

from siliconfer_amd._lib import SFError
from siliconfer_amd.model import Attention, Q4KVCache, QuantizedKVCache, TransformerBlock, compute_rope_freqs, make_quantized_cache
from siliconfer_amd.model.config import ModelConfig

CFG = ModelConfig(hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=4,
                  num_key_value_heads=2, head_dim=32, vocab_size=50)


@pytest.mark.parametrize("D,group,held", [(128, None, 64), (64, None, 64), (96, None, 32), (80, None, 80), (16, None, 16),
                                          (128, 128, 128), (256, 32, 32), (48, 48, 48)])
def test_buffers_growth_and_lengths(D, group, held):
    c = Q4KVCache(10, group)
    assert c.length() == c.nbytes() == 0 and c.buffers() == (None,) * 4
    c.reserve(3, 2, D, 7, "cpu")
    kc, kp, vc, vp = c.buffers()
    assert kc.shape == vc.shape == (3, 2, 10, D // 2) and kp.shape == vp.shape == (3, 2, 10, D // held, 2)
    assert kc.dtype == vc.dtype == torch.uint8 and kp.dtype == vp.dtype == torch.float16
    for t in c.buffers():
        t.copy_(torch.randint(0, 100, t.shape))
    old = [t.clone() for t in c.buffers()]
    c.set_length(9)
    assert c.nbytes() == 2 * 3 * 2 * 9 * (D // 2 + 4 * (D // held))
    c.reserve(3, 2, D, 33, "cpu")
    assert c.capacity == 40
    assert all(torch.equal(a[:, :, :9], b[:, :, :9]) and a.shape[2] == 40 for a, b in zip(c.buffers(), old))
    c.trim(4)
    assert c.length() == 4
    c.trim(100)
    c.trim(-1)
    assert c.length() == 0


def test_refusals():
    for D, group in ((24, None), (272, None), (0, None), (128, 16), (96, 64), (128, 48), (80, 32)):
        with pytest.raises(SFError, match="multiple of 16"):
            Q4KVCache(10, group).reserve(1, 1, D, 1, "cpu")
    c = Q4KVCache(10, growable=False)
    c.reserve(1, 2, 64, 10, "cpu")
    for bad in ((2, 2, 64), (1, 1, 64), (1, 2, 32)):
        with pytest.raises(SFError, match="shape changed"):
            c.reserve(*bad, 1, "cpu")
    with pytest.raises(SFError, match="overflow"):
        c.reserve(1, 2, 64, 11, "cpu")
    for n in (-1, 11):
        with pytest.raises(SFError, match="outside"):
            c.set_length(n)
    empty = Q4KVCache(4)
    with pytest.raises(SFError, match="outside"):
        empty.set_length(0)
    with pytest.raises(SFError, match="holds nothing"):
        empty.attend(torch.zeros(1, 1, 2, 64))
    x = torch.zeros(1, 2, 3, 64)
    for call in (lambda: empty.append(x, x), lambda: empty.update(x, x), lambda: empty.append_rotary(x[0], 1, 1, None)):
        with pytest.raises(SFError):
            call()
    assert empty.buffers() == (None,) * 4 and empty.length() == 0


def test_make_quantized_cache():
    assert [type(c) for c in make_quantized_cache(2)] == [QuantizedKVCache] * 2
    four = make_quantized_cache(3, 8, bits=4, group=32)
    assert [(type(c), c.capacity, c.group) for c in four] == [(Q4KVCache, 8, 32)] * 3
    for kw in (dict(bits=5), dict(group=64), dict(bits=0)):
        with pytest.raises(SFError, match="bits"):
            make_quantized_cache(1, **kw)


def test_norms_of_heads_in_the_module_tree():
    freqs = compute_rope_freqs(CFG)
    plain, normed = (TransformerBlock(CFG, freqs, "cpu", qk_norm=n) for n in (False, True))
    assert plain.self_attn.q_norm is None and not [n for n, _ in plain.named_parameters() if "q_norm" in n or "k_norm" in n]
    a = normed.self_attn
    assert a.q_norm.weight.shape == a.k_norm.weight.shape == (32,) and a.q_norm.eps == CFG.rms_norm_eps
    assert {"self_attn.q_norm.weight", "self_attn.k_norm.weight"} <= {n for n, _ in normed.named_parameters()}
    assert isinstance(a, Attention)


def weights(seed=0, **extra):
    g = np.random.default_rng(seed)
    at, H, D, I = "model.layers.0", 64, 32, 128
    w = {f"{at}.self_attn.{n}_proj.weight": s for n, s in (("q", (4 * D, H)), ("k", (2 * D, H)), ("v", (2 * D, H)), ("o", (H, 4 * D)))}
    w |= {f"{at}.mlp.gate_proj.weight": (I, H), f"{at}.mlp.up_proj.weight": (I, H), f"{at}.mlp.down_proj.weight": (H, I)}
    w |= {f"{at}.input_layernorm.weight": (H,), f"{at}.post_attention_layernorm.weight": (H,)}
    w |= {f"{at}.self_attn.{n}_norm.weight": (D,) for n in extra.get("norms", "")}
    return {n: (0.1 * g.standard_normal(s)).astype(np.float32) for n, s in w.items()}


def test_norms_of_heads_from_a_checkpoint():
    freqs = compute_rope_freqs(CFG)
    w = weights(norms="qk")
    a = TransformerBlock.from_weights(CFG, w, 0, freqs, device="cpu").self_attn
    for n, m in (("q", a.q_norm), ("k", a.k_norm)):
        assert np.array_equal(m.weight.detach().numpy(), w[f"model.layers.0.self_attn.{n}_norm.weight"])
    assert TransformerBlock.from_weights(CFG, weights(), 0, freqs, device="cpu").self_attn.q_norm is None
    for one in "qk":
        with pytest.raises(SFError, match="without the other"):
            TransformerBlock.from_weights(CFG, weights(norms=one), 0, freqs, device="cpu")
