"""Norms of queries' and keys' heads as a layer's modules: two eps, hooks, replacements, over every
form of cache."""

import pytest
import torch

from siliconfer_amd.model import BoundedKVCache, Q4KVCache, QuantizedKVCache
from test_gpu_q4_cache import NEAR, layer

pytestmark = pytest.mark.gpu


class Norm(torch.nn.Module):
    """The norm in elementary operations."""

    def __init__(self, of, eps):
        super().__init__()
        self.weight, self.eps = of.weight, eps

    def forward(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * self.weight


CACHES = {"none": lambda: None, "int8": lambda: QuantizedKVCache(16), "int8 bounded": lambda: BoundedKVCache(64),
          "4 bits": lambda: Q4KVCache(16)}


def run(attn, x, cache):
    out = []
    for a, b in ((0, 20), (20, 21), (21, 24)):
        y, cache = attn(x[:, a:b], cache)
        out.append(y)
    return torch.cat(out, 1)


def err(a, b):
    return ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("cache", list(CACHES))
def test_each_norm_by_its_own_eps(dev, cache, B):
    """Two eps: as with modules that say so in elementary operations (codes: but for those on a border,
    2e-2), and unlike one eps for both."""
    attn, same, plain = layer(dev, None), layer(dev, None), layer(dev, None)
    attn.k_norm.eps = 5.0
    plain.q_norm, plain.k_norm = Norm(plain.q_norm, plain.q_norm.eps), Norm(plain.k_norm, 5.0)
    x = torch.randn(B, 24, 128, generator=torch.Generator().manual_seed(0)).to(dev)
    with torch.no_grad():
        got, want, other = (run(m, x, CACHES[cache]()) for m in (attn, plain, same))
    assert err(got, want) <= (NEAR if cache == "none" else 2e-2)
    assert err(other, want) > 0.1
    if cache == "none":
        for m in (attn, plain):
            m(x)[0].sum().backward()
        for name in ("q_norm", "k_norm"):
            a, b = (getattr(m, name).weight.grad for m in (attn, plain))
            assert err(a, b) <= 2 * NEAR


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("cache", list(CACHES))
def test_hooks_of_the_norms_are_called(dev, cache, B):
    """A hook on k_norm sees every step's heads [B, T, heads, D] and what it returns is used."""
    attn, plain = layer(dev, None), layer(dev, None)
    seen = []

    def double(module, args, out):
        seen.append(tuple(args[0].shape))
        return 2 * out

    handle = attn.k_norm.register_forward_hook(double)
    with torch.no_grad():
        plain.k_norm.weight.mul_(2)
        x = torch.randn(B, 24, 128, generator=torch.Generator().manual_seed(1)).to(dev)
        got, want = (run(m, x, CACHES[cache]()) for m in (attn, plain))
        assert seen == [(B, 20, 2, 64), (B, 1, 2, 64), (B, 3, 2, 64)]
        assert err(got, want) <= (NEAR if cache == "none" else 2e-2)
        handle.remove()
        plain.k_norm.weight.div_(2)
        assert torch.equal(run(attn, x, CACHES[cache]()), run(plain, x, CACHES[cache]()))


@pytest.mark.parametrize("cache", list(CACHES))
@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
def test_one_norm_alone(dev, cache, name):
    """With the other taken out: as with one that leaves its heads as they are."""
    attn, plain = layer(dev, None), layer(dev, None)
    setattr(attn, name, None)
    setattr(plain, name, torch.nn.Identity())
    x = torch.randn(1, 24, 128, generator=torch.Generator().manual_seed(2)).to(dev)
    with torch.no_grad():
        assert torch.equal(run(attn, x, CACHES[cache]()), run(plain, x, CACHES[cache]()))
        assert err(run(layer(dev, None), x, CACHES[cache]()), run(plain, x, CACHES[cache]())) > 0.05


def test_int4_layers_keep_no_graph(dev, tmp_path):
    """Beside int4 projections a checkpoint's head norms take no gradients: steps over a cache of tensors
    without `no_grad` keep no graph. Asked for, they have them; dense layers' norms do as the projections."""
    import numpy as np

    from siliconfer_amd.engine.loader import load_model
    from siliconfer_amd.engine.q4_loader import pack_and_replace_linears
    from siliconfer_amd.model import TransformerBlock, compute_rope_freqs
    from test_loader import TINY, tiny_checkpoint

    tiny_checkpoint(tmp_path, cfg=TINY, seed=1)
    cfg, w = load_model(tmp_path)
    for n in "qk":
        w[f"model.layers.0.self_attn.{n}_norm.weight"] = np.ones(cfg.head_dim, np.float32)
    freqs = compute_rope_freqs(cfg, dev)
    dense = TransformerBlock.from_weights(cfg, w, 0, freqs, device=dev).self_attn
    pack_and_replace_linears(w, cfg, 64, pack_sym=True)
    attn = TransformerBlock.from_weights(cfg, w, 0, freqs, 64, dev).self_attn
    for m, on in ((dense, True), (attn, False)):
        assert m.q_norm.weight.requires_grad is on and m.k_norm.weight.requires_grad is on
    x = torch.randn(1, 4, cfg.hidden_size, generator=torch.Generator().manual_seed(0)).to(dev)
    cache = None
    for t in range(4):
        y, cache = attn(x[:, t:t + 1], cache)
        assert not y.requires_grad and not cache[0].requires_grad
    attn.k_norm.weight.requires_grad_()
    attn(x)[1][0].sum().backward()
    assert attn.k_norm.weight.grad.shape == (cfg.head_dim,)
