"""Gradients through rotary positions: against the formula in 64 bits, against differences, and
through the Attention layer, whose other RoPE route is differentiable as well."""

import numpy as np
import pytest
import torch

from oracle import bounded
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.rotary import rotary
from siliconfer_amd.model import Rotary, rotary_frequencies
from siliconfer_amd.model.config import ModelConfig
from siliconfer_amd.model.layers import Attention, compute_rope_freqs

pytestmark = pytest.mark.gpu


def transpose(g, positions, inv_freq, interleaved, scale):
    """(R^T g, bound on its fp32 arithmetic): the turn by the opposite angle."""
    return bounded.rotary(g, -np.asarray(positions, np.int64), inv_freq, interleaved, scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (96, 32), (10, 6)])
def test_against_the_formula(dev, dtype, interleaved, D, rot):
    g = torch.Generator().manual_seed(D)
    f, scale = rotary_frequencies(rot, 1e4, {"type": "yarn", "factor": 4.0}, trained=128)
    inv = torch.from_numpy(f).to(dev)
    pos = torch.randint(0, 100000, (2, 5), generator=g, dtype=torch.int32).to(dev)
    q = torch.randn(2, 5, 3, D, generator=g).to(dev, dtype).requires_grad_()
    k = torch.randn(2, 2, 5, D, generator=g).to(dev, dtype).requires_grad_()
    gq = torch.randn(2, 5, 3, D, generator=g).to(dev, dtype)
    gk = torch.randn(2, 5, 2, D, generator=g).to(dev, dtype)
    yq, yk = rotary(q, k.transpose(1, 2), pos, inv, interleaved=interleaved, scale=scale)
    with torch.no_grad():  # the values are those of the call without a gradient
        assert torch.equal(yq, rotary(q, None, pos, inv, interleaved=interleaved, scale=scale)[0])
    torch.autograd.backward((yq, yk), (gq, gk))
    for x, got in ((gq, q.grad), (gk, k.grad.transpose(1, 2))):
        want, bound = transpose(x.float().cpu().numpy(), pos.cpu().numpy(), f, interleaved, scale)
        half = torch.finfo(dtype).eps / 2
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # (half a step of fp16's subnormals)
        assert (abs(got.double().cpu().numpy() - want) <= bound * (1 + half) + half * abs(want) + tiny).all()


def test_against_differences(dev):
    """A linear map's differences are its values: <g, R (x + e) - R x> = <R^T g, e>."""
    g = torch.Generator().manual_seed(1)
    inv = torch.from_numpy(rotary_frequencies(16, 1e4)[0]).to(dev)
    pos = torch.arange(7, device=dev)
    x = torch.randn(1, 7, 2, 24, generator=g).to(dev).requires_grad_()
    w = torch.randn(1, 7, 2, 24, generator=g).to(dev)
    (rotary(x, None, pos, inv)[0] * w).sum().backward()
    for _ in range(8):
        e = torch.randn(1, 7, 2, 24, generator=g).to(dev)
        with torch.no_grad():
            a = (w.double() * (rotary(x + e, None, pos, inv)[0].double() - rotary(x - e, None, pos, inv)[0].double())).sum()
        b = 2 * (x.grad.double() * e.double()).sum()
        # a pair's turn takes two roundings of x + e and eight of the products, each half a step of the largest
        # value, at both ends; a gradient eight of the largest weight's
        most = (x.detach().abs() + e.abs()).max()
        bound = 20 * most * w.abs().sum() + 16 * w.abs().max() * e.abs().sum()
        assert abs(a - b).item() <= 2.0 ** -24 * bound.item()


def test_one_output_and_leaves_without_a_gradient(dev):
    inv, pos = torch.ones(4, dtype=torch.float64, device=dev), torch.arange(3, device=dev)
    q, k = torch.randn(1, 3, 2, 8, device=dev, requires_grad=True), torch.randn(1, 3, 1, 8, device=dev)
    yq, yk = rotary(q, k, pos, inv)
    yk.sum().backward()
    assert (q.grad == 0).all()
    q.grad = None
    rotary(q, None, pos, inv)[0].sum().backward()  # (an expanded gradient)
    want, bound = transpose(np.ones((1, 3, 2, 8)), np.arange(3), np.ones(4), False, 1.0)
    assert (abs(q.grad.double().cpu().numpy() - want) <= bound + 2.0 ** -24 * abs(want)).all()
    k.requires_grad_()
    with torch.no_grad():
        assert not rotary(q, k, pos, inv)[0].requires_grad
    with pytest.raises(SFError, match="gradient"):
        rotary(q, k, pos, inv, out_q=torch.empty_like(q))
    assert rotary(q.detach(), None, pos, inv, out_q=torch.empty_like(q))[0].grad_fn is None


def test_through_the_layer(dev):
    """The gradients of the layer's weights with a Rotary of its own frequencies are those of its
    torch route: fp32 angles of positions below 9 apart (2e-5, as the layer's outputs)."""
    c = ModelConfig(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=1e4)
    x = torch.randn(2, 9, 128, generator=torch.Generator().manual_seed(2)).to(dev)
    w = torch.randn(2, 9, 128, generator=torch.Generator().manual_seed(3)).to(dev)
    grads = []
    for rot in (None, Rotary(*rotary_frequencies(64, 1e4))):
        torch.manual_seed(4)
        attn = Attention(c, compute_rope_freqs(c, dev), dev, rot)
        head, kv = attn(x[:, :5])
        tail, _ = attn(x[:, 5:], kv)
        (torch.cat([head, tail], 1) * w).sum().backward()
        grads.append({n: p.grad for n, p in attn.named_parameters()})
    for n, want in grads[0].items():
        got = grads[1][n]
        assert got is not None and ((got - want).norm() / want.norm()).item() <= 2e-5, n
