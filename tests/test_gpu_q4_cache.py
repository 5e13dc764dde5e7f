"""Normed heads, the 4-bit cache and attention over it together, as the layers run them: steps of
a cache against the 64-bit oracle, a layer over every form of cache, its gradients."""

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.kv_q4 import dequantize_kv_q4
from siliconfer_amd.kernels.rotary import rotary
from siliconfer_amd.model import (Attention, BoundedKVCache, Q4KVCache, QuantizedKVCache, Rotary, TransformerBlock,
                                  compute_rope_freqs, rotary_frequencies)
from siliconfer_amd.model.config import ModelConfig

pytestmark = pytest.mark.gpu
H, KVH, D = 6, 2, 64


def weights(dev, seed):
    g = torch.Generator().manual_seed(seed)
    return [(1 + 0.2 * torch.randn(D, generator=g)).to(dev) for _ in range(2)]


@pytest.mark.parametrize("B,steps", [(1, [20] + [1] * 12 + [200, 1]), (3, [5, 1, 1, 16, 0, 1, 9, 1])])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_steps_against_the_oracle(dev, B, steps, normed, interleaved):
    """Every step's q is the (normed and) turned rows, its slots hold k and v within half a code's step and
    the roundings of s and m, what was there stays, and attention is the oracle's over these codes."""
    r = Rotary(*rotary_frequencies(48, 1e4, {"type": "yarn", "factor": 4.0}, trained=64), interleaved)
    cache = Q4KVCache(capacity=16, group=32)
    g = torch.Generator().manual_seed(B)
    qw, kw = weights(dev, B) if normed else (None, None)
    n = 0
    for T in steps:
        qkv = torch.randn(B, T, (H + 2 * KVH) * D, generator=g).to(dev)
        before = [None if t is None else t[:, :, :n].clone() for t in cache.buffers()]
        q = cache.append_rotary(qkv, H, KVH, r, qw, kw)
        x = qkv.view(B, T, H + 2 * KVH, D)
        pos, f = np.arange(n, n + T), r.on("cpu").double().numpy()
        rows = [t.cpu().double().numpy() for t in (x[:, :, :H], x[:, :, H:H + KVH])]
        # (both in 64 bits, with what fp32 steps may lose: the kernels need not round alike)
        (want_q, loss), (want_k, _) = (
            O.qk_norm_rotary(t, w.cpu().double().numpy(), pos, f, 1e-6, interleaved, r.scale) if normed
            else O.bounded.rotary(t, pos, f, interleaved, r.scale) for t, w in zip(rows, (qw, kw)))
        n += T
        assert cache.length() == n and (abs(q.cpu().numpy() - want_q) <= loss + 2.0 ** -24 * (abs(want_q) + loss)).all()
        assert all(b is None or torch.equal(t[:, :, :n - T], b) for t, b in zip(cache.buffers(), before))
        kc, kp, vc, vp = cache.buffers()
        for c, p, want in ((kc, kp, torch.from_numpy(want_k).to(dev)), (vc, vp, x[:, :, H + KVH:].double())):
            got = dequantize_kv_q4(c[:, :, n - T:n], p[:, :, n - T:n]).transpose(1, 2)
            y = want.reshape(B, T, KVH, D // 32, 32)
            # half a step; s and m within half a step of fp16, where s counts up to 15 times
            step = (y.amax(-1) - y.amin(-1)) / 15
            tol = step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -10) + 2.0 ** -10 * y.abs().amax(-1)
            assert ((got.reshape(y.shape) - y).abs() <= tol[..., None]).all()
        if T:
            out = cache.attend(q)
            ref, bound = O.attention(q.double().cpu().numpy(), *(t.cpu().numpy() for t in cache.buffers()), [n] * B)
            assert (abs(out.cpu().numpy() - ref) <= bound + 2.0 ** -24 * (abs(ref) + bound)).all()
    cache.trim(7)
    again = cache.append_rotary(qkv[:, :1], H, KVH, r, qw, kw) if qkv.shape[1] else None
    assert cache.length() == 8 and again.shape == (B, 1, H, D)


def test_update_gives_the_values_that_are_held(dev):
    cache = Q4KVCache(capacity=4)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, KVH, 9, D, generator=g).to(dev).half() for _ in range(2))
    a, b = cache.update(k[:, :, :4], v[:, :, :4])
    c, d = cache.update(k[:, :, 4:], v[:, :, 4:])
    assert c.dtype is torch.float16 and c.shape == d.shape == (2, KVH, 9, D)
    assert torch.equal(c[:, :, :4], a) and torch.equal(d[:, :, :4], b)
    for got, x in ((c, k), (d, v)):
        codes, s, m, _ = O.quantize(x.double().cpu().numpy(), 64)
        want, _ = O.values(O.pack(codes), np.stack([s, m], -1))
        assert torch.equal(got.cpu(), torch.from_numpy(want.astype(np.float32)).half())
    assert cache.nbytes() == 2 * 2 * KVH * 9 * (32 + 4)


CFG = ModelConfig(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=1e4)
# Relative error in the norm of fp32 runs of the layer: each of its sums (projections of 128 and
# 256 terms, norms and scores of 64, softmax of at most 83) loses at most as many half steps of
# 2^-24 as it has terms, 600 in all, or 3.6e-5; a score's error counts whole in its weight, and with
# normed heads (weights under 2) a score is at most 2 * 2 * 64 / 8 = 32, so that its own 270 half
# steps are at most 32 * 270 * 2^-24 = 5.2e-4 of the weight. Together under 6e-4.
NEAR = 6e-4


def layer(dev, rot, qk_norm=True):
    torch.manual_seed(3)
    attn = Attention(CFG, compute_rope_freqs(CFG, dev), dev, rot, qk_norm)
    if qk_norm:
        with torch.no_grad():
            for m in (attn.q_norm, attn.k_norm):
                m.weight.copy_(1 + 0.2 * torch.randn(64).clamp(-4, 4))
    return attn


ROT = {"half": None, "part": Rotary(*rotary_frequencies(32, 1e4), interleaved=True)}


def plain(attn, x, w, values=None):
    """The layer in 64 bits on the CPU: (output, q, k, v), attention over `values` (k, v) where given."""
    B, T, _ = x.shape
    r = attn._rotary_of(None)
    q, k, v = ((x @ w[n].T).reshape(B, T, -1, 64) for n in ("q_proj", "k_proj", "v_proj"))
    q, k = (t / (t.square().mean(-1, keepdim=True) + CFG.rms_norm_eps).sqrt() * w[n] for t, n in ((q, "q_norm"), (k, "k_norm")))
    f = r.on(x.device).double()
    ang = torch.arange(T, dtype=torch.float64)[:, None] * f
    cos, sin = (r.scale * t[:, None, :] for t in (ang.cos(), ang.sin()))

    def turn(t):
        P = len(f)
        a, b = (t[..., 0:2 * P:2], t[..., 1:2 * P:2]) if r.interleaved else (t[..., :P], t[..., P:2 * P])
        y = (a * cos - b * sin, a * sin + b * cos)
        y = torch.stack(y, -1).flatten(-2) if r.interleaved else torch.cat(y, -1)
        return torch.cat([y, t[..., 2 * P:]], -1)

    q, k = turn(q), turn(k)
    kk, vv = (k.transpose(1, 2), v.transpose(1, 2)) if values is None else values
    kk, vv = (t.repeat_interleave(2, 1) for t in (kk, vv))
    s = (q.transpose(1, 2) @ kk.transpose(-1, -2)) / 8
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), float("-inf"))
    out = (s.softmax(-1) @ vv).transpose(1, 2).reshape(B, T, -1)
    return out @ w["o_proj"].T, q, k, v


def leaves(attn):
    return {n: getattr(attn, n).weight for n in ("q_proj", "k_proj", "v_proj", "o_proj", "q_norm", "k_norm")}


@pytest.mark.parametrize("rot", list(ROT))
def test_a_normed_layer_and_its_gradients(dev, rot):
    """Output and gradients of x, the projections and the norms' weights against the formula in 64
    bits. A gradient passes twice the steps that the output does."""
    attn = layer(dev, ROT[rot])
    g = torch.Generator().manual_seed(4)
    x, go = (torch.randn(2, 37, 128, generator=g) for _ in range(2))
    xd = x.to(dev).requires_grad_()
    out, _ = attn(xd)
    out.backward(go.to(dev))
    w = {n: t.detach().cpu().double().requires_grad_() for n, t in leaves(attn).items()}
    x64 = x.double().requires_grad_()
    if attn.rotary is not None:
        attn.rotary.on("cpu")
    want = plain(attn, x64, w)[0]
    want.backward(go.double())

    def err(a, b):
        return ((a.detach().cpu().double() - b).norm() / b.norm()).item()

    assert err(out, want.detach()) <= NEAR
    assert err(xd.grad, x64.grad) <= 2 * NEAR
    for n, t in leaves(attn).items():
        assert err(t.grad, w[n].grad) <= 2 * NEAR, n


@pytest.mark.parametrize("rot", list(ROT))
def test_a_normed_layer_over_every_cache_form(dev, rot):
    """Without a cache, over full-precision tensors, over int8 codes at one sequence and at two, over
    a bound that is not reached (8-bit codes: 2e-2), and over 4 bits: the formula in 64 bits over
    the values that the cache holds."""
    attn = layer(dev, ROT[rot])
    x = torch.randn(2, 40, 128, generator=torch.Generator().manual_seed(6)).to(dev)
    cuts = (0, 25, 26, 33, 40)

    def run(cache, x=x):
        out = []
        for a, b in zip(cuts, cuts[1:]):
            y, cache = attn(x[:, a:b], cache)
            out.append(y)
        return torch.cat(out, 1), cache

    def err(a, b):
        return ((a.cpu().double() - b.cpu().double()).norm() / b.cpu().double().norm()).item()

    with torch.no_grad():
        full, _ = attn(x)
        w = {n: t.detach().cpu().double() for n, t in leaves(attn).items()}
        assert err(full, plain(attn, x.cpu().double(), w)[0]) <= NEAR
        assert err(run(None)[0], full) <= NEAR
        assert err(run(QuantizedKVCache(16))[0], full) <= 2e-2
        assert err(run(BoundedKVCache(64))[0], full) <= 2e-2
        for i in range(2):
            assert err(run(QuantizedKVCache(16), x[i:i + 1])[0], full[i:i + 1]) <= 2e-2
            assert err(run(BoundedKVCache(64), x[i:i + 1])[0], full[i:i + 1]) <= 2e-2
        cache = Q4KVCache(16)
        got, same = run(cache)
        assert same is cache and cache.length() == 40
        kc, kp, vc, vp = (t[:, :, :40].contiguous() for t in cache.buffers())
        held = [dequantize_kv_q4(c, p).cpu().double() for c, p in ((kc, kp), (vc, vp))]
        assert err(got, plain(attn, x.cpu().double(), w, held)[0]) <= NEAR
        # each sequence by itself: the same codes, but for one on a border that another order of a
        # projection's sum moves by a step (range / 15, less than the value it stands beside, of one dim of 64)
        each = [run(Q4KVCache(64), x[i:i + 1])[0] for i in range(2)]
        assert err(torch.cat(each), got) <= 2e-2


def test_a_layer_without_norms_over_four_bits(dev):
    attn = layer(dev, None, qk_norm=False)
    x = torch.randn(2, 9, 128, generator=torch.Generator().manual_seed(7)).to(dev)
    with torch.no_grad():
        cache = Q4KVCache(16)
        got, _ = attn(x, cache)
        q, k, v = ((x @ getattr(attn, n).weight.T).view(2, 9, -1, 64) for n in ("q_proj", "k_proj", "v_proj"))
        r = attn._rotary_of(None)
        q, k = rotary(q, k, torch.arange(9, device=dev), r.on(dev))
        ref, bound = O.attention(q.double().cpu().numpy(), *(t.cpu().numpy() for t in cache.buffers()), [9, 9])
        want = torch.from_numpy(ref).reshape(2, 9, 256) @ attn.o_proj.weight.cpu().double().T
    assert ((got.cpu().double() - want).norm() / want.norm()).item() <= NEAR


def test_a_block_from_a_checkpoint(dev):
    """q_norm and k_norm of a checkpoint are used, by every step of a block over a 4-bit cache."""
    from test_q4_cache import CFG as C, weights as made
    w = made(norms="qk")
    freqs = compute_rope_freqs(C, dev)
    blk = TransformerBlock.from_weights(C, w, 0, freqs, device=dev)
    without = TransformerBlock.from_weights(C, made(), 0, freqs, device=dev)
    x = torch.randn(2, 12, 64, generator=torch.Generator().manual_seed(8)).to(dev)
    with torch.no_grad():
        full, cache = blk(x, Q4KVCache(16))
        steps, parts = Q4KVCache(4), []
        for t in (slice(0, 9), slice(9, 10), slice(10, 12)):
            y, steps = blk(x[:, t], steps)
            parts.append(y)
        assert steps.length() == cache.length() == 12
        # (a code on a border may fall either way, as above)
        assert ((torch.cat(parts, 1) - full).norm() / (full - x).norm()).item() <= 2e-2
        other, _ = without(x, Q4KVCache(16))
        h = x + blk.self_attn(blk.input_layernorm(x), Q4KVCache(16))[0]
        assert torch.equal(h + blk.mlp(blk.post_attention_layernorm(h)), full)
    assert not torch.equal(other, full)


def test_two_host_threads_and_two_streams(dev):
    """A cache's steps from two threads at once, on one stream and on one each, at sizes whose
    workspaces differ, give what one thread gives."""
    import threading

    r = Rotary(*rotary_frequencies(64, 1e4))
    r.on(dev)

    def inputs(i):
        g = torch.Generator().manual_seed(20 + i)
        return [torch.randn(1 + i, T, (H + 2 * KVH) * D, generator=g).to(dev) for T in (3000 - 1700 * i, 1, 1, 40, 1)], weights(dev, i)

    def work(args):
        cache, out = Q4KVCache(512), []
        for x in args[0]:
            q = cache.append_rotary(x, H, KVH, r, *args[1])
            out += [q, cache.attend(q), cache.attend(q[:, -1:].contiguous(), out_dtype=torch.bfloat16)]
        return out + [t[:, :, :cache.length()].clone() for t in cache.buffers()]

    args = [inputs(i) for i in range(2)]
    want = [work(x) for x in args]
    torch.cuda.synchronize()
    for own in (False, True):
        got, wrong = [None, None], []

        def run(i):
            try:
                with torch.cuda.stream(torch.cuda.Stream(dev) if own else torch.cuda.default_stream(dev)):
                    for _ in range(5):
                        got[i] = work(args[i])
                    torch.cuda.synchronize()
            except BaseException as e:  # noqa: BLE001 (handed to the test)
                wrong.append(e)

        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert not wrong, wrong
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals(dev):
    cache = Q4KVCache(4, growable=False)
    r = Rotary(*rotary_frequencies(64, 1e4))
    qkv = torch.zeros(1, 3, (H + 2 * KVH) * D, device=dev)
    for bad in (qkv[0], qkv[..., :-1], qkv.double()):
        with pytest.raises(SFError):
            cache.append_rotary(bad.contiguous(), H, KVH, r)
    with pytest.raises(SFError, match="does not hold"):
        cache.append_rotary(qkv, 5, 2, r)
    assert cache.buffers() == (None,) * 4
    cache.append_rotary(qkv, H, KVH, r)
    with pytest.raises(SFError, match="overflow"):
        cache.append_rotary(qkv, H, KVH, r)
    assert cache.length() == 3
    k = torch.zeros(1, KVH, 2, D, device=dev)
    with pytest.raises(SFError, match="same shape"):
        cache.append(k, k.half())
    with pytest.raises(SFError):
        cache.append(k.double(), k.double())
    with pytest.raises(SFError, match="does not match"):
        cache.attend(torch.zeros(1, 1, H, 32, device=dev))
    assert cache.length() == 3
