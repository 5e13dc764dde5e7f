"""The bounded cache's operators together, as the framework runs them: tokens turned
and appended, attention that scores the slots, eviction, and drawn tokens, step by step
against the 64-bit oracle; the Attention module over a bounded cache; generation from
given numbers."""

import numpy as np
import pytest
import torch

from oracle import bounded
from siliconfer_amd._lib import SFError
from siliconfer_amd.engine.generate import SamplingParams, generate, sample_token
from siliconfer_amd.kernels.rotary import rotary
from siliconfer_amd.kernels.sampling import sample
from siliconfer_amd.model import BoundedKVCache, QuantizedKVCache, Rotary, rotary_frequencies
from siliconfer_amd.model.config import ModelConfig
from siliconfer_amd.model.layers import Attention, compute_rope_freqs
from siliconfer_amd.model.llama import LlamaModel

pytestmark = pytest.mark.gpu
H, KVH, D = 6, 2, 64


def buffers(c):
    return [t.cpu().numpy().copy() for t in (*c.buffers(), c.scores, c.positions)]


@pytest.mark.parametrize("B,steps", [(1, [20] + [1] * 30), (3, [5, 1, 1, 16, 1, 9] + [1] * 12)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_steps_against_the_oracle(dev, B, steps, interleaved):
    r = Rotary(*rotary_frequencies(48, 1e4, {"type": "yarn", "factor": 4.0}, trained=64), interleaved)
    cache = BoundedKVCache(budget=16, recent=4, slack=3)
    g = torch.Generator().manual_seed(B)
    seen = length = 0
    for T in steps:
        qkv = torch.randn(B, T, (H + 2 * KVH) * D, generator=g).to(dev)
        q = cache.append_rotary(qkv, H, KVH, r)
        length, seen = length + T, seen + T
        assert cache.length() == length and cache.seen == seen
        x = qkv.view(B, T, H + 2 * KVH, D)
        pos = torch.arange(seen - T, seen, device=dev)
        want_q, _ = rotary(x[:, :, :H], None, pos, r.on(dev), interleaved=interleaved, scale=r.scale)
        assert torch.equal(q, want_q)
        kc, ks, vc, vs, sc, ps = buffers(cache)
        assert (sc[:, :, length - T:length] == 0).all()
        assert np.array_equal(ps[:, :, length - T:length], np.broadcast_to(pos.cpu().numpy(), (B, KVH, T)))
        out = cache.attend(q)
        ref, add, ob, ab = bounded.attention_scored(q.cpu().numpy(), kc, ks, vc, vs, [length] * B)
        assert (abs(out.cpu().numpy() - ref) <= ob + 2.0 ** -24 * abs(ref)).all()
        before = buffers(cache)
        want = sc.astype(np.float64) + add
        assert (abs(before[4] - want) <= ab + 2.0 ** -24 * abs(want)).all()
        cache.evict()
        if length > 16 + 3:
            expect, n = bounded.evict(before, before[4], before[5], [length] * B, [seen] * B, 16, 4)
            length = int(n[0])
            assert length == 16
            after = buffers(cache)
            # as bytes: slots never written hold anything, NaN too
            assert all(np.array_equal(a.view(np.uint8), e.view(np.uint8)) for a, e in zip(after, expect))
            assert set(range(seen - 4, seen)) <= set(after[5][0, 0, :16].tolist())
        assert cache.length() == length <= 19


def test_the_cache_s_own_rules(dev):
    cache = BoundedKVCache(budget=8, slack=2)
    k = torch.randn(1, 2, 12, 64, generator=torch.Generator().manual_seed(0)).to(dev)
    cache.append(k[:, :, :5], k[:, :, :5])
    cache.trim(3)
    assert cache.length() == cache.seen == 3
    cache.append(k, k)
    assert cache.length() == cache.seen == 15 and cache.positions[0, 0, :15].tolist() == list(range(15))
    cache.evict()
    assert cache.length() == 8 and cache.seen == 15
    with pytest.raises(SFError, match="cannot be trimmed"):
        cache.trim(4)
    with pytest.raises(SFError):
        cache.set_length(2)
    for bad in ((0,), (8, 9), (8, 2, -1)):
        with pytest.raises(SFError):
            BoundedKVCache(*bad)


def layer(dev, rot):
    c = ModelConfig(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=1e4)
    torch.manual_seed(3)
    return Attention(c, compute_rope_freqs(c, dev), dev, rot)


@pytest.mark.parametrize("rot", [None, Rotary(*rotary_frequencies(32, 1e4), interleaved=True)], ids=["half", "part"])
def test_attention_within_the_bound_equals_the_unbounded_cache(dev, rot):
    """A bound that is never reached: prompts (scored by their last rows), chunks and
    single tokens give what the plain int8 cache gives, which for `rot` holds the same
    codes (2e-5: fp32 sums in another order) and for rotate-half codes of fp32 angles
    (the 2e-3 bar of the attention tests)."""
    attn = layer(dev, rot)
    g = torch.Generator().manual_seed(4)
    plain, bound = QuantizedKVCache(64), BoundedKVCache(budget=200)
    for T in (40, 7, 1, 1, 33, 1):
        x = torch.randn(1, T, 128, generator=g).to(dev)
        with torch.no_grad():
            a, _ = attn(x, plain)
            b, c = attn(x, bound)
        assert c is bound and b.shape == a.shape
        err = ((a - b).norm() / a.norm()).item()
        assert err <= (2e-5 if rot else 2e-3), (T, err)
    assert bound.length() == plain.length() == 83
    # every observed row adds 1 a query head: 4 heads over 2 kv heads, of the prompts' rows the last 16
    assert torch.allclose(bound.scores[0, :, :83].sum(-1).cpu(), torch.full((2,), 2.0 * (16 + 7 + 1 + 1 + 16 + 1)), rtol=1e-5)


def test_batched_attention_over_a_bounded_cache(dev):
    """A batch equals its sequences one by one, past evictions (2e-5 as above)."""
    attn = layer(dev, None)
    g = torch.Generator().manual_seed(5)
    both, each = BoundedKVCache(24, 6, 4), [BoundedKVCache(24, 6, 4) for _ in range(2)]
    for T in [30] + [1] * 12 + [18, 1, 1]:
        x = torch.randn(2, T, 128, generator=g).to(dev)
        with torch.no_grad():
            a, _ = attn(x, both)
            b = torch.cat([attn(x[i:i + 1], each[i])[0] for i in range(2)])
        assert ((a - b).norm() / b.norm()).item() <= 2e-5, T
    assert both.length() == each[0].length() <= 28
    for i in range(2):
        n = both.length()
        assert torch.equal(both.positions[i, :, :n], each[i].positions[0, :, :n])


def test_rotary_over_every_cache_form(dev):
    """The same layer without a cache, over full-precision tensors and over int8 codes."""
    rot = Rotary(*rotary_frequencies(32, 1e4), interleaved=True)
    attn = layer(dev, rot)
    x = torch.randn(1, 9, 128, generator=torch.Generator().manual_seed(6)).to(dev)
    with torch.no_grad():
        full, _ = attn(x)
        head, kv = attn(x[:, :5])
        tail, _ = attn(x[:, 5:], kv)
        int8, _ = attn(x, QuantizedKVCache(16))
    assert ((torch.cat([head, tail], 1) - full).norm() / full.norm()).item() <= 2e-5
    assert ((int8 - full).norm() / full.norm()).item() <= 2e-2  # 8-bit codes


def test_side_streams_keep_to_their_own_workspaces(dev):
    """The same calls, interleaved over two streams, give what one stream gives."""
    g = torch.Generator().manual_seed(9)
    r = Rotary(*rotary_frequencies(64, 1e4))
    qkv = [torch.randn(2, 600 if i == 0 else 1, (H + 2 * KVH) * D, generator=g).to(dev) for i in range(6)]
    logits = torch.randn(4, 40000, generator=g).to(dev)
    u = torch.rand(4, generator=g).to(dev)

    def work():
        cache, out = BoundedKVCache(300, 30, 0), []
        for x in qkv:
            q = cache.append_rotary(x, H, KVH, r)
            out.append(cache.attend(q[:, -8:].contiguous()))
            cache.evict()
            n = cache.length()
            out += [cache.scores[:, :, :n].clone(), cache.positions[:, :, :n].clone(), sample(logits, u, top_p=0.9)]
        return out

    want = work()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_rotary_refuses_outputs_that_share_memory(dev):
    q = torch.zeros(1, 3, 2, 64, device=dev)
    f = Rotary(*rotary_frequencies(64)).on(dev)
    pos = torch.arange(3, device=dev)
    with pytest.raises(SFError, match="share memory"):
        rotary(q, None, pos, f, out_q=q[:, :1].expand(1, 3, 2, 64))
    with pytest.raises(SFError, match="head's dims"):
        rotary(q.transpose(2, 3), None, pos, f[:1])
    for bad in (pos.float(), pos[:2], pos.view(3, 1)):
        with pytest.raises(SFError, match="positions"):
            rotary(q, None, bad, f)
    for bad in (f.float(), f.view(2, 16), torch.cat([f, f])):
        with pytest.raises(SFError):
            rotary(q, None, pos, bad)


def test_sample_refusals(dev):
    x, u = torch.zeros(2, 10, device=dev), torch.zeros(2, device=dev)
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    for args, kw in (((x.t(), u), {}), ((x[0], u), {}), ((x, u.double()), {}), ((x, u[:1]), {}), ((x.double(), u), {}),
                     ((x, u), dict(top_k=u)), ((x, u), dict(temperature=u[:1])), ((x, u), dict(hist=i)),
                     ((x, u[:1]), dict(at=i)), ((x, u), dict(at=i, hist=u)), ((x, u), dict(out=u)),
                     ((x, u), dict(top_p=0.0)), ((x, u), dict(min_p=2.0)), ((x, u), dict(temperature=float("nan")))):
        with pytest.raises(SFError):
            sample(*args, **kw)


@pytest.fixture(scope="module")
def model():
    c = ModelConfig(hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                    num_key_value_heads=1, head_dim=64, vocab_size=1000, rope_theta=1e4, tie_word_embeddings=True)
    return LlamaModel.random_init(c, seed=7, group_size=64, max_seq=96, std=0.15)


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7, top_k=40, top_p=0.9), dict(min_p=0.05), dict(temperature=0.0)])
def test_generate_from_given_numbers(dev, model, kw):
    """Every token is the oracle's draw from the step's logits; replays, callbacks and the
    end of sequence behave as in the greedy path."""
    u = np.random.default_rng(8).random(40).astype(np.float32)
    params = SamplingParams(max_tokens=40, **kw)
    prompt = [5, 17, 300, 4, 9]
    got = generate(model, prompt, params, uniforms=u)
    p = dict(temperature=params.temperature, top_k=params.top_k, top_p=float(np.float32(params.top_p)),
             min_p=float(np.float32(params.min_p)))
    p["temperature"] = float(np.float32(p["temperature"]))
    model.reset()
    model.prefill(prompt, want_logits=True)
    for i, tok in enumerate(got.token_ids):
        want, _, near = bounded.sample(model.logits.cpu().numpy(), float(u[i]), **p)
        assert tok == want or tok in near, (i, tok, want)
        model.token.fill_(tok)
        model.decode_step(logits=True)
        model.pos += 1
    seen = []
    again = generate(model, prompt, params, uniforms=torch.from_numpy(u), on_token=seen.append)
    assert again.token_ids == got.token_ids == seen
    eos = got.token_ids[20]
    cut = generate(model, prompt, params, uniforms=u.tolist(), eos_token_id=eos)
    assert cut.token_ids == got.token_ids[:got.token_ids.index(eos) + 1]
    if params.temperature == 0:
        assert got.token_ids == generate(model, prompt, params).token_ids


def test_generate_refusals(dev, model):
    with pytest.raises(SFError, match="3 uniforms for 4 tokens"):
        generate(model, [1], SamplingParams(max_tokens=4), uniforms=[0.1, 0.2, 0.3])
    with pytest.raises(SFError, match="repetition penalty"):
        generate(model, [1], SamplingParams(max_tokens=1, repetition_penalty=1.2), uniforms=[0.1])
    with pytest.raises(SFError, match="min_p <= 1"):
        generate(model, [1], SamplingParams(max_tokens=1, min_p=1.5), uniforms=[0.1])


def test_sample_token_min_p(dev):
    x = torch.log(torch.tensor([0.5, 0.3, 0.15, 0.05], device=dev))
    g = torch.Generator(device=dev).manual_seed(0)
    drawn = {sample_token(x, SamplingParams(min_p=0.4), generator=g) for _ in range(200)}
    assert drawn == {0, 1}


def test_two_host_threads_on_one_stream(dev):
    """Attention, eviction and sampling called from two threads at once, on the same stream and at
    different sizes, give what one thread gives."""
    import threading

    def inputs(i):
        g = torch.Generator().manual_seed(20 + i)
        return (torch.randn(1 + i, 900 - 500 * i, (H + 2 * KVH) * D, generator=g).to(dev),
                torch.randn(3 + 5 * i, 30000 + 60000 * i, generator=g).to(dev), torch.rand(3 + 5 * i, generator=g).to(dev))

    r = Rotary(*rotary_frequencies(64, 1e4))
    r.on(dev)

    def work(qkv, logits, u):
        out = []
        for _ in range(15):
            cache = BoundedKVCache(200, 20, 0)
            q = cache.append_rotary(qkv, H, KVH, r)
            out.append(cache.attend(q[:, -8:].contiguous()))
            cache.evict()
            out += [cache.scores[:, :, :200].clone(), cache.positions[:, :, :200].clone(), sample(logits, u, top_p=0.9)]
        return out

    data = [inputs(i) for i in range(2)]
    want, got = [work(*d)[:4] for d in data], [None, None]

    def thread(i):
        got[i] = work(*data[i])

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 60
        for j, t in enumerate(got[i]):
            assert torch.equal(t, want[i][j % 4]), (i, j)


def test_buffers_after_a_long_prompt(dev):
    """A prompt far past the bound: after its eviction the cache's buffers have their own size again
    and hold the oracle's choice; the steps behind it run on."""
    r = Rotary(*rotary_frequencies(64, 1e4))
    cache, g = BoundedKVCache(24, 6, 4), torch.Generator().manual_seed(11)
    for T in (500, 1, 1, 300, 1):
        q = cache.append_rotary(torch.randn(2, T, (H + 2 * KVH) * D, generator=g).to(dev), H, KVH, r)
        cache.attend(q[:, -8:].contiguous())
        length, seen, before = cache.length(), cache.seen, buffers(cache)
        cache.evict()
        cache.release()
        if length > 28:
            expect, _ = bounded.evict(before, before[4], before[5], [length] * 2, [seen] * 2, 24, 6)
            for got, want in zip(buffers(cache), expect):
                assert got.shape[2] == 29 and np.array_equal(got[:, :, :24], want[:, :, :24])
        assert cache.capacity == cache.buffers()[0].shape[2] == 29 and cache.length() <= 28


def test_a_layer_s_cache_after_a_long_prompt(dev):
    """The layer's own path leaves a prompt's buffers at the bound."""
    attn, cache = layer(dev, None), BoundedKVCache(24, 6, 4)
    x = torch.randn(2, 400, 128, generator=torch.Generator().manual_seed(12)).to(dev)
    with torch.no_grad():
        for T in (400, 1, 100, 1):
            attn(x[:, :T], cache)
            assert all(t.shape[2] == 29 for t in (*cache.buffers(), cache.scores, cache.positions))
    assert cache.length() == 25 and cache.seen == 502


@pytest.mark.parametrize("rot", [None, lambda: Rotary(*rotary_frequencies(32, 1e4))], ids=["half", "given"])
@pytest.mark.parametrize("where", ["cuda", "cuda:0"])
def test_a_layer_s_first_call_does_not_wait_for_the_device(dev, rot, where):
    """The frequencies are on the device from the layer's construction on: no call copies to or from the host."""
    attn, cache = layer(where, rot and rot()), BoundedKVCache(40, 8, 4)
    x = torch.randn(2, 30, 128, generator=torch.Generator().manual_seed(13)).to(dev)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        with torch.no_grad():
            outs = [attn(x[:, :T], cache)[0] for T in (30, 1, 20, 1)]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    # other frequencies given to the layer later are taken from then on
    other = compute_rope_freqs(ModelConfig(head_dim=64, rope_theta=50.0), dev)
    again, cache = layer(where, rot and rot()), BoundedKVCache(40, 8, 4)
    with torch.no_grad():
        assert torch.equal(again(x, cache)[0], outs[0])
        again.rope_freqs, cache = other, BoundedKVCache(40, 8, 4)
        assert torch.equal(again(x, cache)[0], outs[0]) == (rot is not None)
