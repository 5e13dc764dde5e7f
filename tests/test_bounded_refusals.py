"""Refusals of the bounded cache's operators and of sampling, without a GPU: the C entry
points check shapes, types, pointers and workspaces before any launch, the Python ones
devices and shapes."""

import subprocess
import sys

import pytest
import torch

from siliconfer_amd import _lib
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.attention import attention_decode_scored
from siliconfer_amd.kernels.eviction import evict
from siliconfer_amd.kernels.rotary import rotary, rotary_kv_append
from siliconfer_amd.kernels.sampling import sample
from siliconfer_amd.model import BoundedKVCache, QuantizedKVCache, Rotary, rotary_frequencies

P = 4096  # a pointer that is never followed: every call below is refused before its launch
F32, F16, BF16 = _lib.SF_F32, _lib.SF_F16, _lib.SF_BF16


def refused(rc, code, text):
    assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())


def rot(**kw):
    a = dict(q=P, q_out=P, k=P, k_out=P, dtype=F32, positions=P, pos_i64=0, pos_per_seq=1, inv_freq=P, pairs=32,
             scale=1.0, interleaved=0, B=1, T=1, H=14, KVH=2, D=64, strides=None, stream=None)
    a.update(kw)
    return _lib.load().sf_rotary(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(q=None), -1, "null pointer"), (dict(k_out=None), -1, "null pointer"), (dict(positions=None), -1, "null"),
    (dict(inv_freq=None), -1, "null"), (dict(dtype=3), -1, "bad dtype"), (dict(pairs=0), -1, "rotated pairs"),
    (dict(pairs=33), -1, "33 rotated pairs in a head of 64"), (dict(pairs=513, D=2048), -2, "at most 512"),
    (dict(B=-1), -1, "invalid rotary shape"), (dict(H=0), -1, "invalid rotary shape"),
    (dict(B=1 << 16, T=1 << 16), -1, "exceed the grid"),
])
def test_rotary_c(kw, code, text):
    refused(rot(**kw), code, text)


def test_nothing_to_do_is_no_error():
    assert rot(T=0) == 0 and rot(B=0, q=None) == 0
    assert append(T=0) == 0
    assert samp(B=0, logits=None) == 0


def append(**kw):
    a = dict(qkv=P, in_dtype=F32, positions=P, pos_i64=0, pos_per_seq=1, inv_freq=P, pairs=32, scale=1.0,
             interleaved=0, q_out=P, q_dtype=F32, k_codes=P, k_scales=P, v_codes=P, v_scales=P, scale_dtype=F16,
             slots=None, scores=None, lengths=None, start=0, B=1, T=1, H=14, KVH=2, D=64, T_cap=128, stream=None)
    a.update(kw)
    return _lib.load().sf_rotary_kv_append(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(start=128), -1, "KV cache overflow: 128 + 1 > capacity 128"), (dict(start=-1), -1, "overflow"),
    (dict(start=2 ** 31 - 1, T=2), -1, "overflow"),
    (dict(H=13), -1, "not a multiple"), (dict(KVH=0), -1, "not a multiple"), (dict(D=66), -2, "D % 8 == 0"),
    (dict(D=264), -2, "D <= 256"), (dict(scale_dtype=BF16), -1, "bad scale dtype"), (dict(q_dtype=9), -1, "bad input"),
    (dict(v_scales=None), -1, "null"), (dict(B=1 << 20, T=1 << 10, lengths=P), -1, "exceed the grid"),
])
def test_append_c(kw, code, text):
    refused(append(**kw), code, text)


def scored(**kw):
    a = dict(q=P, q_dtype=F32, k_codes=P, k_scales=P, v_codes=P, v_scales=P, scale_dtype=F16, scores=P, out=P,
             out_dtype=F32, ws=P, ws_bytes=1 << 40, B=1, Tq=1, H=14, KVH=2, lengths=None, T=100, T_max=100, T_cap=128,
             D=64, scale=0.125, n_splits=0, stream=None)
    a.update(kw)
    return _lib.load().sf_attn_decode_scored_i8kv(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=101), -1, "invalid attention shape"), (dict(T=-1), -1, "invalid attention shape"),
    (dict(T_max=129), -1, "invalid attention shape"), (dict(lengths=P, T_max=-1), -1, "invalid attention shape"),
    (dict(B=0), -1, "invalid attention shape"), (dict(Tq=0), -1, "invalid attention shape"),
    (dict(H=15), -1, "not a multiple"), (dict(D=264), -1, "exceeds kernel's compile-time max 256"),
    (dict(D=60), -2, "multiple of 8"), (dict(Tq=33), -2, "at most 32"), (dict(H=258), -2, "at most 128"),
    (dict(scale_dtype=BF16), -1, "bad scale dtype"), (dict(q_dtype=-1), -1, "bad q/out dtype"),
    (dict(scores=None), -1, "null"), (dict(k_codes=P + 4), -1, "8-byte aligned"), (dict(q=P + 8), -1, "16-byte"),
    (dict(ws=None), -1, "workspace"), (dict(ws=P + 16), -1, "256-byte aligned"), (dict(ws_bytes=100), -1, "too small"),
    (dict(B=70000), -1, "exceed the grid"),
])
def test_scored_c(kw, code, text):
    refused(scored(**kw), code, text)


def ev(**kw):
    a = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, scale_dtype=F16, scores=P, positions=P, lengths=None, T=100,
             seen=None, seen_host=200, budget=50, recent=10, out=P, ws=P, ws_bytes=1 << 40, B=1, KVH=2, T_cap=128,
             D=64, stream=None)
    a.update(kw)
    return _lib.load().sf_kv_evict(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=129), -1, "129 slots of a capacity of 128"), (dict(T=-1), -1, "slots of a capacity"),
    (dict(budget=0, recent=0), -1, "budget > 0"), (dict(recent=51), -1, "recent <= budget"),
    (dict(recent=-1), -1, "0 <= recent"), (dict(D=12), -2, "D % 8 == 0"), (dict(T_cap=1 << 21), -2, "at most 2097151"),
    (dict(KVH=70000), -1, "exceed the grid"), (dict(positions=None), -1, "null"), (dict(out=None), -1, "null"),
    (dict(v_codes=P + 1), -1, "8-byte aligned"), (dict(ws=None), -1, "16-byte aligned"),
    (dict(ws_bytes=8), -1, "too small"), (dict(lengths=P, out=P), -1, "lengths_out must not be lengths"),
])
def test_evict_c(kw, code, text):
    refused(ev(**kw), code, text)


def samp(**kw):
    a = dict(logits=P, dtype=F32, stride=1000, B=2, V=1000, u=P, t=1.0, k=0, p=1.0, m=0.0, ts=None, ks=None, ps=None,
             ms=None, tokens=P, lp=None, at=None, add=0, un=2, hist=None, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.load().sf_sample(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(V=0), -1, "invalid sampling shape"), (dict(B=-1), -1, "invalid sampling shape"),
    (dict(V=(1 << 24) + 1), -2, "at most 16777216"), (dict(dtype=3), -1, "bad dtype"), (dict(stride=-1), -1, "row stride"),
    (dict(t=float("nan")), -1, "temperature"), (dict(k=-1), -1, "top_k >= 0"), (dict(p=0.0), -1, "top_p > 0"),
    (dict(p=float("nan")), -1, "top_p > 0"), (dict(m=1.5), -1, "min_p <= 1"), (dict(m=-0.1), -1, "0 <= min_p"),
    (dict(u=None), -1, "null"), (dict(tokens=None), -1, "null"), (dict(ws=None), -1, "256-byte aligned"),
    (dict(at=P, un=1), -1, "1 numbers for 2 rows"), (dict(hist=P), -1, "hist without at"),
    (dict(ws_bytes=100), -1, "too small"), (dict(B=1 << 30, V=1 << 20), -1, "exceed the grid"),
])
def test_sample_c(kw, code, text):
    refused(samp(**kw), code, text)


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.sf_attn_scored_workspace_bytes(1, 1, 14, 3, 100, 64, 0) == 0  # 14 heads over 3
    one = lib.sf_attn_scored_workspace_bytes(1, 1, 14, 2, 1000, 64, 4)
    assert one >= 14 * (4 * 64 + 4 * 2 + 1000) * 4
    assert lib.sf_attn_scored_workspace_bytes(64, 32, 128, 8, 131072, 128, 0) > 2 ** 32
    assert lib.sf_kv_evict_workspace_bytes(2, 4, 100, 300) >= 2 * 4 * (4 + 100 * 8)
    assert lib.sf_kv_evict_workspace_bytes(2, 4, 300, 100) > 0
    assert lib.sf_sample_workspace_bytes(3, 0) == 0 and lib.sf_sample_workspace_bytes(3, 100) > 0


def test_python_layers_refuse_host_tensors_and_shapes():
    q, f, pos = torch.zeros(1, 1, 2, 64), torch.zeros(32, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(SFError, match="device tensor"):
        rotary(q, None, pos, f)
    kc, ks = torch.zeros(1, 1, 8, 64, dtype=torch.int8), torch.zeros(1, 1, 8)
    with pytest.raises(SFError, match="device tensor"):
        rotary_kv_append(torch.zeros(1, 1, 256), pos, f, kc, ks, kc, ks, n_heads=2, lengths=0)
    with pytest.raises(SFError, match="device tensor"):
        attention_decode_scored(torch.zeros(1, 2, 64), kc, ks, kc, ks, ks, lengths=3)
    with pytest.raises(SFError, match="device tensor"):
        evict(kc, ks, kc, ks, ks, ks.int(), 8, 8, 4)
    with pytest.raises(SFError, match="device tensor"):
        sample(torch.zeros(2, 10), torch.zeros(2))


def test_cache_checks():
    c, s, i = torch.zeros(1, 2, 8, 64, dtype=torch.int8), torch.zeros(1, 2, 8), torch.zeros(1, 2, 8, dtype=torch.int32)
    cpu = torch.device("cpu")
    _lib.check_cache(cpu, c, s, c, s, i, s)
    for bad in ((c.short(), s, c, s, i, s), (c, s.half(), c, s, i, s), (c, s.bfloat16(), c, s.bfloat16(), i, s),
                (c, s, c, s, i.long(), s), (c, s, c, s, i, s.double()), (c, s[:, :, :7], c, s, i, s),
                (c, s.unsqueeze(-1), c, s, i, s), (c.transpose(2, 3), s, c, s, i, s)):
        with pytest.raises(SFError):
            _lib.check_cache(cpu, *bad)
    for bad in (-1, 2 ** 31, torch.zeros(2), torch.zeros(3, dtype=torch.int32)):
        with pytest.raises(SFError):
            _lib.lengths_arg(bad, 2, cpu)


def test_a_bounded_cache_starts_again():
    """trim(0) begins a new sequence in the same buffers, tokens dropped or not."""
    cache = BoundedKVCache(4, slack=2)
    for length, seen in ((4, 9), (5, 5), (0, 0)):
        cache._len, cache.seen = length, seen
        cache.trim(0)
        assert cache.length() == 0 and cache.seen == 0
    cache._len, cache.seen = 4, 9
    with pytest.raises(SFError, match="cannot be trimmed"):
        cache.trim(3)
    cache.trim(9)
    assert cache.length() == 4 and cache.seen == 9


def test_a_bounded_cache_gives_a_prompt_s_buffers_back(monkeypatch):
    """Past an eviction the buffers go back to budget + slack + 1 slots with what was kept: by
    release(), or by the first append that fits. (The eviction itself is stood in for on the host.)"""
    from siliconfer_amd.kernels import eviction

    def newest(kc, ks, vc, vs, scores, positions, length, seen, budget, recent):
        for t in (kc, ks, vc, vs, scores, positions):
            t[:, :, :budget] = t[:, :, length - budget:length].clone()

    monkeypatch.setattr(eviction, "evict", newest)
    cache = BoundedKVCache(20, 5, slack=3)

    def fill(T):  # what append_rotary does, without its kernel
        n = cache._len
        cache.reserve(2, 3, 16, n + T, torch.device("cpu"))
        for i, t in enumerate((*cache.buffers(), cache.scores, cache.positions)):
            at = torch.arange(cache.seen, cache.seen + T) + i
            t[:, :, n:n + T] = at.to(t.dtype).view(1, 1, T, *[1] * (t.dim() - 3))
        cache._len, cache.seen = n + T, cache.seen + T

    def check(first, n):
        for i, t in enumerate((*cache.buffers(), cache.scores, cache.positions)):
            want = (torch.arange(first, first + n) + i).to(t.dtype)
            assert t.shape[2] == 24 == cache.capacity and t.is_contiguous()
            assert torch.equal(t[:, :, :n].reshape(2, 3, n, -1)[..., 0], want.expand(2, 3, n))

    fill(7)
    assert cache.buffers()[0].shape[2] == 24
    cache.evict()
    check(0, 7)
    fill(100)
    assert cache.buffers()[0].shape[2] >= 107
    cache.evict()
    assert cache.length() == 20 and cache.seen == 107
    cache.release()
    check(87, 20)
    fill(100)
    cache.evict()
    fill(2)
    check(187, 22)
    before = [t.data_ptr() for t in cache.buffers()]
    for _ in range(7):  # a decode loop stays in its buffers
        fill(1)
        cache.evict()
    assert [t.data_ptr() for t in cache.buffers()] == before and cache.length() == 21
    cache.trim(0)
    fill(200)
    assert cache.buffers()[0].shape[2] >= 200
    cache.release()  # (does not fit)
    assert cache.buffers()[0].shape[2] >= 200 and cache.length() == 200
    cache.trim(22)
    fill(2)
    check(0, 24)


@pytest.mark.parametrize("scale_dtype,size", [(torch.float16, 2), (torch.float32, 4)])
def test_a_bounded_cache_s_size(scale_dtype, size):
    """nbytes counts a slot's codes and scales, and its score and position a kv head."""
    cache = BoundedKVCache(20, scale_dtype=scale_dtype)
    assert cache.nbytes() == 0
    cache.reserve(2, 3, 16, 10, torch.device("cpu"))
    cache._len = 10
    assert cache.nbytes() == sum(t[:, :, :10].numel() * t.element_size()
                                 for t in (*cache.buffers(), cache.scores, cache.positions))
    assert cache.nbytes() == 2 * 3 * 10 * (2 * (16 + size) + 8)


COUNT = r"""
extern "C" {
int launches = 0;
unsigned __hipPushCallConfiguration(...) { ++launches; return 1; }  // (not 0: the launch is left out)
}
"""
ASK = """
import ctypes, sys
count = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)  # found before the runtime's own
lib = ctypes.CDLL(sys.argv[2])
i, p, z = ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t
f = lib.sf_attn_decode_scored_i8kv
f.argtypes = [p, i, p, p, p, p, i, p, p, i, p, z, i, i, i, i, p, i, i, i, i, ctypes.c_float, i, p]
for T_max in map(int, sys.argv[3:]):
    print(f(4096, 0, 4096, 4096, 4096, 4096, 1, 4096, 4096, 0, 4096, 1 << 62, 65535, 1, 1, 1, 4096, 0, T_max, T_max, 64,
            0.125, 1, None), ctypes.c_int.in_dll(count, "launches").value)
"""


def test_scored_attention_checks_both_grids_before_a_launch(tmp_path):
    """65535 sequences of 2^23 slots, 256 a workgroup of the second launch, are past 2^31 workgroups with
    its rows: refused with nothing launched (the launch is stood in for by a counter)."""
    (tmp_path / "count.cpp").write_text(COUNT)
    so = tmp_path / "count.so"
    subprocess.run(["g++", "-shared", "-fPIC", str(tmp_path / "count.cpp"), "-o", str(so)], check=True)
    got = subprocess.run([sys.executable, "-c", ASK, str(so), _lib.LIB_PATH, str(1 << 23), str((1 << 23) + 1), "4096"],
                         check=True, capture_output=True, text=True, timeout=100).stdout.split()
    assert got[:4] == ["-1", "0", "-1", "0"], got
    assert got[5] == "2", got  # (the counter counts: a call within the grid has its two launches)


def test_scored_attention_s_longest_cache():
    """Slots are rounded up to tiles and blocks in 32 bits: lengths within 255 of 2^31 are refused by name."""
    lib = _lib.load()
    for T in (0x7fffff01, 0x7fffffe0, 0x7fffffff):
        refused(scored(ws_bytes=1 << 62, T=T, T_max=T, T_cap=T, D=8), -2, "2147483392 slots")
        assert lib.sf_attn_scored_workspace_bytes(1, 1, 14, 2, T, 8, 0) == 0
    assert lib.sf_attn_scored_workspace_bytes(1, 1, 14, 2, 0x7fffff00, 8, 0) > 14 * 4 * 0x7fffff00


@pytest.mark.parametrize("big", [2 ** 32 + 5, 2 ** 31, -(2 ** 32) + 5])
def test_numbers_past_32_bits_are_refused(big):
    """They would reach the C entries cut to their low half."""
    kc, ks = torch.zeros(1, 1, 8, 64, dtype=torch.int8), torch.zeros(1, 1, 8)
    q, x, u = torch.zeros(1, 2, 64), torch.zeros(2, 10), torch.zeros(2)
    for call in (lambda: evict(kc, ks, kc, ks, ks, ks.int(), 8, 8, big),
                 lambda: evict(kc, ks, kc, ks, ks, ks.int(), 8, 8, 4, big),
                 lambda: sample(x, u, top_k=big), lambda: sample(x, u, at=ks, at_add=big),
                 lambda: attention_decode_scored(q, kc, ks, kc, ks, ks, lengths=3, add=big),
                 lambda: attention_decode_scored(q, kc, ks, kc, ks, ks, lengths=3, max_length=big),
                 lambda: attention_decode_scored(q, kc, ks, kc, ks, ks, lengths=3, n_splits=big)):
        with pytest.raises(SFError, match="32 bits"):
            call()


def test_a_refused_append_leaves_no_buffers_behind():
    """Buffers made for a call that is then refused would not fit the next, right one."""
    rot = Rotary(*rotary_frequencies(64))
    cpu = torch.zeros(1, 3, 6 * 64)
    for qkv, heads, kv_heads in ((cpu, 4, 1), (torch.zeros(3, 6 * 64), 4, 1), (torch.zeros(1, 3, 385), 4, 1),
                                 (torch.zeros(1, 3, 7 * 64), 3, 2), (torch.zeros(1, 3, 6 * 60), 4, 1),
                                 (torch.zeros(1, 3, 6 * 264), 4, 1), (cpu, 4, 0), (cpu, 0, 1)):
        cache = BoundedKVCache(16)
        with pytest.raises(SFError):
            cache.append_rotary(qkv, heads, kv_heads, rot)
        assert cache.buffers() == (None,) * 4 and cache.length() == cache.seen == 0
    k = torch.zeros(1, 2, 3, 64)
    for made in (BoundedKVCache(16), QuantizedKVCache(16)):
        for a, b in ((k, k), (k, k[:, :1]), (k.double(), k.double())):
            with pytest.raises(SFError):
                made.append(a, b)
            assert made.buffers() == (None,) * 4 and made.length() == 0


def test_a_reservation_in_a_bounded_cache_is_kept(monkeypatch):
    """reserve() holds through appends and evictions that cut nothing; buffers go back past a cut only."""
    from siliconfer_amd.kernels import eviction
    monkeypatch.setattr(eviction, "evict", lambda *a: None)
    cache, cpu = BoundedKVCache(20, 5, slack=3), torch.device("cpu")
    cache.reserve(1, 2, 16, 400, cpu)
    first = [t.data_ptr() for t in (*cache.buffers(), cache.scores, cache.positions)]
    for n in range(1, 24):
        cache.reserve(1, 2, 16, n, cpu)  # as an append does
        cache._len = cache.seen = n
        cache.evict()
    assert [t.data_ptr() for t in (*cache.buffers(), cache.scores, cache.positions)] == first
    cache.reserve(1, 2, 16, 24, cpu)
    cache._len = cache.seen = 24
    cache.evict()
    assert cache.length() == 20
    cache.reserve(1, 2, 16, 21, cpu)
    assert cache.buffers()[0].shape[2] == 24
