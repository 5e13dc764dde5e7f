"""Rotary positions given row by row (sf_rotary, sf_rotary_kv_append) against the
64-bit oracle. Bounds: the oracle's fp32 arithmetic bound plus half a step of the
output's type (torch.finfo(t).eps / 2 of the value)."""

import numpy as np
import pytest
import torch

from oracle import attention as A
from oracle import bounded
from siliconfer_amd.kernels.rotary import rotary, rotary_kv_append

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def freqs(P, theta=1e4):
    return theta ** (-np.arange(P, dtype=np.float64) / P)


def check(got, x, positions, f, interleaved, scale):
    ref, bound = bounded.rotary(x.double().cpu().numpy(), positions.cpu().numpy(), f, interleaved, scale)
    g = got.double().cpu().numpy()
    tol = bound + torch.finfo(got.dtype).eps / 2 * (abs(ref) + bound) + 1e-30
    if got.dtype == torch.float16:
        tol += 2.0 ** -25  # half a subnormal step
    assert (abs(g - ref) <= tol).all(), float((abs(g - ref) / tol).max())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,KVH,D,P", [(1, 1, 14, 2, 64, 32), (2, 3, 4, 1, 128, 32), (1, 257, 2, 2, 80, 16),
                                           (3, 1, 5, 5, 6, 3), (1, 2, 1, 1, 2, 1), (1, 5, 3, 1, 256, 128),
                                           (2, 2, 9, 3, 96, 19), (1, 1, 2, 1, 1024, 512)])
def test_rotary(dev, dtype, interleaved, B, T, H, KVH, D, P):
    g = torch.Generator().manual_seed(B * T + D)
    q = torch.randn(B, T, H, D, generator=g).to(DT[dtype]).to(dev)
    k = torch.randn(B, T, KVH, D, generator=g).to(DT[dtype]).to(dev)
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32).to(dev)
    f = freqs(P)
    for positions in (pos, pos.long(), pos[0].contiguous()):
        yq, yk = rotary(q, k, positions, torch.from_numpy(f).to(dev), interleaved=interleaved, scale=1.25)
        check(yq, q, positions, f, interleaved, 1.25)
        check(yk, k, positions, f, interleaved, 1.25)


def test_far_and_negative_positions(dev):
    q = torch.randn(1, 4, 2, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    pos = torch.tensor([[2 ** 31 - 1, 0, -7, 12345678]], device=dev, dtype=torch.int64)
    f = freqs(32, 1e6)
    y, none = rotary(q, None, pos, torch.from_numpy(f).to(dev))
    assert none is None
    check(y, q, pos, f, False, 1.0)
    assert torch.equal(y[:, 1], q[:, 1])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("P", [32, 16, 5])
def test_strides_and_in_place(dev, dtype, interleaved, P):
    """Heads before rows, slices of a fused buffer at odd offsets, outputs in place."""
    g = torch.Generator().manual_seed(3)
    f = torch.from_numpy(freqs(P)).to(dev)
    pos = torch.arange(100, 107, device=dev)
    fused = torch.randn(2, 7, 6 * 64 + 3, generator=g).to(DT[dtype]).to(dev)
    for off in (0, 3):
        q = fused[:, :, off:off + 256].unflatten(-1, (4, 64))
        k = fused[:, :, off + 256:off + 384].unflatten(-1, (2, 64))
        heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
        want_q, want_k = rotary(q.contiguous(), k.contiguous(), pos, f, interleaved=interleaved)
        got_q, got_k = rotary(q, k, pos, f, interleaved=interleaved)
        assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
        out = torch.empty_like(heads_first)
        got_q, _ = rotary(heads_first, None, pos, f, interleaved=interleaved, out_q=out)
        assert got_q is out and torch.equal(out, want_q)
        own = fused.clone()
        q2, k2 = own[:, :, off:off + 256].unflatten(-1, (4, 64)), own[:, :, off + 256:off + 384].unflatten(-1, (2, 64))
        rotary(q2, k2, pos, f, interleaved=interleaved, out_q=q2, out_k=k2)
        assert torch.equal(q2, want_q) and torch.equal(k2, want_k)
        own[:, :, off:off + 384] = fused[:, :, off:off + 384]
        assert torch.equal(own, fused)  # nothing beside the heads was written


@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("in_dtype", list(DT))
@pytest.mark.parametrize("B,T,H,KVH,D,P,interleaved", [(1, 1, 14, 2, 64, 32, False), (3, 2, 8, 4, 128, 32, True),
                                                       (2, 5, 3, 3, 80, 20, False), (1, 33, 2, 1, 256, 128, True),
                                                       (2, 1, 4, 1, 8, 3, False), (1, 300, 14, 2, 64, 32, False)])
def test_append(dev, scale_dtype, in_dtype, B, T, H, KVH, D, P, interleaved):
    g = torch.Generator().manual_seed(D + T)
    cap = T + 9
    qkv = torch.randn(B, T, (H + 2 * KVH) * D, generator=g).to(DT[in_dtype]).to(dev)
    qkv[0, 0, H * D:(H + 1) * D] = 0  # a zero key: scale 1
    pos = torch.randint(0, 100000, (B, T), generator=g).to(dev)
    lengths = torch.randint(0, 9, (B,), generator=g, dtype=torch.int32).to(dev)
    f = freqs(P)
    codes = [torch.full((B, KVH, cap, D), 99, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.full((B, KVH, cap), 7.0, dtype=scale_dtype, device=dev) for _ in range(2)]
    where = torch.full((B, KVH, cap), -5, dtype=torch.int32, device=dev)
    scores = torch.full((B, KVH, cap), 3.0, device=dev)
    q = rotary_kv_append(qkv, pos, torch.from_numpy(f).to(dev), codes[0], scales[0], codes[1], scales[1], n_heads=H,
                         lengths=lengths, interleaved=interleaved, scale=0.75, slot_positions=where, scores=scores)
    x = qkv.unflatten(-1, (H + 2 * KVH, D))
    check(q, x[:, :, :H], pos, f, interleaved, 0.75)
    turned, _ = rotary(x[:, :, H:H + KVH].float(), None, pos, torch.from_numpy(f).to(dev), interleaved=interleaved,
                       scale=0.75)
    for t, c, s in ((turned, codes[0], scales[0]), (x[:, :, H + KVH:].float(), codes[1], scales[1])):
        rc, rs = A.quantize_kv(t.transpose(1, 2).cpu().numpy())  # of the rotated values in fp32
        for b in range(B):
            n = int(lengths[b])
            assert np.array_equal(c[b, :, n:n + T].cpu().numpy(), rc[b])
            assert np.array_equal(s[b, :, n:n + T].cpu().numpy(), rs[b, ..., 0].astype(s.cpu().numpy().dtype))
            rest = torch.ones(cap, dtype=torch.bool)
            rest[n:n + T] = False
            assert (c[b, :, rest] == 99).all() and (s[b, :, rest] == 7).all()
            assert (where[b, :, n:n + T] == pos[b]).all() and (where[b, :, rest] == -5).all()
            assert (scores[b, :, n:n + T] == 0).all() and (scores[b, :, rest] == 3).all()


def test_append_past_the_capacity(dev):
    """A token whose slot lies past the capacity is not stored; its q is still turned."""
    B, T, H, KVH, D = 2, 4, 2, 1, 64
    qkv = torch.randn(B, T, 4 * D, generator=torch.Generator().manual_seed(0)).to(dev)
    f = torch.from_numpy(freqs(32)).to(dev)
    pos = torch.arange(T, device=dev)
    guard = torch.full((3, B, KVH, 6, D), 99, dtype=torch.int8, device=dev)
    scales = torch.full((2, B, KVH, 6), 7.0, device=dev)
    lengths = torch.tensor([4, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    q = rotary_kv_append(qkv, pos, f, guard[0], scales[0], guard[1], scales[1], n_heads=H, lengths=lengths)
    want, _ = rotary(qkv.unflatten(-1, (4, D))[:, :, :H], None, pos, f)
    assert torch.equal(q, want)
    assert (guard[:2, 0, :, :4] == 99).all() and (guard[:2, 1] == 99).all() and (guard[2] == 99).all()
    assert not (guard[:2, 0, :, 4:] == 99).all(dim=-1).any()


def test_scalar_length_and_16_bit_q(dev):
    qkv = torch.randn(1, 2, 4 * 64, generator=torch.Generator().manual_seed(5)).to(dev)
    f = torch.from_numpy(freqs(32)).to(dev)
    pos = torch.tensor([9, 10], device=dev)
    bufs = lambda: (torch.zeros(1, 1, 8, 64, dtype=torch.int8, device=dev), torch.zeros(1, 1, 8, device=dev))
    (kc, ks), (vc, vs), (kc2, ks2), (vc2, vs2) = (bufs() for _ in range(4))
    a = rotary_kv_append(qkv, pos, f, kc, ks, vc, vs, n_heads=2, lengths=3, out_dtype=torch.bfloat16)
    b = rotary_kv_append(qkv, pos, f, kc2, ks2, vc2, vs2, n_heads=2,
                         lengths=torch.tensor([3], dtype=torch.int32, device=dev))
    assert a.dtype == torch.bfloat16 and torch.equal(a, b.bfloat16())
    assert torch.equal(kc, kc2) and torch.equal(vs, vs2)
