"""The 4-bit cache: codes and parameters against the 64-bit oracle (equal, a code next to a
border aside), the turned q to the oracle's bound, slots that are left alone, reading back."""

import numpy as np
import pytest
import torch

from oracle import bounded
from oracle import kv_q4 as O
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.kv_q4 import dequantize_kv_q4, kv_append_q4, rotary_kv_append_q4

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def buffers(B, KVH, cap, D, group, dev):
    """Two caches' buffers, filled with what must not change."""
    g = torch.Generator().manual_seed(99)
    out = []
    for _ in range(2):
        out += [torch.randint(0, 256, (B, KVH, cap, D // 2), generator=g, dtype=torch.uint8).to(dev),
                torch.randn(B, KVH, cap, D // group, 2, generator=g).half().to(dev)]
    return out


def same(codes, params, before, x, slots, group, turned=False):
    """x [B, KVH, T, D] in 64 bits lies at slots[b] .. of the buffers, and the rest is as it was."""
    T, cap = x.shape[2], codes.shape[2]
    want_c, want_p = (t.cpu().numpy().copy() for t in before)
    c, s, m, border = O.quantize(x, group)
    loose = np.zeros(want_c.shape[:-1] + (x.shape[-1],), bool)
    for b, at in enumerate(slots):
        for t in range(T):
            if at >= 0 and at + t < cap:
                want_c[b, :, at + t] = O.pack(c[b, :, t])
                want_p[b, :, at + t, :, 0], want_p[b, :, at + t, :, 1] = s[b, :, t], m[b, :, t]
                # values as they came have exact borders (ties too); of turned ones cos and sin are off by 2e-14, the
                # norm by a few 2^-53: 1e-11 of a step at the most here
                loose[b, :, at + t] = turned & (border[b, :, t] < 1e-9) & (border[b, :, t] > 0)
    assert (loose.mean() < 1e-6) and np.array_equal(params.cpu().numpy(), want_p, equal_nan=True)
    got = codes.cpu().numpy()
    for half, shift in ((0, 0), (1, 4)):
        assert (((got >> shift & 15) == (want_c >> shift & 15)) | loose[..., half::2]).all()


GEOMETRIES = [(14, 2, 64, 64, 32), (4, 1, 128, 64, 64), (3, 3, 128, 32, 20), (2, 2, 80, 80, 7), (9, 3, 96, 32, 48),
              (2, 1, 256, 128, 128), (5, 1, 16, 16, 8), (2, 1, 256, 256, 1), (1, 1, 192, 64, 33), (32, 8, 128, 128, 64),
              (3, 1, 48, 48, 12), (2, 2, 112, 112, 56)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,KVH,D,group,P", GEOMETRIES)
def test_fused_rows(dev, dtype, interleaved, H, KVH, D, group, P):
    B, T, cap = 3, 5, 40
    g = torch.Generator().manual_seed(D + P)
    qkv = torch.randn(B, T, (H + 2 * KVH) * D, generator=g).to(DT[dtype]).to(dev)
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32).to(dev)
    w = (1 + 0.3 * torch.randn(2, D, generator=g)).to(DT[dtype]).to(dev)
    f = 1e4 ** (-np.arange(P, dtype=np.float64) / P)
    inv = torch.from_numpy(f).to(dev)
    x = qkv.double().cpu().numpy().reshape(B, T, H + 2 * KVH, D)
    lengths = torch.tensor([7, 37, -1], dtype=torch.int32, device=dev)  # the second runs over the end, the third has no slots
    for qw, kw in ((None, None), (w[0], w[1]), (None, w[1])):
        kc, kp, vc, vp = buffers(B, KVH, cap, D, group, dev)
        before = [t.clone() for t in (kc, kp, vc, vp)]
        for out in (torch.float32, DT[dtype]):
            q = rotary_kv_append_q4(qkv, pos, inv, kc, kp, vc, vp, n_heads=H, lengths=lengths, q_weight=qw, k_weight=kw,
                                    eps=1e-5, interleaved=interleaved, scale=1.5, out_dtype=out)
            side = lambda t, w: t if w is None else t * O.inv_rms(t, 1e-5)[0] * w.double().cpu().numpy()
            n = side(x[:, :, :H], qw)
            want, bound = bounded.rotary(n, pos.cpu().numpy(), f, interleaved, float(np.float32(1.5)))
            tol = bound + torch.finfo(out).eps / 2 * (abs(want) + bound) + 2.0 ** -25
            assert q.dtype is out and (abs(q.double().cpu().numpy() - want) <= tol).all()
        k = bounded.rotary(side(x[:, :, H:H + KVH], kw), pos.cpu().numpy(), f, interleaved, 1.5)[0]
        same(kc, kp, before[:2], k.transpose(0, 2, 1, 3), lengths.tolist(), group, True)
        same(vc, vp, before[2:], x[:, :, H + KVH:].transpose(0, 2, 1, 3), lengths.tolist(), group)
    # one length for all, positions a row for all
    kc, kp, vc, vp = buffers(B, KVH, cap, D, group, dev)
    before = [t.clone() for t in (kc, kp, vc, vp)]
    rotary_kv_append_q4(qkv, pos[0].long().contiguous(), inv, kc, kp, vc, vp, n_heads=H, lengths=cap - T)
    k = bounded.rotary(x[:, :, H:H + KVH], pos[0].cpu().numpy(), f)[0]
    same(kc, kp, before[:2], k.transpose(0, 2, 1, 3), [cap - T] * B, group, True)
    with pytest.raises(SFError, match="overflow"):
        rotary_kv_append_q4(qkv, pos, inv, kc, kp, vc, vp, n_heads=H, lengths=cap - T + 1)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("KVH,D,group", [(2, 64, 32), (1, 128, 128), (3, 80, 80), (2, 256, 64), (1, 96, 96), (1, 16, 16)])
def test_turned_rows_and_reading_back(dev, dtype, KVH, D, group):
    B, T, cap = 2, 6, 17
    g = torch.Generator().manual_seed(D)
    k, v = torch.randn(2, B, T, KVH, D, generator=g).to(DT[dtype]).to(dev).transpose(2, 3)  # strided rows
    kc, kp, vc, vp = buffers(B, KVH, cap, D, group, dev)
    before = [t.clone() for t in (kc, kp, vc, vp)]
    kv_append_q4(k, v, kc, kp, vc, vp, lengths=3)
    same(kc, kp, before[:2], k.double().cpu().numpy(), [3] * B, group)
    same(vc, vp, before[2:], v.double().cpu().numpy(), [3] * B, group)
    odd = torch.randn(B, KVH, T, D + 3, generator=g).to(DT[dtype]).to(dev)[..., 3:]  # rows off 16 bytes are copied
    kv_append_q4(odd, odd, kc, kp, vc, vp, lengths=torch.full((B,), 3, dtype=torch.int32, device=dev))
    same(kc, kp, before[:2], odd.double().cpu().numpy(), [3] * B, group)
    for out in DT.values():
        for a, b in ((0, cap), (3, 9), (16, 17), (5, 5)):
            got = dequantize_kv_q4(kc[:, :, a:b], kp[:, :, a:b], out)
            want = O.values(kc[:, :, a:b].cpu().numpy(), kp[:, :, a:b].float().cpu().numpy())[0]
            # m + s code rounded to fp32, then to the type
            assert got.dtype is out and got.shape == want.shape
            tol = (torch.finfo(out).eps / 2 + 2.0 ** -24) * (1 + 2.0 ** -8) * abs(want) + 2.0 ** -25
            assert (abs(got.double().cpu().numpy() - want) <= tol).all()
    # half a step of s, half a step of m's and s's rounding (2^-11 of m, of 15 s) and of fp32
    new = dequantize_kv_q4(kc[:, :, 3:9], kp[:, :, 3:9])
    s, m = (kp[:, :, 3:9, :, i].float().repeat_interleave(group, -1) for i in (0, 1))
    assert ((new - odd.float()).abs() <= 0.5 * s + 2.0 ** -10 * (m.abs() + 15 * s)).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,KVH,D,group,P", [(32, 8, 128, 64, 64), (14, 2, 64, 32, 32), (6, 3, 80, 80, 12), (3, 1, 256, 128, 128),
                                             (1, 1, 16, 16, 8)])
def test_many_rows_equal_their_parts(dev, H, KVH, D, group, P, interleaved):
    """Enough heads that a workgroup takes several in turn: the bits of the same rows in parts, and
    nothing else of the cache."""
    hb = 256 // (1 << (D // 8 - 1).bit_length())  # heads that a workgroup's threads hold
    B = 2
    T = 3 * 1024 * hb // (B * (H + 2 * KVH)) + 37
    part = T // 3 + 1
    g = torch.Generator(device=dev).manual_seed(D)
    qkv = torch.randn(B, T, (H + 2 * KVH) * D, generator=g, device=dev).half()
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32, device=dev)
    w = (1 + 0.3 * torch.randn(2, D, generator=g, device=dev)).half()
    inv = torch.from_numpy(1e4 ** (-np.arange(P, dtype=np.float64) / P)).to(dev)
    lengths = torch.tensor([5, 90], dtype=torch.int32, device=dev)
    one, two = (buffers(B, KVH, T + 50, D, group, dev) for _ in range(2))  # (the second sequence runs over the end)
    how = dict(n_heads=H, q_weight=w[0], k_weight=w[1], interleaved=interleaved, out_dtype=torch.float16)
    q = rotary_kv_append_q4(qkv, pos, inv, *one, lengths=lengths, **how)
    parts = [rotary_kv_append_q4(qkv[:, a:a + part].contiguous(), pos[:, a:a + part].contiguous(), inv, *two, lengths=lengths + a,
                                 **how) for a in range(0, T, part)]
    assert torch.equal(torch.cat(parts, 1), q)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(one, two))


@pytest.mark.parametrize("H,KVH,D,group,P", [(32, 8, 128, 64, 64), (1, 1, 16, 16, 4), (14, 2, 64, 32, 32)])
def test_many_sequences_equal_one_by_one(dev, H, KVH, D, group, P):
    """One token each of more sequences than a workgroup takes heads, lengths of their own."""
    B = 1500
    g = torch.Generator(device=dev).manual_seed(D)
    qkv = torch.randn(B, 1, (H + 2 * KVH) * D, generator=g, device=dev)
    pos = torch.randint(0, 1 << 20, (B, 1), generator=g, device=dev)
    inv = torch.from_numpy(1e4 ** (-np.arange(P, dtype=np.float64) / P)).to(dev)
    lengths = torch.randint(-2, 9, (B,), generator=g, dtype=torch.int32, device=dev)
    one, two = (buffers(B, KVH, 7, D, group, dev) for _ in range(2))
    q = rotary_kv_append_q4(qkv, pos, inv, *one, n_heads=H, lengths=lengths)
    some = [0, 1, 2, 127, 128, 511, 777, 1498, 1499]
    for i in some:
        at = slice(i, i + 1)
        part = [t[at].clone() for t in two]  # (buffers of their own: a cache starts on 16 bytes)
        y = rotary_kv_append_q4(qkv[at], pos[at], inv, *part, n_heads=H, lengths=lengths[at])
        assert torch.equal(y, q[at])
        assert all(torch.equal(a[at].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, part)), i


@pytest.mark.parametrize("D,group", [(48, 48), (80, 80), (112, 112), (96, 32), (240, 240), (256, 64), (64, 64)])
def test_reading_back_many_slots(dev, D, group):
    """Slots that several workgroups share, at words a slot that divide a workgroup's and that do not."""
    kc, kp, _, _ = buffers(2, 3, 307, D, group, dev)
    for a, b in ((0, 307), (6, 300)):
        want = O.values(kc[:, :, a:b].cpu().numpy(), kp[:, :, a:b].float().cpu().numpy())[0]
        for out in DT.values():
            got = dequantize_kv_q4(kc[:, :, a:b], kp[:, :, a:b], out)
            # m + s code rounded to fp32, then to the type
            tol = (torch.finfo(out).eps / 2 + 2.0 ** -24) * (1 + 2.0 ** -8) * abs(want) + 2.0 ** -25
            assert (abs(got.double().cpu().numpy() - want) <= tol).all()


def test_ties_constants_and_ranges(dev):
    """Exact ties go to the even code; a constant group is its minimum; a range past fp16's ends
    is held at them; what is not finite reads back as NaN, in its group alone."""
    x = torch.zeros(1, 1, 7, 64, device=dev)
    x[0, 0, 0, :32] = torch.arange(32, device=dev).float() * 0.5  # 0, 0.5 .. 15.5: s = f16(15.5 / 15), no ties
    x[0, 0, 1, :31] = torch.arange(31, device=dev).float() * 0.5  # 0 .. 15: s = 1, every half a tie
    x[0, 0, 2] = 2.5
    x[0, 0, 3, 0], x[0, 0, 3, 1] = 1e30, -1e30
    x[0, 0, 4, 40] = float("nan")
    x[0, 0, 5, 3] = float("-inf")
    x[0, 0, 6] = 1e-12 * torch.arange(64, device=dev)
    kc, kp, vc, vp = buffers(1, 1, 8, 64, 32, dev)
    before = [t.clone() for t in (kc, kp, vc, vp)]
    kv_append_q4(x, x, kc, kp, vc, vp, lengths=1)
    c, s, m, _ = O.quantize(x.double().cpu().numpy(), 32)
    assert torch.equal(kc[0, 0, 1:].cpu(), torch.from_numpy(O.pack(c)[0, 0]))
    assert np.array_equal(kp[0, 0, 1:].cpu().numpy(), np.stack([s, m], -1)[0, 0], equal_nan=True)
    assert torch.equal(kc[:, :, :1], before[0][:, :, :1]) and torch.equal(vc, kc.where(kc == vc, vc))
    y = dequantize_kv_q4(kc, kp)[0, 0, 1:]
    assert (c[0, 0, 1, :31:2] == np.arange(16)).all() and (c[0, 0, 1, 1:31:2] % 2 == 0).all()
    assert (y[2] == 2.5).all() and y[3].isfinite().all() and y[3, 1] == -65504
    assert y[4, 32:].isnan().all() and y[4, :32].isfinite().all() and y[5, :32].isnan().all() and (y[6] == 0).all()


def test_streams_and_graphs(dev):
    """Replays append where the device lengths say, as the eager call does."""
    g = torch.Generator().manual_seed(8)
    B, H, KVH, D = 2, 4, 2, 128
    qkv = torch.randn(B, 1, (H + 2 * KVH) * D, generator=g).to(dev)
    inv = torch.from_numpy(1e4 ** (-np.arange(64) / 64.0)).to(dev)
    w = torch.ones(2, D, device=dev)
    held, eager = ([torch.zeros_like(t) for t in buffers(B, KVH, 9, D, 64, dev)] for _ in range(2))
    lengths, pos = torch.tensor([0, 3], dtype=torch.int32, device=dev), torch.tensor([[0], [3]], dtype=torch.int32, device=dev)
    call = lambda bufs, ln, p: rotary_kv_append_q4(qkv, p, inv, *bufs, n_heads=H, lengths=ln, q_weight=w[0], k_weight=w[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(held, lengths, pos)
        lengths.add_(1)
        pos.add_(1)
    ln, p = lengths.clone(), pos.clone()
    for i in range(4):
        graph.replay()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            want = call(eager, ln, p)
        torch.cuda.synchronize()
        ln += 1
        p += 1
        assert torch.equal(q, want) and all(torch.equal(a, b) for a, b in zip(held, eager)), i
    assert lengths.tolist() == [4, 7]


def test_refusals(dev):
    kc, kp, vc, vp = buffers(1, 2, 8, 64, 32, dev)
    k = torch.randn(1, 2, 3, 64, device=dev)
    inv, pos = torch.ones(32, dtype=torch.float64, device=dev), torch.arange(3, device=dev)
    qkv = torch.randn(1, 3, 8 * 64, device=dev)
    for bufs in ((kc.char(), kp, vc, vp), (kc, kp.float(), vc, vp), (kc, kp, vc[:, :, :4], vp), (kc, kp[:, :, :4], vc, vp[:, :, :4]),
                 (kc.transpose(1, 2), kp, vc, vp), (kc.cpu(), kp, vc, vp), (kc, kp[..., :1], vc, vp[..., :1])):
        with pytest.raises(SFError, match="k/v codes must be"):
            kv_append_q4(k, k, *bufs, lengths=0)
        with pytest.raises(SFError, match="k/v codes must be"):
            rotary_kv_append_q4(qkv, pos, inv, *bufs, n_heads=4, lengths=0)
    for a, text in (((k, k.half()), "same shape"), ((k[:, :1], k[:, :1]), "do not match a cache"), ((k.cpu(), k.cpu()), "device")):
        with pytest.raises(SFError, match=text):
            kv_append_q4(*a, kc, kp, vc, vp, lengths=0)
    with pytest.raises(SFError, match="overflow"):
        kv_append_q4(k, k, kc, kp, vc, vp, lengths=6)
    for bad, text in ((dict(n_heads=5), "does not match"), (dict(q_weight=inv), "q_weight"), (dict(positions=pos[:2]), "positions"),
                      (dict(inv_freq=inv.float()), "inv_freq"), (dict(qkv=qkv.int()), "dtype")):
        a = dict(qkv=qkv, positions=pos, inv_freq=inv, n_heads=4, lengths=0, q_weight=None)
        with pytest.raises(SFError, match=text):
            rotary_kv_append_q4(k_codes=kc, k_params=kp, v_codes=vc, v_params=vp, **{**a, **bad})
    with pytest.raises(SFError, match="codes must be uint8"):
        dequantize_kv_q4(kc, kp.float())
    bad = torch.zeros(1, 1, 2, 3, 2, dtype=torch.float16, device=dev)  # groups of 16 in a head of 48
    with pytest.raises(SFError, match="group=16"):
        dequantize_kv_q4(torch.zeros(1, 1, 2, 24, dtype=torch.uint8, device=dev), bad)
