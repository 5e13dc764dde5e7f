"""Heads normed and turned in one pass, and the gradients, against the 64-bit oracle (its
bounds plus half a step of the output's type) and against differences."""

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.rotary import qk_norm_rotary

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def freqs(P, theta=1e4):
    return theta ** (-np.arange(P, dtype=np.float64) / P)


def close(got, want, bound):
    g = got.detach().double().cpu().numpy()
    tol = bound * (1 + 2.0 ** -8) + torch.finfo(got.dtype).eps / 2 * abs(want) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    assert g.shape == want.shape and (abs(g - want) <= tol).all(), float((abs(g - want) / tol).max())


SHAPES = [(1, 1, 14, 2, 64, 32), (2, 3, 4, 1, 128, 64), (1, 65, 2, 2, 80, 16), (3, 1, 5, 5, 6, 3), (1, 2, 1, 1, 2, 1),
          (1, 5, 3, 1, 256, 128), (2, 2, 9, 3, 96, 19), (1, 300, 32, 8, 128, 32), (2, 7, 1, 1, 16, 8), (1, 9, 1, 1, 8, 4),
          (1, 4, 3, 1, 255, 100), (1, 3, 2, 1, 250, 2)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,KVH,D,P", SHAPES)
def test_forward_and_gradients(dev, dtype, interleaved, B, T, H, KVH, D, P):
    g = torch.Generator().manual_seed(B * T + D)
    new = lambda *s: torch.randn(*s, generator=g)
    q = (2 * new(B, T, H, D)).to(DT[dtype]).to(dev).requires_grad_()
    k = (2 * new(B, T, KVH, D)).to(DT[dtype]).to(dev).requires_grad_()
    wq, wk = ((1 + 0.3 * new(D)).to(dev).requires_grad_() for _ in range(2))
    gq, gk = (new(B, T, n, D).to(DT[dtype]).to(dev) for n in (H, KVH))
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32).to(dev)
    f = freqs(P)
    how = dict(eps=1e-5, interleaved=interleaved, scale=1.25)
    y = qk_norm_rotary(q, k, pos, torch.from_numpy(f).to(dev), wq, wk, **how)
    got = torch.autograd.grad(y, (q, k, wq, wk), (gq, gk))
    p = pos.cpu().numpy()
    for i, (x, w, gy) in enumerate(((q, wq, gq), (k, wk, gk))):
        x64, w64, g64 = (t.detach().double().cpu().numpy() for t in (x, w, gy))
        close(y[i], *O.qk_norm_rotary(x64, w64, p, f, **how))
        dx, dw, edx, edw = O.qk_norm_rotary_backward(x64, w64, g64, p, f, **how)
        close(got[i], dx, edx)
        close(got[2 + i], dw, edw)
    with torch.no_grad():
        again = qk_norm_rotary(q, k, pos.long(), torch.from_numpy(f).to(dev), wq, wk, **how)
        one = qk_norm_rotary(q, None, pos, torch.from_numpy(f).to(dev), wq, **how)
    assert torch.equal(again[0], y[0]) and torch.equal(again[1], y[1]) and torch.equal(one[0], y[0]) and one[1] is None


@pytest.mark.parametrize("B,T,H,KVH,D,P", [(2, 32768, 1, 1, 8, 4), (2, 40001, 1, 1, 6, 3), (3, 1, 40000, 33000, 8, 4),
                                           (2, 2, 32767, 1, 16, 8), (5000, 1, 3, 1, 8, 4), (3, 32767, 1, 1, 8, 2)])
def test_many_rows_heads_and_sequences(dev, B, T, H, KVH, D, P):
    """Past what a lane divides by a product: rows a sequence, heads a row, sequences of a workgroup."""
    g = torch.Generator().manual_seed(T)
    q, k = (torch.randn(B, T, n, D, generator=g).to(dev).requires_grad_() for n in (H, KVH))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(dev).requires_grad_() for _ in range(2))
    gq, gk = (torch.randn(B, T, n, D, generator=g).to(dev) for n in (H, KVH))
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32).to(dev)
    y = qk_norm_rotary(q, k, pos, torch.from_numpy(freqs(P)).to(dev), wq, wk)
    got = torch.autograd.grad(y, (q, k, wq, wk), (gq, gk))
    for i, (x, w, gy) in enumerate(((q, wq, gq), (k, wk, gk))):
        x64, w64, g64 = (t.detach().double().cpu().numpy() for t in (x, w, gy))
        close(y[i], *O.qk_norm_rotary(x64, w64, pos.cpu().numpy(), freqs(P)))
        dx, dw, edx, edw = O.qk_norm_rotary_backward(x64, w64, g64, pos.cpu().numpy(), freqs(P))
        close(got[i], dx, edx)
        close(got[2 + i], dw, edw)


@pytest.mark.parametrize("dtype", list(DT))
def test_strides_in_place_and_weight_types(dev, dtype):
    g = torch.Generator().manual_seed(3)
    B, T, H, KVH, D = 2, 5, 4, 2, 64
    rows = torch.randn(B, T, (H + 2 * KVH) * D + 8, generator=g).to(DT[dtype]).to(dev)
    q = rows[..., 8:8 + H * D].unflatten(-1, (H, D))
    k = rows[..., 8 + H * D:8 + (H + KVH) * D].unflatten(-1, (KVH, D))
    odd = torch.randn(B, H, T, D + 1, generator=g).to(DT[dtype]).to(dev)[..., 1:].transpose(1, 2)  # no 16-byte rows
    pos = torch.arange(T, device=dev)
    f = freqs(32)
    inv = torch.from_numpy(f).to(dev)
    for wdt in DT.values():
        w = (1 + 0.3 * torch.randn(2, D, generator=g)).to(wdt).to(dev)
        a, b = qk_norm_rotary(q, k, pos, inv, w[0], w[1])
        assert a.is_contiguous() and b.is_contiguous()
        w64 = w.double().cpu().numpy()
        close(a, *O.qk_norm_rotary(q.double().cpu().numpy(), w64[0], np.arange(T), f))
        close(b, *O.qk_norm_rotary(k.double().cpu().numpy(), w64[1], np.arange(T), f))
        close(qk_norm_rotary(odd, None, pos, inv, w[0])[0], *O.qk_norm_rotary(odd.double().cpu().numpy(), w64[0], np.arange(T), f))
        x = q.detach().clone().requires_grad_()
        ww = w[0].clone().requires_grad_()
        qk_norm_rotary(x.expand(B, T, H, D), None, pos, inv, ww)[0].sum().backward()  # (a gradient of stride 0)
        dx, dw, edx, edw = O.qk_norm_rotary_backward(x.detach().double().cpu().numpy(), w64[0], np.ones(q.shape), np.arange(T), f)
        close(x.grad, dx, edx)
        assert ww.grad.dtype is wdt
        close(ww.grad, dw, edw)
    before = rows.clone()
    a, b = qk_norm_rotary(q, k, pos, inv, w[0], w[1])
    qk_norm_rotary(q, k, pos, inv, w[0], w[1], out_q=q, out_k=k)
    assert torch.equal(q, a) and torch.equal(k, b)
    assert torch.equal(rows[..., :8], before[..., :8]) and torch.equal(rows[..., 8 + (H + KVH) * D:], before[..., 8 + (H + KVH) * D:])


def test_shared_leaves_and_far_positions(dev):
    """One tensor as q and k, one weight for both sides: the gradients add up."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, 3, 2, 64, generator=g).to(dev).requires_grad_()
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(dev).requires_grad_()
    pos = torch.tensor([[2 ** 31 - 1, 0, -7]], device=dev)
    f = freqs(32, 1e6)
    a, b = qk_norm_rotary(x, x, pos, torch.from_numpy(f).to(dev), w, w)
    assert torch.equal(a, b)
    ga, gb = torch.randn(2, 1, 3, 2, 64, generator=g).to(dev)
    torch.autograd.backward((a, b), (ga, gb))
    parts = [O.qk_norm_rotary_backward(x.detach().double().cpu().numpy(), w.detach().double().cpu().numpy(),
                                       t.double().cpu().numpy(), pos.cpu().numpy(), f) for t in (ga, gb)]
    for got, i in ((x.grad, 0), (w.grad, 1)):
        want = parts[0][i] + parts[1][i]
        close(got, want, parts[0][i + 2] + parts[1][i + 2] + 2.0 ** -24 * (abs(parts[0][i]) + abs(parts[1][i])))


def test_against_differences(dev):
    """The oracle's gradient against central differences of the oracle's values, and the
    kernel's values between two points against its gradient at their middle: the third
    derivative's part of it is h^2 times terms of the gradient's size."""
    g = torch.Generator().manual_seed(5)
    f = freqs(8)
    x = torch.randn(1, 4, 2, 24, generator=g).double().numpy()
    w = 1 + 0.2 * torch.randn(24, generator=g).double().numpy()
    gy = torch.randn(1, 4, 2, 24, generator=g).double().numpy()
    value = lambda x, w: (gy * O.qk_norm_rotary(x, w, np.arange(4), f)[0]).sum()
    dx, dw, _, _ = O.qk_norm_rotary_backward(x, w, gy, np.arange(4), f)
    h = 1e-5
    for _ in range(6):
        e, ew = torch.randn(x.shape, generator=g).numpy().astype(np.float64), torch.randn(24, generator=g).numpy().astype(np.float64)
        want = (value(x + h * e, w + h * ew) - value(x - h * e, w - h * ew)) / (2 * h)
        # rounding: 1e-16 of the value's terms over h; curvature: h^2 of them times a few
        assert abs(want - (dx * e).sum() - (dw * ew).sum()) < 1e-7 * (abs(gy).sum() + 1)
    q = torch.from_numpy(x).float().to(dev).requires_grad_()
    wt = torch.from_numpy(w).float().to(dev).requires_grad_()
    y = qk_norm_rotary(q, None, torch.arange(4, device=dev), torch.from_numpy(f).to(dev), wt)[0]
    got = torch.autograd.grad(y, (q, wt), torch.from_numpy(gy).float().to(dev))
    dx, dw, edx, edw = O.qk_norm_rotary_backward(q.detach().double().cpu().numpy(), wt.detach().double().cpu().numpy(),
                                                 torch.from_numpy(gy).float().double().numpy(), np.arange(4), f)
    close(got[0], dx, edx)
    close(got[1], dw, edw)


def test_rows_that_hold_no_numbers(dev):
    """A head of zeros gives zeros, one with an infinity or NaN NaN throughout, and its neighbours
    keep theirs."""
    x = torch.randn(1, 1, 4, 64, device=dev)
    x[0, 0, 1] = 0
    x[0, 0, 2, 5] = float("nan")
    pos, inv, w = torch.zeros(1, dtype=torch.int32, device=dev), torch.from_numpy(freqs(32)).to(dev), torch.ones(64, device=dev)
    y = qk_norm_rotary(x, None, pos, inv, w)[0]
    alone = qk_norm_rotary(x[:, :, :1].contiguous(), None, pos, inv, w)[0]
    assert torch.equal(y[:, :, :1], alone) and (y[0, 0, 1] == 0).all() and y[0, 0, 2].isnan().all() and y[0, 0, 3].isfinite().all()


def test_streams_and_graphs(dev):
    """On a side stream, and captured with its backward: replays equal the eager call's bits."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, 70, 4, 128, generator=g).to(dev, torch.bfloat16)
    w = (1 + 0.2 * torch.randn(128, generator=g)).to(dev)
    gy = torch.randn(1, 70, 4, 128, generator=g).to(dev, torch.bfloat16)
    pos, inv = torch.arange(70, device=dev), torch.from_numpy(freqs(64)).to(dev)

    def step(x, w, gy):
        q, ww = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = qk_norm_rotary(q, None, pos, inv, ww)[0]
        return (y.detach(), *torch.autograd.grad(y, (q, ww), gy))

    want = step(x, w, gy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step(x, w, gy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    graph = torch.cuda.CUDAGraph()
    sx = x.clone()
    with torch.cuda.graph(graph):
        held = step(sx, w, gy)
    for i in range(3):
        sx.copy_(x if i != 1 else 2 * x)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(sx, w, gy)
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), i


def test_no_rows(dev):
    q = torch.empty(2, 0, 3, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = qk_norm_rotary(q, None, torch.empty(0, dtype=torch.int32, device=dev), torch.from_numpy(freqs(32)).to(dev), w)[0]
    y.sum().backward()
    assert y.shape == q.shape and q.grad.shape == q.shape and (w.grad == 0).all()


def test_a_graph_of_the_gradients_is_refused(dev):
    """With create_graph the gradients are the same, and cannot be differentiated."""
    q = torch.randn(1, 3, 2, 64, generator=torch.Generator().manual_seed(0)).to(dev).requires_grad_()
    w = torch.ones(64, device=dev, requires_grad=True)
    pos, f = torch.arange(3, device=dev), torch.from_numpy(freqs(32)).to(dev)
    y = qk_norm_rotary(q, None, pos, f, w)[0].square().sum()
    want = torch.autograd.grad(y, (q, w), retain_graph=True)
    got = torch.autograd.grad(y, (q, w), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got[0].sum().backward()


def test_a_side_without_heads(dev):
    """k of no heads: its weights' gradient is zeros."""
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 3, 4, 64, generator=g).to(dev).requires_grad_()
    k = torch.empty(2, 3, 0, 64, device=dev, requires_grad=True)
    w = [torch.ones(64, device=dev, requires_grad=True) for _ in range(2)]
    pos, f = torch.arange(3, device=dev), torch.from_numpy(freqs(32)).to(dev)
    for _ in range(3):  # (memory that held something else)
        torch.full((1 << 16,), float("nan"), device=dev)
        y, z = qk_norm_rotary(q, k, pos, f, *w)
        assert z.shape == k.shape
        grads = torch.autograd.grad(y.sum(), (q, k, *w), allow_unused=True)
        alone = torch.autograd.grad(qk_norm_rotary(q, None, pos, f, w[0])[0].sum(), (q, w[0]))
        assert torch.equal(grads[0], alone[0]) and torch.equal(grads[2], alone[1])
        assert grads[1].shape == k.shape and (grads[3] == 0).all()


def test_refusals(dev):
    q, w = torch.randn(1, 2, 3, 64, device=dev), torch.ones(64, device=dev)
    pos, inv = torch.arange(2, device=dev), torch.from_numpy(freqs(32)).to(dev)
    for bad, text in ((dict(q_weight=w[:32]), "q_weight"), (dict(k=q), "k_weight"), (dict(k_weight=w), "without k"),
                      (dict(k=q, k_weight=w.half()), "dtype"), (dict(k=q.half(), k_weight=w), "match q"),
                      (dict(positions=torch.arange(3, device=dev)), "positions"), (dict(inv_freq=inv.float()), "inv_freq"),
                      (dict(out_q=torch.empty(1, 2, 3, 64, device=dev, dtype=torch.half)), "out_q"),
                      (dict(out_q=torch.empty(1, 1, 3, 64, device=dev).expand(1, 2, 3, 64)), "share memory")):
        a = dict(q=q, k=None, positions=pos, inv_freq=inv, q_weight=w, k_weight=None)
        with pytest.raises(SFError, match=text):
            qk_norm_rotary(**{**a, **bad})
    with pytest.raises(SFError, match="at most 256"):
        qk_norm_rotary(torch.randn(1, 2, 1, 512, device=dev), None, pos, inv, torch.ones(512, device=dev))
    with pytest.raises(SFError, match="gradient take no out"):
        qk_norm_rotary(q.requires_grad_(), None, pos, inv, w, out_q=torch.empty_like(q))
