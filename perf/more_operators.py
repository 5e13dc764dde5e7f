"""The work of a decoder layer whose heads are normed before they turn and whose KV cache
is held in 4 bits.

A case is a dict of plain values whose "kind" names the call:

  norm    `kernels.rotary.qk_norm_rotary`: every q and k head normed by its root mean
          square, weighted and rotated in one pass
  train   the same with its gradients in q, k and both weights
  append  `kernels.kv_q4.rotary_kv_append_q4`: fused q|k|v rows, (normed and) turned, k and
          v into a cache in groups of 4-bit codes; then `dequantize_kv_q4` of the new slots
  attend  `kernels.kv_q4.attention_q4kv`: attention over such a cache, from one token a
          sequence to a prompt's rows
  step    `rotary_kv_append_q4`, then `attention_q4kv`: one token a sequence through a layer

Where `own` is false, `run` computes them with elementary torch operations.
`exact` restates each in 64 bits. A group of g dims is held as codes 0..15 beside two fp16
numbers: x is m + s c with m the group's minimum and s a fifteenth of its range.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6


def listed() -> list[dict]:
    return [
        # one decoded token of the 0.5B geometry: the smallest call, where latency counts
        dict(name="norm_token", kind="norm", batch=1, rows=1, heads=14, kv_heads=2, dim=64, rot=64,
             interleaved=False, theta=1e6, far=500, dtype="bf16"),
        # a long prompt (ragged) of the 8B geometry
        dict(name="norm_prompt", kind="norm", batch=1, rows=8191, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, theta=5e5, far=8191, dtype="bf16"),
        # a training batch's layer, interleaved pairs over half the head
        dict(name="norm_train", kind="train", batch=4, rows=1021, heads=32, kv_heads=8, dim=128, rot=64,
             interleaved=True, theta=1e4, far=1021, dtype="bf16"),
        # the 0.5B geometry's layer in fp32, as it is checked against differences
        dict(name="norm_train_small", kind="train", batch=1, rows=300, heads=14, kv_heads=2, dim=64, rot=64,
             interleaved=False, theta=1e6, far=300, dtype="f32"),
        # eight sequences' next tokens, rows as a quantized projection leaves them
        dict(name="append_batch", kind="append", batch=8, rows=1, heads=32, kv_heads=8, dim=128, group=64,
             norm=True, interleaved=False, theta=5e5, start=2001, dtype="f32", out="f32"),
        # a prompt's rows into an empty cache
        dict(name="append_prompt", kind="append", batch=1, rows=4095, heads=32, kv_heads=8, dim=128, group=64,
             norm=True, interleaved=False, theta=5e5, start=0, dtype="bf16", out="bf16"),
        # one decoded token of the 0.5B geometry
        dict(name="attend_small", kind="attend", batch=1, rows=1, heads=14, kv_heads=2, dim=64, group=64,
             cached=1501, dtype="f16", out="f32"),
        # the rows of a short continuation, fp32 queries, the finest groups
        dict(name="attend_window", kind="attend", batch=1, rows=16, heads=14, kv_heads=2, dim=64, group=32,
             cached=2000, dtype="f32", out="f32"),
        # batched decode of the 8B geometry over long ragged caches
        dict(name="attend_long", kind="attend", batch=4, rows=1, heads=32, kv_heads=8, dim=128, group=64,
             cached=32767, dtype="bf16", out="bf16"),
        # one sequence with a context of 128 Ki tokens less one
        dict(name="attend_far", kind="attend", batch=1, rows=1, heads=32, kv_heads=8, dim=128, group=128,
             cached=131071, dtype="f16", out="f16"),
        # a prompt behind a cached prefix
        dict(name="attend_prompt", kind="attend", batch=1, rows=1500, heads=32, kv_heads=8, dim=128, group=64,
             cached=1800, dtype="bf16", out="bf16"),
        # sixteen sequences' tokens through one layer
        dict(name="step_batch", kind="step", batch=16, rows=1, heads=32, kv_heads=8, dim=128, group=64,
             norm=True, interleaved=False, theta=5e5, cached=4001, dtype="f32", out="f32"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_GEOMETRIES = [(14, 2, 64), (14, 2, 64), (32, 8, 128), (32, 8, 128), (32, 32, 128), (14, 14, 64), (9, 3, 80),
               (12, 1, 96), (16, 4, 256), (40, 2, 128)]


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "train", "train", "append", "append", "attend", "attend", "attend", "attend",
                       "step"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads, kv_heads, dim = rng.choice(_GEOMETRIES)
    if kind in ("norm", "train"):
        batch = rng.choice([1, 1, 2, 16])
        most = (8191 if kind == "norm" else 4084) * 40 * 128 * 2
        rows = _log_int(rng, 1, 8191)
        rows = max(1, min(rows, most // (batch * (heads + kv_heads) * dim * _SIZE[dtype])))
        return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 2 * (dim // 5)]), interleaved=rng.random() < 0.5,
                    theta=rng.choice([1e4, 5e5, 1e6]), far=_log_int(rng, max(rows, 100), 1000000), dtype=dtype)
    group = rng.choice([dim] + [g for g in (32, 64) if dim % g == 0 and g < dim])
    out = rng.choice(["f32", dtype])
    if kind == "append":
        batch = rng.choice([1, 1, 2, 8])
        most = 4095 * 48 * 128 * 2
        rows = _log_int(rng, 1, 4095)
        rows = max(1, min(rows, most // (batch * (heads + 2 * kv_heads) * dim * _SIZE[dtype])))
        return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, group=group,
                    norm=rng.random() < 0.6, interleaved=rng.random() < 0.3, theta=rng.choice([1e4, 5e5, 1e6]),
                    start=rng.choice([0, _log_int(rng, 1, 4000)]), dtype=dtype, out=out)
    batch = rng.choice([1, 1, 2, 4, 8])
    cached = _log_int(rng, 20, 65536)
    cached = max(20, min(cached, 131071 * 8 * 128 // (batch * kv_heads * dim)))
    if kind == "step":
        return dict(kind=kind, batch=batch, rows=1, heads=heads, kv_heads=kv_heads, dim=dim, group=group,
                    norm=rng.random() < 0.6, interleaved=rng.random() < 0.3, theta=rng.choice([1e4, 5e5, 1e6]),
                    cached=cached, dtype="f32", out="f32")
    rows = rng.choice([1, 1, 1, 3, 16, _log_int(rng, 17, 1500)])
    rows = max(1, min(rows, cached, 1500 * 32 * 1800 * 128 // (2 * batch * heads * cached * dim)))
    return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, group=group,
                cached=cached, dtype=dtype, out=out)


def _cache(case: dict, cap: int, normal) -> dict:
    """A cache as it was appended: codes two a byte (the even dim in the low half), and
    (s, m) a group."""
    state, g = {}, case["group"]
    shape = (case["batch"], case["kv_heads"], cap, case["dim"])
    for name in ("k", "v"):
        x = normal(*shape).unflatten(-1, (-1, g))
        m = x.amin(dim=-1, keepdim=True).half()
        s = ((x.amax(dim=-1, keepdim=True) - m) / 15).half()
        c = torch.round((x - m.float()) / s.float()).clamp_(0, 15).flatten(-2).to(torch.uint8)
        state[name + "_codes"] = c[..., 0::2] | c[..., 1::2] << 4
        state[name + "_params"] = torch.cat([s, m], dim=-1)
    return state


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device=dev)
    state = {"case": case}
    kind, B, H, KVH, D = case["kind"], case["batch"], case["heads"], case["kv_heads"], case["dim"]
    dtype, T = _DTYPES[case["dtype"]], case["rows"]
    if kind != "attend":
        rot = case.get("rot", D)
        state["inv_freq"] = torch.from_numpy(case["theta"] ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)).to(dev)
    if kind in ("norm", "train") or (kind != "attend" and case["norm"]):
        state["q_weight"] = 1.0 + 0.2 * normal(D)
        state["k_weight"] = 1.0 + 0.2 * normal(D)
    if kind in ("norm", "train"):
        state["q"] = (2.0 * normal(B, T, H, D)).to(dtype)
        state["k"] = (2.0 * normal(B, T, KVH, D)).to(dtype)
        start = (uniform(B, 1) * max(case["far"] - T, 1)).to(torch.int32)
        state["positions"] = (start + torch.arange(T, device=dev, dtype=torch.int32)).contiguous()
        if kind == "train":
            state["leaves"] = tuple(state[k].requires_grad_() for k in ("q", "k", "q_weight", "k_weight"))
            state["grads"] = normal(B, T, H, D).to(dtype), normal(B, T, KVH, D).to(dtype)
        return state
    if kind == "append":
        n, g = case["start"], case["group"]
        cap = n + T + 61
        state["positions"] = torch.arange(n, n + T, device=dev, dtype=torch.int32)
        for name in ("k", "v"):
            state[name + "_codes"] = torch.zeros(B, KVH, cap, D // 2, dtype=torch.uint8, device=dev)
            state[name + "_params"] = torch.zeros(B, KVH, cap, D // g, 2, dtype=torch.float16, device=dev)
    else:
        n = case["cached"]
        cap = n + 37 if n % 2 else n + 64
        lengths = torch.full((B,), n, dtype=torch.int32, device=dev)
        if B > 1:  # ragged sequences, one of them full
            lengths[1:] = (n * (0.3 + 0.7 * uniform(B - 1))).to(torch.int32).clamp_(min=min(n, max(T, 1)))
        state["lengths"] = lengths
        state.update(_cache(case, cap, normal))
    if kind == "attend":
        state["q"] = (1.5 * normal(B, T, H, D)).to(dtype)
        return state
    state["qkv"] = (1.5 * normal(B, T, (H + 2 * KVH) * D)).to(dtype)
    if kind == "step":
        state["positions"] = lengths[:, None].contiguous()
    return state


# ---- the plain forms ---------------------------------------------------------
def _turned(a, b, c, s):
    return a * c - b * s, b * c + a * s


def _rotate(x, positions, inv_freq, interleaved, sign=1.0):
    """x [B, T, heads, D] turned by its rows' positions, in x's own width."""
    angle = positions.double()[..., None] * inv_freq
    c, s = ((t.to(x.dtype))[..., None, :] for t in (torch.cos(angle), sign * torch.sin(angle)))
    r = 2 * inv_freq.numel()
    if interleaved:
        y = torch.stack(_turned(x[..., 0:r:2], x[..., 1:r:2], c, s), dim=-1).flatten(-2)
    else:
        y = torch.cat(_turned(x[..., :r // 2], x[..., r // 2:r], c, s), dim=-1)
    return torch.cat([y, x[..., r:]], dim=-1)


def _inv_rms(x):
    return torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS)


def _plain_norm(s, x, w):
    x = x.detach().float()
    y = x * _inv_rms(x) * w.detach()
    return _rotate(y, s["positions"], s["inv_freq"], s["case"]["interleaved"])


def _plain_train(s, x, w, gy):
    """(output, gradient of x, gradient of w) for the gradient gy of the output."""
    y = _plain_norm(s, x, w).to(x.dtype)
    g = _rotate(gy.float(), s["positions"], s["inv_freq"], s["case"]["interleaved"], -1.0)
    x, w = x.detach().float(), w.detach()
    r = _inv_rms(x)
    n = x * r
    gn = g * w
    dx = r * (gn - n * (gn * n).mean(dim=-1, keepdim=True))
    return y, dx.to(gy.dtype), (g * n).sum(dim=(0, 1, 2))


def _plain_append(s, slots):
    """The turned q; k and v go into the slots [B, T]. Codes are chosen in 64 bits: next to
    a border they depend on every last place."""
    c = s["case"]
    B, T, H, KVH, D, g = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["dim"], c["group"]
    x = s["qkv"].reshape(B, T, H + 2 * KVH, D)
    q, k, v = x[:, :, :H].float(), x[:, :, H:H + KVH].double(), x[:, :, H + KVH:].double()
    if c["norm"]:
        q, k = (y * _inv_rms(y) * w for y, w in ((q, s["q_weight"]), (k, s["k_weight"])))
    q, k = (_rotate(y, s["positions"], s["inv_freq"], c["interleaved"]) for y in (q, k))
    at = (torch.arange(B, device=x.device)[:, None], slice(None), slots)
    for name, y in (("k", k), ("v", v)):
        y = y.unflatten(-1, (-1, g))
        lo, hi = y.amin(dim=-1, keepdim=True), y.amax(dim=-1, keepdim=True)
        m, sc = lo.float().half(), ((hi - lo) / 15).float().half()
        step = torch.where(sc == 0, torch.ones_like(sc), sc).double()
        code = torch.where(sc == 0, torch.zeros_like(y), torch.round((y - m.double()) / step).clamp(0, 15))
        code = code.flatten(-2).to(torch.uint8)
        s[name + "_codes"][at] = code[..., 0::2] | code[..., 1::2] << 4
        s[name + "_params"][at] = torch.cat([sc, m], dim=-1)
    return q.to(_DTYPES[c["out"]])


def _values(codes, params):
    """What codes [..., D / 2] and params [..., D / g, 2] stand for, fp32."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float().unflatten(-1, (params.shape[-2], -1))
    return (c * params[..., 0:1].float() + params[..., 1:2].float()).flatten(-2)


def _plain_attend(s, q, lengths):
    """q [B, T, H, D] over the first lengths[b] slots, row t up to slot lengths[b] - T + t."""
    c = s["case"]
    B, T, H, D = q.shape
    KVH, G = c["kv_heads"], c["heads"] // c["kv_heads"]
    n = min(c["cached"] + (T if c["kind"] == "step" else 0), s["k_codes"].shape[2])
    K, V = (_values(s[k + "_codes"][:, :, :n], s[k + "_params"][:, :, :n]) for k in ("k", "v"))
    rows = q.float().reshape(B, T, KVH, G, D).permute(0, 2, 1, 3, 4).reshape(B, KVH, T * G, D)
    x = torch.matmul(rows, K.transpose(-1, -2)) * D ** -0.5
    last = (lengths[:, None] - T + torch.arange(T, device=q.device)).repeat_interleave(G, dim=1)[:, None, :, None]
    x = x.masked_fill(torch.arange(n, device=q.device) > last, float("-inf"))
    top = x.amax(dim=-1, keepdim=True)
    w = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(dim=-1, keepdim=True)
    out = torch.matmul(w, V) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(B, KVH, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D).to(_DTYPES[c["out"]])


# ---- one pass ----------------------------------------------------------------
_calls = None


def _framework():
    global _calls
    if _calls is None:
        from siliconfer_amd.kernels.kv_q4 import attention_q4kv, dequantize_kv_q4, rotary_kv_append_q4
        from siliconfer_amd.kernels.rotary import qk_norm_rotary
        _calls = dict(norm=qk_norm_rotary, append=rotary_kv_append_q4, attend=attention_q4kv, values=dequantize_kv_q4)
    return _calls


def _own_append(s, lengths):
    c = s["case"]
    return _framework()["append"](s["qkv"], s["positions"], s["inv_freq"], s["k_codes"], s["k_params"], s["v_codes"],
                                  s["v_params"], n_heads=c["heads"], lengths=lengths, q_weight=s.get("q_weight"),
                                  k_weight=s.get("k_weight"), eps=_EPS, interleaved=c["interleaved"],
                                  out_dtype=_DTYPES[c["out"]])


def run(state: dict):
    s, c = state, state["case"]
    kind, T = c["kind"], c["rows"]
    if kind == "norm":
        if own:
            return _framework()["norm"](s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"],
                                        eps=_EPS, interleaved=c["interleaved"])
        return _plain_norm(s, s["q"], s["q_weight"]).to(s["q"].dtype), _plain_norm(s, s["k"], s["k_weight"]).to(s["k"].dtype)
    if kind == "train":
        if own:
            y = _framework()["norm"](s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"],
                                     eps=_EPS, interleaved=c["interleaved"])
            d = torch.autograd.grad(y, s["leaves"], s["grads"])
        else:
            (yq, dq, dwq), (yk, dk, dwk) = (_plain_train(s, s[n], s[n + "_weight"], g)
                                            for n, g in zip(("q", "k"), s["grads"]))
            y, d = (yq, yk), (dq, dk, dwq, dwk)
        return {"q": y[0].detach(), "k": y[1].detach(), "dq": d[0], "dk": d[1], "dq_weight": d[2], "dk_weight": d[3]}
    if kind == "append":
        n = c["start"]
        if own:
            q = _own_append(s, n)
        else:
            q = _plain_append(s, torch.arange(n, n + T, device=s["qkv"].device).expand(c["batch"], T))
        new = lambda name: (s[name + "_codes"][:, :, n:n + T], s[name + "_params"][:, :, n:n + T])
        values = _framework()["values"] if own else _values
        return {"q": q, "k": values(*new("k")), "v": values(*new("v"))}
    if kind == "attend":
        if own:
            return _framework()["attend"](s["q"], s["k_codes"], s["k_params"], s["v_codes"], s["v_params"],
                                          lengths=s["lengths"], out_dtype=_DTYPES[c["out"]])
        return _plain_attend(s, s["q"], s["lengths"])
    # the cache's codes come back within `out`: its newest slot is among those attended to
    if own:
        q = _own_append(s, s["lengths"])
        out = _framework()["attend"](q, s["k_codes"], s["k_params"], s["v_codes"], s["v_params"],
                                     lengths=s["lengths"], add=T, out_dtype=_DTYPES[c["out"]])
    else:
        q = _plain_append(s, (s["lengths"][:, None] + torch.arange(T, device=s["qkv"].device)).long())
        out = _plain_attend(s, q, s["lengths"] + T)
    return {"out": out, "k_params": s["k_params"], "v_params": s["v_params"]}


def work(case: dict) -> dict:
    kind, B, T, H, KVH, D = case["kind"], case["batch"], case["rows"], case["heads"], case["kv_heads"], case["dim"]
    size = _SIZE[case["dtype"]]
    if kind in ("norm", "train"):
        n = B * T * (H + KVH) * D
        # x in, y out; its gradient in and x's gradient out beside them
        return {"bytes": n * size * (2 if kind == "norm" else 4) + 4 * B * T, "flops": n * (8 if kind == "norm" else 24)}
    slot = 2 * KVH * (D // 2 + 4 * (D // case["group"]))  # codes and parameters of k and v
    new = B * T * ((H + 2 * KVH) * D * size + H * D * _SIZE[case["out"]] + slot)
    if kind == "append":
        return {"bytes": new + B * T * (slot + 2 * KVH * D * 4), "flops": B * T * (H + 2 * KVH) * D * 8}
    n = case["cached"]
    n_all = n + (B - 1) * 0.65 * n if B > 1 else n  # the sequences' expected lengths together
    pairs = T * n_all - B * T * (T - 1) / 2  # (row, slot) pairs that are seen
    bytes_ = n_all * slot + B * T * H * D * (size + _SIZE[case["out"]])
    return {"bytes": bytes_ + (new if kind == "step" else 0), "flops": 4.0 * pairs * H * D}


# ---- 64 bits -----------------------------------------------------------------
def _turn64(x, angle, interleaved):
    """Pairs as complex numbers times e^(i angle); x [B, T, heads, D] in 64 bits."""
    r = 2 * angle.shape[-1]
    pairs = x[..., :r].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    axis = -1 if interleaved else -2
    z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1)) * torch.polar(torch.ones_like(angle), angle)[..., None, :]
    return torch.cat([torch.stack([z.real, z.imag], dim=axis).flatten(-2), x[..., r:]], dim=-1)


def _norm64(x, w):
    return w * x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + _EPS)


def _cached64(y, group):
    """The values and the (s, m) that y [..., D] is cached as; 15 code borders counted."""
    y = y.unflatten(-1, (-1, group))
    lo, hi = y.min(dim=-1, keepdim=True).values, y.max(dim=-1, keepdim=True).values
    half = lambda t: t.float().half().double()
    m, s = half(lo), half((hi - lo) / 15)
    # code k + 1 is taken past s (k + 1/2), at it only from an odd k (ties go to the even code)
    code = torch.zeros_like(y)
    for k in range(15):
        code += (y - m > s * (k + 0.5)) | ((y - m == s * (k + 0.5)) & (k % 2 == 1) & (s > 0))
    code = torch.where(s > 0, code, torch.zeros_like(code))
    return (m + s * code).flatten(-2), torch.cat([s, m], dim=-1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, B, T, H, KVH, D = case["kind"], case["batch"], case["rows"], case["heads"], case["kv_heads"], case["dim"]
    G = H // KVH
    if kind != "attend":
        angle = s["positions"].double()[..., None] * s["inv_freq"]
    if kind in ("norm", "train"):
        x = [s[k].detach().double().requires_grad_() for k in ("q", "k", "q_weight", "k_weight")]
        y = [_turn64(_norm64(x[i], x[i + 2]), angle, case["interleaved"]) for i in range(2)]
        if kind == "norm":
            return y[0].detach(), y[1].detach()
        d = torch.autograd.grad(y, x, [g.double() for g in s["grads"]])
        return {"q": y[0], "k": y[1], "dq": d[0], "dk": d[1], "dq_weight": d[2], "dk_weight": d[3]}
    if kind != "attend":
        x = s["qkv"].double().reshape(B, T, H + 2 * KVH, D)
        q, k, v = x.split([H, KVH, KVH], dim=2)
        if case["norm"]:
            q, k = _norm64(q, s["q_weight"].double()), _norm64(k, s["k_weight"].double())
        q, k = (_turn64(t, angle, case["interleaved"]) for t in (q, k))
        new = {n: _cached64(t.transpose(1, 2), case["group"]) for n, t in (("k", k), ("v", v))}
        if kind == "append":
            return {"q": q, "k": new["k"][0], "v": new["v"][0]}
    else:
        q = s["q"].double()
    lengths = s["lengths"].tolist()
    params = {n: s[n + "_params"].double() for n in ("k", "v")}
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=q.device)
    for b in range(B):
        kv = []
        for n in ("k", "v"):
            m = lengths[b]
            codes = s[n + "_codes"][b, :, :m]
            c = torch.zeros(KVH, m, D, dtype=torch.float64, device=q.device)
            c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
            p = params[n][b, :, :m].repeat_interleave(case["group"], dim=-2)
            y = p[..., 1] + p[..., 0] * c
            if kind == "step":
                y = torch.cat([y, new[n][0][b]], dim=1)
                params[n][b, :, m:m + T] = new[n][1][b]
            kv.append(y)
        m = kv[0].shape[1]
        seen = torch.arange(m, device=q.device) <= torch.arange(m - T, m, device=q.device)[:, None]
        for h in range(KVH):
            z = torch.einsum("tgd,md->tgm", q[b, :, h * G:(h + 1) * G], kv[0][h]) / math.sqrt(D)
            w = torch.softmax(z.masked_fill(~seen[:, None], float("-inf")), dim=-1)
            out[b, :, h * G:(h + 1) * G] = torch.einsum("tgm,md->tgd", w, kv[1][h])
    if kind == "attend":
        return out
    return {"out": out, "k_params": params["k"], "v_params": params["v"]}
