"""The work of a bounded KV cache's decode step and of drawing the token behind it.

A case is a dict of plain values whose "kind" names the call:

  rotary   `kernels.rotary.rotary`: q and k rows rotated at given positions (both
           pair layouts, part of the head, scaled frequencies)
  attend   `kernels.attention.attention_decode_scored`: attention over an int8 cache
           whose softmax weights are added to a score a slot
  evict    `kernels.eviction.evict`: the slots with the least score leave the cache
  step     `kernels.rotary.rotary_kv_append`, then `attention_decode_scored`: one
           token a sequence through a layer's cache
  sample   `kernels.sampling.sample`: a token a row from given random numbers under
           temperature, top-k, top-p and min-p

Where `own` is false, `run` computes them with elementary torch operations.
`exact` restates each in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed() -> list[dict]:
    return [
        # one decoded token of the 0.5B geometry: the smallest call, where latency counts
        dict(name="rotary_token", kind="rotary", batch=1, rows=1, heads=14, kv_heads=2, dim=64, rot=64,
             interleaved=False, scaling="none", theta=1e6, far=500, dtype="bf16"),
        # sixteen sequences' tokens far into long contexts: interleaved pairs over half the
        # head, frequencies stretched for sixteen times the trained length
        dict(name="rotary_far_batch", kind="rotary", batch=16, rows=1, heads=32, kv_heads=8, dim=128,
             rot=64, interleaved=True, scaling="yarn", theta=1e4, far=500000, dtype="f16"),
        # a long prompt (ragged) of the 8B geometry
        dict(name="rotary_prompt", kind="rotary", batch=1, rows=8191, heads=32, kv_heads=8, dim=128,
             rot=128, interleaved=False, scaling="linear", theta=5e5, far=8191, dtype="bf16"),
        # one decoded token of the 0.5B geometry over a cache bounded at some 1500 slots
        dict(name="attend_small", kind="attend", batch=1, rows=1, heads=14, kv_heads=2, dim=64,
             cached=1501, dtype="f16", out="f32"),
        # batched decode of the 8B geometry over long ragged caches
        dict(name="attend_long", kind="attend", batch=4, rows=1, heads=32, kv_heads=8, dim=128,
             cached=8191, dtype="bf16", out="bf16"),
        # the last sixteen rows of a prompt scoring the cache behind them, fp32 queries
        dict(name="attend_window", kind="attend", batch=1, rows=16, heads=14, kv_heads=2, dim=64,
             cached=2000, dtype="f32", out="f32"),
        # a decoder's cache 64 tokens past its bound, the newest quarter kept
        dict(name="evict_step", kind="evict", batch=1, kv_heads=2, dim=64, cached=1088, budget=1024,
             recent=256),
        # four prompts cut to a quarter
        dict(name="evict_prompt", kind="evict", batch=4, kv_heads=8, dim=128, cached=8191,
             budget=2048, recent=64),
        # eight sequences' tokens through one layer's cache of the 8B geometry
        dict(name="step_batch", kind="step", batch=8, rows=1, heads=32, kv_heads=8, dim=128,
             cached=2001, dtype="f32", out="f32"),
        # one sequence's next token under the usual filters
        dict(name="sample_one", kind="sample", batch=1, vocab=151936, dtype="f32", temperature=0.8,
             top_k=50, top_p=0.95, min_p=0.0, mixed=False),
        # eight sequences of a small vocabulary at temperature alone
        dict(name="sample_plain", kind="sample", batch=8, vocab=32000, dtype="f32", temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0, mixed=False),
        # a serving batch, each row with settings of its own, some greedy
        dict(name="sample_batch", kind="sample", batch=64, vocab=151936, dtype="bf16", temperature=0.9,
             top_k=200, top_p=0.9, min_p=0.02, mixed=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_GEOMETRIES = [(14, 2, 64), (32, 8, 128), (32, 32, 128), (14, 14, 64), (9, 3, 80), (12, 1, 96),
               (16, 4, 256), (40, 2, 128)]


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "rotary", "attend", "attend", "attend", "evict", "evict", "step",
                       "sample", "sample", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads, kv_heads, dim = rng.choice(_GEOMETRIES)
    if kind == "rotary":
        batch = rng.choice([1, 1, 2, 16])
        rows = _log_int(rng, 1, 8191)
        rows = max(1, min(rows, 8191 * 40 * 128 * 2 // (batch * (heads + kv_heads) * dim * _SIZE[dtype])))
        return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 2 * (dim // 5)]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn"]), theta=rng.choice([1e4, 5e5, 1e6]),
                    far=_log_int(rng, max(rows, 100), 1000000), dtype=dtype)
    if kind == "evict":
        batch = rng.choice([1, 1, 2, 4])
        cached = _log_int(rng, 20, 32768)
        cached = min(cached, 4 * 8 * 8191 * 128 // (batch * kv_heads * dim))
        budget = max(1, int(cached * rng.choice([0.1, 0.25, 0.5, 0.9, 0.98])))
        return dict(kind=kind, batch=batch, kv_heads=kv_heads, dim=dim, cached=cached, budget=budget,
                    recent=int(budget * rng.choice([0.0, 0.1, 0.5])))
    if kind == "sample":
        vocab = rng.choice([32000, 50257, 151936, _log_int(rng, 100, 200000)])
        batch = min(_log_int(rng, 1, 64), max(1, 64 * 151936 // (vocab * (2 if dtype == "f32" else 1))))
        return dict(kind=kind, batch=batch, vocab=vocab, dtype=dtype,
                    temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice([0, 0, 1, 40, 1000]),
                    top_p=rng.choice([1.0, 0.95, 0.8]), min_p=rng.choice([0.0, 0.0, 0.05]),
                    mixed=rng.random() < 0.4)
    batch = rng.choice([1, 1, 2, 4, 8])
    rows = 1 if kind == "step" else rng.choice([1, 1, 1, 3, 16])
    cached = _log_int(rng, 20, 16384)
    cached = max(17, min(cached, 4 * 8 * 8191 * 128 // (batch * kv_heads * dim * (1 if rows < 3 else 4))))
    return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim,
                cached=cached, dtype="f32" if kind == "step" else dtype,
                out=rng.choice(["f32", "f32", "same"]) if dtype != "f32" and kind != "step" else "f32")


def _out_dtype(case: dict) -> torch.dtype:
    return _DTYPES[case["dtype"] if case["out"] == "same" else case["out"]]


def _frequencies(case: dict) -> tuple[np.ndarray, float]:
    """The angle a position of each pair, 64 bits, and the factor on cos and sin."""
    rot, theta = case["rot"], case["theta"]
    f = theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "yarn":  # slow pairs stretched by 16, fast ones as they are
        factor, trained = 16.0, 32768.0
        at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _cache(case: dict, cap: int, normal) -> dict:
    """Keys and values in int8 with an fp16 scale a token and head, as appended."""
    state = {}
    for name in ("k", "v"):
        x = normal(case["batch"], case["kv_heads"], cap, case["dim"])
        s = x.abs().amax(dim=-1, keepdim=True) / 127.0
        state[name + "_codes"] = torch.round(x / s).to(torch.int8)
        state[name + "_scales"] = s[..., 0].to(torch.float16)
    return state


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device=dev)
    state = {"case": case}
    kind = case["kind"]
    if kind == "sample":
        B, V = case["batch"], case["vocab"]
        # a head of likely tokens that falls off with the logarithm of the rank
        rank = torch.argsort(uniform(B, V), dim=-1).float()
        state["logits"] = (12.0 - 1.3 * torch.log1p(rank) + 0.7 * normal(B, V)).to(_DTYPES[case["dtype"]])
        state["u"] = uniform(B)
        if case["mixed"]:
            r = uniform(4, B)
            state["temperature"] = torch.where(r[3] < 0.1, torch.zeros_like(r[3]), case["temperature"] * (0.5 + r[0]))
            state["top_k"] = (case["top_k"] * 2 * r[1]).to(torch.int32)
            state["top_p"] = 1.0 - (1.0 - case["top_p"]) * 2 * r[2]
            state["min_p"] = case["min_p"] * 2 * r[3]
        else:
            for k in ("temperature", "top_k", "top_p", "min_p"):
                state[k] = case[k]
        return state
    B, KVH, D = case["batch"], case["kv_heads"], case["dim"]
    if kind == "rotary":
        T = case["rows"]
        state["q"] = normal(B, T, case["heads"], D).to(_DTYPES[case["dtype"]])
        state["k"] = normal(B, T, KVH, D).to(_DTYPES[case["dtype"]])
        start = (uniform(B, 1) * max(case["far"] - T, 1)).to(torch.int32)
        state["positions"] = (start + torch.arange(T, device=dev, dtype=torch.int32)).contiguous()
        f, state["scale"] = _frequencies(case)
        state["inv_freq"] = torch.from_numpy(f).to(dev)
        return state
    n = case["cached"]
    cap = n + 37 if n % 2 else n + 64
    lengths = torch.full((B,), n, dtype=torch.int32, device=dev)
    if B > 1:  # ragged sequences, one of them full
        lengths[1:] = (n * (0.3 + 0.7 * uniform(B - 1))).to(torch.int32).clamp_(min=1)
    state["lengths"] = lengths
    if kind == "evict":
        state.update(_cache(case, cap, normal))
        # accumulated weights are skewed; positions of a cache that was cut before
        scores = -torch.log(uniform(B, KVH, cap) + 1e-9) ** 2
        order = torch.argsort(uniform(B, KVH, cap), dim=-1)
        positions = torch.gather(torch.cumsum((1 + 3 * uniform(B, KVH, cap)).to(torch.int64), dim=-1), -1, order)
        inside = torch.arange(cap, device=dev) < lengths[:, None, None]
        state["seen"] = (positions.masked_fill(~inside, 0).amax(dim=(1, 2)) + 1).to(torch.int32)
        state["meta"] = torch.stack([scores.view(torch.int32), positions.to(torch.int32)])
        return state
    state.update(_cache(case, cap, normal))
    G = case["heads"] // KVH
    state["scores"] = uniform(B, KVH, cap) * (8.0 * G / n)  # after some sixteen tokens
    if kind == "attend":
        state["q"] = (1.5 * normal(B, case["rows"], case["heads"], D)).to(_DTYPES[case["dtype"]])
        return state
    state["qkv"] = normal(B, case["rows"], (KVH * G + 2 * KVH) * D)
    state["positions"] = (lengths[:, None] * 3 + torch.arange(case["rows"], device=dev, dtype=torch.int32)).contiguous()
    state["inv_freq"] = torch.from_numpy(1e6 ** (-np.arange(0, D, 2, dtype=np.float64) / D)).to(dev)
    state["slot_positions"] = torch.zeros(B, KVH, cap, dtype=torch.int32, device=dev)
    return state


# ---- the plain forms ---------------------------------------------------------
def _rotate(x, positions, inv_freq, scale, interleaved):
    angle = positions[..., None].double() * inv_freq
    c, s = ((scale * t).float()[:, :, None] for t in (torch.cos(angle), torch.sin(angle)))
    r = 2 * inv_freq.numel()
    xf = x.float()
    if interleaved:
        a, b = xf[..., 0:r:2], xf[..., 1:r:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = xf[..., :r // 2], xf[..., r // 2:r]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, xf[..., r:]], dim=-1)


def _plain_rotary(s):
    c = s["case"]
    turn = lambda x: _rotate(x, s["positions"], s["inv_freq"], s["scale"], c["interleaved"]).to(x.dtype)
    return turn(s["q"]), turn(s["k"])


def _plain_attend(s, q, lengths, out_dtype):
    """q [B, T, H, D] over the first lengths[b] slots, row t up to slot lengths[b] - T + t."""
    B, T, H, D = q.shape
    KVH = s["k_codes"].shape[1]
    n = min(s["case"]["cached"] + s["case"]["rows"], s["k_codes"].shape[2])
    K = s["k_codes"][:, :, :n].float() * s["k_scales"][:, :, :n, None].float()
    V = s["v_codes"][:, :, :n].float() * s["v_scales"][:, :, :n, None].float()
    rows = q.float().reshape(B, T, KVH, H // KVH, D).permute(0, 2, 1, 3, 4).reshape(B, KVH, -1, D)
    x = torch.matmul(rows, K.transpose(-1, -2)) * D ** -0.5
    last = lengths[:, None] - T + torch.arange(T, device=q.device)
    last = last[:, None, :, None].expand(B, 1, T, H // KVH).reshape(B, 1, -1, 1)
    seen = torch.arange(n, device=q.device) <= last
    x = x.masked_fill(~seen, float("-inf"))
    top = x.amax(dim=-1, keepdim=True)
    w = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(dim=-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(w, V).reshape(B, KVH, T, H // KVH, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    s["scores"][:, :, :n] += w.sum(dim=2)
    return out.to(out_dtype)


def _plain_step(s):
    c = s["case"]
    B, T, H, KVH, D = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].reshape(B, T, H + 2 * KVH, D)
    turned = _rotate(x[:, :, :H + KVH], s["positions"], s["inv_freq"], 1.0, False)
    slots = (s["lengths"][:, None] + torch.arange(T, device=x.device)).long()
    at = (torch.arange(B, device=x.device)[:, None], slice(None), slots)
    for name, new in (("k", turned[:, :, H:]), ("v", x[:, :, H + KVH:])):
        top = new.abs().amax(dim=-1)
        scale = torch.where(top == 0, torch.ones_like(top), top / torch.full_like(top, 127.0))
        s[name + "_codes"][at] = torch.round(new / scale[..., None]).clamp(-128, 127).to(torch.int8)
        s[name + "_scales"][at] = scale.to(torch.float16)
    s["slot_positions"][at] = s["positions"][..., None].expand(B, T, KVH)
    s["scores"][at] = 0.0
    return _plain_attend(s, turned[:, :, :H], s["lengths"] + T, _out_dtype(c))


def _plain_evict(s, scores, positions):
    c = s["case"]
    n, budget = c["cached"], c["budget"]
    slot = torch.arange(n, device=scores.device)
    live = slot < s["lengths"][:, None, None]
    key = torch.where(torch.isnan(scores[..., :n]), torch.full_like(scores[..., :n], float("-inf")), scores[..., :n]).double()
    key = torch.where(positions[..., :n] >= (s["seen"] - c["recent"])[:, None, None], torch.full_like(key, float("inf")), key)
    order = torch.argsort(key.masked_fill(~live, float("-inf")), dim=-1, descending=True, stable=True)
    kept = torch.zeros(order.shape, dtype=torch.bool, device=order.device).scatter_(
        -1, order, (slot < budget).expand(order.shape)) & live
    over = (s["lengths"] > budget)[:, None, None]
    kept = torch.where(over, kept, live)
    hole, donor = ~kept & (slot < budget) & over, kept & (slot >= budget)
    b, h, to = torch.nonzero(hole, as_tuple=True)  # both in ascending order a head, equally many
    at = torch.nonzero(donor, as_tuple=True)[2]
    for t in (s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], scores, positions):
        t[b, h, to] = t[b, h, at]
    return torch.clamp(s["lengths"], max=budget)


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    col = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((B, 1), float(np.float32(v)), dtype=torch.float64, device=x.device)
    temperature, top_k, top_p, min_p = (col(s[k]) for k in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = temperature <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    w = torch.where(greedy, (torch.arange(V, device=x.device) == 0).double(), w)
    kth = torch.gather(x, 1, torch.where(top_k > 0, top_k, torch.full_like(top_k, V)).clamp(1, V).long() - 1)
    w = torch.where(x >= kth, w, torch.zeros_like(w))
    before = torch.cumsum(w, dim=-1) - w
    keep = (before <= top_p * w.sum(dim=-1, keepdim=True)) | (top_p >= 1)
    w = torch.where(keep & (w >= min_p), w, torch.zeros_like(w))
    run_ = torch.cumsum(w, dim=-1)
    at = (run_ <= s["u"].double()[:, None] * run_[:, -1:]).sum(dim=-1, keepdim=True).clamp(max=V - 1)
    logprob = torch.log(torch.gather(w, 1, at) / run_[:, -1:])
    return torch.gather(order, 1, at)[:, 0].to(torch.int32), logprob[:, 0].float()


# ---- one pass ----------------------------------------------------------------
_calls = None


def _framework():
    global _calls
    if _calls is None:
        from siliconfer_amd.kernels.attention import attention_decode_scored
        from siliconfer_amd.kernels.eviction import evict
        from siliconfer_amd.kernels.rotary import rotary, rotary_kv_append
        from siliconfer_amd.kernels.sampling import sample
        _calls = dict(attend=attention_decode_scored, evict=evict, rotary=rotary,
                      append=rotary_kv_append, sample=sample)
    return _calls


def run(state: dict):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "rotary":
        if own:
            return _framework()["rotary"](s["q"], s["k"], s["positions"], s["inv_freq"],
                                          interleaved=c["interleaved"], scale=s["scale"])
        return _plain_rotary(s)
    if kind == "sample":
        if own:
            return _framework()["sample"](s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                          top_p=s["top_p"], min_p=s["min_p"], logprobs=True)
        return _plain_sample(s)
    if kind == "evict":
        # scores and positions as a decode loop would hand them in again: a pass moves
        # them with the cache, and the next pass is to have the same choice to make
        meta = s["meta"].clone()
        scores, positions = meta[0].view(torch.float32), meta[1]
        if own:
            lengths = _framework()["evict"](s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], scores,
                                            positions, s["lengths"], s["seen"], c["budget"], c["recent"])
        else:
            lengths = _plain_evict(s, scores, positions)
        # the codes are moved and not computed: they come back as they are, beside their scales
        return {"lengths": lengths, "scores": scores, "positions": positions, "k": s["k_codes"],
                "k_scales": s["k_scales"], "v": s["v_codes"], "v_scales": s["v_scales"]}
    if own:
        f = _framework()
        q, add = (s["q"], 0) if kind == "attend" else (
            f["append"](s["qkv"], s["positions"], s["inv_freq"], s["k_codes"], s["k_scales"], s["v_codes"],
                        s["v_scales"], n_heads=c["heads"], lengths=s["lengths"],
                        slot_positions=s["slot_positions"], scores=s["scores"]), c["rows"])
        out = f["attend"](q, s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["scores"],
                          lengths=s["lengths"], add=add, out_dtype=_out_dtype(c))
    elif kind == "attend":
        out = _plain_attend(s, s["q"], s["lengths"], _out_dtype(c))
    else:
        out = _plain_step(s)
    return {"out": out, "scores": s["scores"]}


def work(case: dict) -> dict:
    kind, B = case["kind"], case["batch"]
    if kind == "sample":
        n = B * case["vocab"]
        return {"bytes": n * _SIZE[case["dtype"]] + 12 * B, "flops": 4 * n}
    KVH, D = case["kv_heads"], case["dim"]
    if kind == "rotary":
        heads = B * case["rows"] * (case["heads"] + KVH)
        return {"bytes": 2 * heads * D * _SIZE[case["dtype"]] + 4 * B * case["rows"], "flops": 3 * heads * case["rot"]}
    n = case["cached"]
    n_all = n + (B - 1) * 0.65 * n if B > 1 else n  # the sequences' expected lengths together
    if kind == "evict":
        # every score and position read (and copied); the kept slots behind the budget move
        # into the holes before it: budget (n - budget) / n of them where the choice is even
        budget = case["budget"]
        over = [n] + [0.65 * n] * (B - 1)
        moved = sum(budget * (1 - budget / m) for m in over if m > budget)
        return {"bytes": KVH * (n_all * 8 + moved * 2 * (2 * D + 12)), "flops": KVH * n_all}
    rows = B * case["rows"] * case["heads"] * D
    flops = 4.0 * n_all * case["rows"] * case["heads"] * D
    bytes_ = KVH * n_all * (2 * D + 4 + 8) + rows * (_SIZE[case["dtype"]] + (4 if _out_dtype(case) == torch.float32 else 2))
    if kind == "step":
        bytes_ += B * case["rows"] * KVH * (2 * D * 5)
    return {"bytes": bytes_, "flops": flops}


# ---- 64 bits -----------------------------------------------------------------
def _turn64(x, angle, scale, interleaved):
    """Pairs as complex numbers times scale e^(i angle); x [B, T, heads, D] in 64 bits."""
    r = 2 * angle.shape[-1]
    pairs = x[..., :r].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    axis = -1 if interleaved else -2
    z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1)) * torch.polar(torch.full_like(angle, scale), angle)[:, :, None]
    y = torch.stack([z.real, z.imag], dim=axis).flatten(-2)
    return torch.cat([y, x[..., r:]], dim=-1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "sample":
        lp = torch.empty(case["batch"], dtype=torch.float64)
        for b in range(case["batch"]):
            get = lambda k: float(s[k][b]) if isinstance(s[k], torch.Tensor) else float(np.float32(s[k]))
            x = np.sort(s["logits"][b].double().cpu().numpy())[::-1]
            if get("temperature") <= 0:
                lp[b] = 0.0
                continue
            w = np.exp((x - x[0]) / get("temperature"))
            k = int(get("top_k"))
            if 0 < k < w.size:
                w = w[:int(np.searchsorted(-x, -x[k - 1], side="right"))]
            if get("top_p") < 1:
                w = w[:int(np.searchsorted(np.cumsum(w) - w, get("top_p") * w.sum(), side="right"))]
            w = w[w >= get("min_p")]
            at = int(np.searchsorted(np.cumsum(w), float(s["u"][b]) * w.sum(), side="right"))
            lp[b] = math.log(w[min(at, w.size - 1)] / w.sum())
        return None, lp
    if kind == "evict":
        return None  # nothing is computed: the outputs are the inputs' own values
    if kind == "rotary":
        angle = s["positions"].double()[..., None] * s["inv_freq"]
        return tuple(_turn64(s[k].double(), angle, s["scale"], case["interleaved"]) for k in ("q", "k"))
    B, T, H, KVH, D = case["batch"], case["rows"], case["heads"], case["kv_heads"], case["dim"]
    G = H // KVH
    lengths = s["lengths"].tolist()
    kv = [(s[k + "_codes"].double() * s[k + "_scales"].double()[..., None]) for k in ("k", "v")]
    scores = s["scores"].double()
    if kind == "step":
        x = s["qkv"].double().reshape(B, T, H + 2 * KVH, D)
        turned = _turn64(x[:, :, :H + KVH], s["positions"].double()[..., None] * s["inv_freq"], 1.0, False)
        q = turned[:, :, :H]
        for b in range(B):
            for t in range(T):
                at = lengths[b] + t
                for y, new in zip(kv, (turned[b, t, H:], x[b, t, H + KVH:])):
                    # codes from the values as they are held in 32 bits, the scale as stored
                    f = new.float()
                    sc = f.abs().amax(-1, keepdim=True).cpu().numpy() / np.float32(127)
                    codes = np.rint(f.cpu().numpy() / np.where(sc == 0, 1, sc).astype(np.float32))
                    y[b, :, at] = torch.from_numpy(codes.astype(np.float64) * sc.astype(np.float16).astype(np.float64)).to(y.device)
                scores[b, :, at] = 0.0
            lengths[b] += T
    else:
        q = s["q"].double()
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=q.device)
    for b in range(B):
        for t in range(T):
            m = lengths[b] - T + t + 1
            if m <= 0:
                continue
            for h in range(KVH):
                w = torch.softmax(q[b, t, h * G:(h + 1) * G] @ kv[0][b, h, :m].T / math.sqrt(D), dim=-1)
                out[b, t, h * G:(h + 1) * G] = w @ kv[1][b, h, :m]
                scores[b, h, :m] += w.sum(dim=0)
    return {"out": out, "scores": scores}
