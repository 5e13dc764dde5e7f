"""Rotary frequencies from a model's config (siliconfer_amd/model/rope.py), on the CPU: a checkpoint's
rope_scaling entry, read by ModelConfig.from_dict, gives what the entry itself gives."""

import dataclasses
import math

import numpy as np
import pytest

from siliconfer_amd._lib import SFError
from siliconfer_amd.model.config import ModelConfig, RoPEScalingConfig
from siliconfer_amd.model.rope import Rotary, rotary_frequencies

ENTRIES = [
    {"type": "linear", "factor": 4.0},
    {"type": "dynamic", "factor": 2.0},
    {"rope_type": "dynamic", "factor": 4.0, "original_max_position_embeddings": 2048},
    {"type": "yarn", "factor": 4.0},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 16.0, "beta_fast": 16.0, "beta_slow": 2.0},
    {"rope_type": "yarn", "factor": 4.0, "beta_fast": 16, "attention_factor": 1.0},
    {"type": "yarn", "factor": 4.0, "beta_fast": None, "attention_factor": None,
     "original_max_position_embeddings": None, "mscale": None, "truncate": True},
    {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 1024},
]


def config(entry):
    return ModelConfig.from_dict({"hidden_size": 512, "num_attention_heads": 8, "head_dim": 64, "rope_theta": 1e4,
                                  "max_position_embeddings": 4096, "rope_scaling": entry})


def closed(entry, length):
    """The published forms, pair by pair in plain arithmetic, of a head of 64 at theta 1e4."""
    e = {k: v for k, v in entry.items() if v is not None}
    kind, s, r, base = e.get("type", e.get("rope_type")), e["factor"], 64, 1e4
    trained = e.get("original_max_position_embeddings", 4096)
    f = [base ** (-2 * i / r) for i in range(r // 2)]
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind == "dynamic":
        n = max(length, trained)
        grown = base * (s * n / trained - (s - 1)) ** (r / (r - 2))
        return [grown ** (-2 * i / r) for i in range(r // 2)], 1.0
    if kind == "llama3":
        keep = [(trained * x / (2 * math.pi) - e["low_freq_factor"]) / (e["high_freq_factor"] - e["low_freq_factor"])
                for x in f]
        keep = [min(max(k, 0.0), 1.0) for k in keep]
        return [x / s * (1 - k) + x * k for x, k in zip(f, keep)], 1.0
    dim = lambda turns: r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(math.floor(dim(e.get("beta_fast", 32.0))), 0), min(math.ceil(dim(e.get("beta_slow", 1.0))), r - 1)
    ramp = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(r // 2)]
    return ([x / s * k + x * (1 - k) for x, k in zip(f, ramp)],
            e.get("attention_factor", 0.1 * math.log(s) + 1.0))


@pytest.mark.parametrize("entry", ENTRIES)
def test_a_config_gives_what_its_entry_gives(entry):
    want, scale = closed(entry, 8192)
    c = config(entry)
    for made in (c, ModelConfig.from_dict(c.to_dict())):  # (also after a round trip through a saved config)
        got = Rotary.from_config(made, length=8192)
        # a power, a logarithm and a few products in 64 bits: 2^-53 times the exponent's size (ln 1e5) and some steps
        assert np.allclose(got.inv_freq, want, rtol=64 * 2.0 ** -53, atol=0)
        assert math.isclose(got.scale, scale, rel_tol=1e-15)
    f, s = rotary_frequencies(64, 1e4, entry, trained=4096, length=8192)
    assert np.array_equal(got.inv_freq, f) and got.scale == s


def test_an_entry_made_by_hand():
    c = ModelConfig(head_dim=64, rope_theta=1e4, max_position_embeddings=4096, rope_scaling=RoPEScalingConfig("dynamic", 2.0))
    f, _ = rotary_frequencies(64, 1e4, {"type": "dynamic", "factor": 2.0}, trained=4096, length=8192)
    assert np.array_equal(Rotary.from_config(c, length=8192).inv_freq, f)
    c.rope_scaling = dataclasses.replace(c.rope_scaling, factor=4.0)
    f, _ = rotary_frequencies(64, 1e4, {"type": "dynamic", "factor": 4.0}, trained=4096, length=8192)
    assert np.array_equal(Rotary.from_config(c, length=8192).inv_freq, f)
    c.rope_scaling.original_max_position_embeddings = 2048
    f, _ = rotary_frequencies(64, 1e4, {"type": "dynamic", "factor": 4.0}, trained=2048, length=8192)
    assert np.array_equal(Rotary.from_config(c, length=8192).inv_freq, f)
    # the field reads as the reference has it, and its rule without one is llama3's
    assert RoPEScalingConfig("llama3", 8.0).original_max_position_embeddings == 8192
    assert config({"type": "llama3", "factor": 8.0}).rope_scaling.original_max_position_embeddings == 8192
    f, _ = rotary_frequencies(64, 1e4, {"type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192})
    assert np.array_equal(Rotary.from_config(config({"type": "llama3", "factor": 8.0})).inv_freq, f)


@pytest.mark.parametrize("field", [{"mscale": 1.0}, {"mscale_all_dim": 0.707}, {"truncate": False}])
def test_fields_that_would_change_the_result_are_refused(field):
    entry = {"type": "yarn", "factor": 4.0, **field}
    with pytest.raises(SFError, match=next(iter(field))):
        rotary_frequencies(64, 1e4, entry, trained=4096)
    with pytest.raises(SFError, match=next(iter(field))):
        Rotary.from_config(config(entry))


def test_frequencies_are_not_copied_while_a_graph_is_recorded(monkeypatch):
    """A copy from host memory would end the recording: a first on() there is refused."""
    import torch

    r = Rotary(*rotary_frequencies(16))
    cpu = torch.device("cpu")
    assert r.on("cpu") is r.on(cpu)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    assert r.on(cpu).shape == (8,)
    with pytest.raises(SFError, match="before a graph is recorded"):
        r.on(torch.device("cuda", 0))
