"""Rotary frequencies and their scalings (siliconfer_amd/model/rope.py), on the CPU."""

import math

import numpy as np
import pytest

from siliconfer_amd._lib import SFError
from siliconfer_amd.model.config import ModelConfig, RoPEScalingConfig, rope_freqs
from siliconfer_amd.model.rope import Rotary, rotary_frequencies


def test_default_and_linear():
    f, s = rotary_frequencies(64, 1e6)
    assert s == 1.0 and f.dtype == np.float64 and f.shape == (32,)
    assert f[0] == 1.0 and math.isclose(f[31], 1e6 ** (-62 / 64), rel_tol=1e-14)
    g, s = rotary_frequencies(64, 1e6, {"type": "linear", "factor": 4.0})
    assert s == 1.0 and np.array_equal(g, f / 4)


def test_llama3_is_the_configuration_s():
    c = ModelConfig(head_dim=128, rope_theta=500000.0,
                    rope_scaling=RoPEScalingConfig("llama3", 8.0, 1.0, 4.0, 8192))
    r = Rotary.from_config(c)
    # fp32 powers, divisions and the ramp there: a few steps of 2^-24, more where the exponent of a power
    # with a large logarithm is rounded (ln(5e5) 2^-24 relative)
    assert np.allclose(r.inv_freq, rope_freqs(c), rtol=2 * math.log(5e5) * 2.0 ** -23, atol=0)
    assert r.scale == 1.0 and not r.interleaved


def test_dynamic():
    f, _ = rotary_frequencies(64, 1e4)
    same, _ = rotary_frequencies(64, 1e4, {"rope_type": "dynamic", "factor": 2.0}, trained=2048, length=1000)
    assert np.allclose(same, f, rtol=1e-14, atol=0)
    far, _ = rotary_frequencies(64, 1e4, {"rope_type": "dynamic", "factor": 2.0}, trained=2048, length=4096)
    # the slowest pair at length 4096 = 2 x 2048 turns 3 times slower (2 * 2 - 1), the fastest as before
    assert far[0] == 1.0 and math.isclose(far[31], f[31] / 3, rel_tol=1e-12)


def test_yarn():
    f, _ = rotary_frequencies(128, 1e4)
    sc = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    y, s = rotary_frequencies(128, 1e4, sc)
    assert math.isclose(s, 0.1 * math.log(16) + 1)
    turns = 4096 * f / (2 * math.pi)
    assert np.array_equal(y[turns > 40], f[turns > 40])           # fast pairs as they are
    assert np.allclose(y[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-14, atol=0)  # slow ones stretched
    between = (turns < 30) & (turns > 1.2)
    assert (y[between] < f[between]).all() and (y[between] > f[between] / 16).all()
    assert rotary_frequencies(128, 1e4, dict(sc, attention_factor=0.5))[1] == 0.5


def test_part_of_the_head():
    c = ModelConfig(head_dim=96, rope_theta=1e4)
    assert Rotary.from_config(c, rotary_dim=32, interleaved=True).inv_freq.shape == (16,)
    with pytest.raises(SFError, match="exceeds the head"):
        Rotary.from_config(c, rotary_dim=98)


@pytest.mark.parametrize("args", [(0,), (3,), (64, 0.0), (64, 1e4, {"type": "nonesuch"}),
                                  (64, 1e4, {"type": "yarn", "factor": 2.0}), (64, 1e4, {"type": "linear", "factor": 0}),
                                  (2, 1e4, {"type": "dynamic", "factor": 2.0}, 100)])
def test_refusals(args):
    with pytest.raises(SFError):
        rotary_frequencies(*args)
