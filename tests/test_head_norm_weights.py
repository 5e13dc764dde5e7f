"""Head norms of a checkpoint that are of another kind are refused, without a GPU."""

import numpy as np
import pytest

from siliconfer_amd._lib import SFError
from siliconfer_amd.model import TransformerBlock, compute_rope_freqs
from test_q4_cache import CFG, weights

AT = "model.layers.0.self_attn"


@pytest.mark.parametrize("side", "qk")
@pytest.mark.parametrize("shape", [(1,), (), (64,), (128,), (4, 32), (1, 32)])
def test_weights_of_another_shape(side, shape):
    """One weight for all dims, or one a dim of the whole projection (a norm over all heads together)."""
    w = weights(norms="qk") | {f"{AT}.{side}_norm.weight": np.ones(shape, np.float32)}
    with pytest.raises(SFError, match=f"{side}_norm.weight"):
        TransformerBlock.from_weights(CFG, w, 0, compute_rope_freqs(CFG), device="cpu")


def test_a_bias():
    w = weights(norms="qk") | {f"{AT}.k_norm.bias": np.ones(32, np.float32)}
    with pytest.raises(SFError, match="bias"):
        TransformerBlock.from_weights(CFG, w, 0, compute_rope_freqs(CFG), device="cpu")
