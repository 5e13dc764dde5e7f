"""make_quantized_cache at 4 bits, without a GPU: what it cannot hold is refused."""

import pytest
import torch

from siliconfer_amd._lib import SFError
from siliconfer_amd.model import make_quantized_cache


def test_scales_of_another_type():
    assert make_quantized_cache(1, 8, torch.float16, 4)[0].capacity == 8
    assert make_quantized_cache(1, 8, torch.float32)[0].scale_dtype is torch.float32
    for dtype in (torch.float32, torch.bfloat16):
        with pytest.raises(SFError, match="float16"):
            make_quantized_cache(1, 8, dtype, bits=4)
