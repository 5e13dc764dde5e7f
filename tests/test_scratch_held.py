"""Large workspaces are a call's own, without a GPU: a thread does not keep them for good."""

import pytest
import torch

from siliconfer_amd import _lib
from siliconfer_amd.kernels import attention

CPU = torch.device("cpu")


@pytest.mark.parametrize("get", [_lib.scratch, attention.workspace], ids=["scratch", "attention"])
def test_a_large_one_is_not_kept(monkeypatch, get):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    small = get(CPU, 21, 1000)
    large = get(CPU, 21, (64 << 20) + 1)
    assert large.numel() > 64 << 20 and large.data_ptr() != small.data_ptr()
    assert get(CPU, 21, 1000).data_ptr() == small.data_ptr()
    assert get(CPU, 21, (64 << 20) + 1).data_ptr() != large.data_ptr()  # (large is still in use)
    most = get(CPU, 21, 64 << 20)
    assert get(CPU, 21, 1000).data_ptr() == most.data_ptr()
    assert max(t.numel() for t in _lib._scratch.held.values()) <= 64 << 20
