"""Forward-mode derivatives of the turned (and normed) heads are refused, not dropped."""

import pytest
import torch
from torch.autograd import forward_ad

from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.rotary import qk_norm_rotary, rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("at", range(4))
def test_tangents_are_refused(dev, at, grad):
    x = [torch.randn(1, 3, 2, 64, device=dev), torch.randn(1, 3, 1, 64, device=dev), torch.ones(64, device=dev), torch.ones(64, device=dev)]
    pos, f = torch.arange(3, device=dev), torch.ones(32, dtype=torch.float64, device=dev)
    x[0].requires_grad_(grad)
    calls = [lambda q, k, a, b: qk_norm_rotary(q, k, pos, f, a, b)] + ([lambda q, k, a, b: rotary(q, k, pos, f)] if at < 2 else [])
    for call in calls:
        want = call(*x)
        with forward_ad.dual_level():
            assert all(torch.equal(a, b) for a, b in zip(call(*x), want))  # (no tangent: as ever)
            with pytest.raises(SFError, match="forward-mode"):
                call(*(forward_ad.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate(x)))
