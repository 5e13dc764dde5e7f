"""Refusals of the 4-bit attention's C entry without a GPU: where its output may start, scales that are
no numbers."""

import pytest

from test_q4_refusals import P, attend, refused


@pytest.mark.parametrize("kw", [dict(out=P + 8), dict(out=P + 2, Tq=1500, T=100), dict(out=P + 4, n_splits=2)])
def test_out_starts_on_16_bytes(kw):
    refused(attend(**kw), -1, "16-byte")


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_a_scale_is_finite(scale):
    """(A NaN would have weighed every slot alike, an infinity as a large number.)"""
    refused(attend(scale=scale), -1, "not finite")
