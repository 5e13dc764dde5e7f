"""Refusals of the 4-bit attention's C entry without a GPU: where its output may start."""

import pytest

from test_q4_refusals import P, attend, refused


@pytest.mark.parametrize("kw", [dict(out=P + 8), dict(out=P + 2, Tq=1500, T=100), dict(out=P + 4, n_splits=2)])
def test_out_starts_on_16_bytes(kw):
    refused(attend(**kw), -1, "16-byte")
