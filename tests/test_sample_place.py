"""The bins of sf_sample (siliconfer_amd/csrc/sample_place.h), compiled for the host: a logit's place
within its bin, and with it its weight, is the same whichever maximum the bins are counted from, so
that a row's sums over its chunks' bins are the sums over the row's own."""

import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "siliconfer_amd", "csrc")

SHIM = r"""
#include <xmmintrin.h>
#include "sample_place.h"
// of n logits: bins and weights below the bin of the maximum m; returns the bin number of m
extern "C" double bins(const float *x, long n, double temperature, float m, int *bin, unsigned long long *w) {
  const unsigned mode = _mm_getcsr();  // a library that is loaded beside may have turned subnormals off; kernels have them
  _mm_setcsr(mode & ~0x8040u);
  const volatile float T = (float)temperature;
  const double per = bins_per_logit(T), top = top_bin(m, per);
  for (long i = 0; i < n; ++i) {
    const Binned b = bin_of(x[i], per, top);
    bin[i] = b.bin;
    w[i] = b.w;
  }
  _mm_setcsr(mode);
  return top;
}
"""


@pytest.fixture(scope="module")
def bins(tmp_path_factory):
    d = tmp_path_factory.mktemp("place")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-I", CSRC, str(d / "shim.cpp"),
                    "-o", str(d / "shim.so")], check=True)
    f = ctypes.CDLL(str(d / "shim.so")).bins
    f.restype = ctypes.c_double
    f.argtypes = [ctypes.c_void_p, ctypes.c_long, ctypes.c_double, ctypes.c_float, ctypes.c_void_p, ctypes.c_void_p]

    def call(x, T, m):
        x = np.ascontiguousarray(x, np.float32)
        b, w = np.empty(x.size, np.int32), np.empty(x.size, np.uint64)
        top = f(x.ctypes.data, x.size, T, m, b.ctypes.data, w.ctypes.data)
        return b, w, top
    return call


CASES = [(T, lambda r, T=T: r.normal(0, 4 * T, 20000)) for T in (0.3, 0.7, 1.0, 1.37, 30.0, 1e30)] + [
    # (places around -1.5 2^20, -2^19, 2^19, 0 and past 2^53 bins)
    (1e-4, lambda r: -19.6608 + r.uniform(-0.003, 0.003, 20000)), (1.0, lambda r: -196608 + r.uniform(-31, 0, 20000)),
    (1.0, lambda r: -65536 + r.uniform(-20, 20, 20000)), (1.0, lambda r: 65536 + r.uniform(-20, 20, 20000)),
    (1.0, lambda r: r.normal(0, 1e-40, 20000)), (1.0, lambda r: r.uniform(-0.1, 0.1, 20000) * 2.0 ** r.integers(-30, 0, 20000)),
    (1e-44, lambda r: r.normal(0, 1, 20000)), (math.inf, lambda r: r.normal(0, 1e30, 20000)),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_places_do_not_depend_on_the_maximum(bins, case):
    T, draw = CASES[case]
    x = draw(np.random.default_rng(case)).astype(np.float32)
    x = np.sort(x)[::-1]
    x = np.concatenate([x, [np.float32(-np.inf), np.float32(np.nan)]])
    b0, w0, top0 = bins(x, T, x[0])
    assert b0[0] == 0 and (b0[-2:] >= 256).all() and (np.diff(b0[:-2]) >= 0).all()
    for first in (1, 7, 100, 1000, 5000, 15000):
        b, w, top = bins(x[first:], T, x[first])
        assert b[0] == 0
        inside = (b < 256) & (b0[first:] < 256)
        assert (b0[first:][inside] - b[inside] == top0 - top).all()
        assert np.array_equal(w[inside], w0[first:][inside]), (T, first, int((w[inside] != w0[first:][inside]).sum()))
        # who is inside the row's bins is inside the chunk's
        assert (b[b0[first:] < 256] < 256).all()


def test_weights(bins):
    """A weight is 2^36 e^y, y the distance from its bin's middle: 3e-10 of itself and the place's 2^-33 of a bin."""
    r = np.random.default_rng(0)
    for T in (0.5, 1.0, 2.0):
        x = np.sort(r.uniform(-31 * T, 0, 5000).astype(np.float32))[::-1]
        _, w, _ = bins(x, T, x[0])
        z = x.astype(np.float64) / (0.125 * T)
        part = z - np.floor(z)
        clear = (part > 2.0 ** -30) & (part < 1 - 2.0 ** -30)  # (of a border between two bins)
        want = 2.0 ** 36 * np.exp(0.125 * (part - 0.5))
        assert clear.sum() > 4900 and np.allclose(w[clear].astype(np.float64), want[clear], rtol=4e-10)
