"""The sampler's fp64 exponential (csrc/exp_neg.cuh), compiled for the host: its additions, multiplications
and fused multiply-adds are those of the device."""
import ctypes
import subprocess

import numpy as np
import pytest

from .conftest import ROOT

SHIM = """
#include <cmath>
#include <cstdint>
#include <cstring>
#define __device__
#define __forceinline__ inline
using std::fma;
static double __hiloint2double(int hi, int lo) {
  const uint64_t b = (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
  double d;
  std::memcpy(&d, &b, 8);
  return d;
}
static int __double2loint(double d) {
  uint64_t b;
  std::memcpy(&b, &d, 8);
  return (int)(uint32_t)b;
}
#include "exp_neg.cuh"
extern "C" void run(const double* x, double* y, long n) {
  for (long i = 0; i < n; ++i) y[i] = sq::exp_neg(x[i]);
}
"""


@pytest.fixture(scope="module")
def exp_neg(tmp_path_factory):
    d = tmp_path_factory.mktemp("exp_neg")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-I",
                    f"{ROOT}/squish_b200/csrc", "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))

    def f(x):
        x = np.ascontiguousarray(x, dtype=np.float64)
        y = np.empty_like(x)
        p = ctypes.POINTER(ctypes.c_double)
        lib.run(x.ctypes.data_as(p), y.ctypes.data_as(p), ctypes.c_long(x.size))
        return y

    return f


def test_error_stays_within_four_ulp(exp_neg):
    rng = np.random.default_rng(0)
    half = (np.arange(1, 1020) - 0.5) * np.log(2)  # where the reduction changes its multiple of ln 2
    x = -np.concatenate([rng.uniform(0, 707, 200000), rng.uniform(0, 1, 100000), 10.0 ** rng.uniform(-18, 0, 50000),
                         half, half * (1 + 1e-15), half * (1 - 1e-15), np.arange(707.0)])
    assert np.finfo(np.longdouble).nmant >= 63
    want = np.exp(x.astype(np.longdouble))  # 64-bit mantissa: 2^-11 ulp of a double
    err = np.abs(exp_neg(x).astype(np.longdouble) - want) / np.spacing(want.astype(np.float64)).astype(np.longdouble)
    assert err.max() <= 4.0, float(err.max())


def test_ends_of_the_range(exp_neg):
    assert exp_neg([0.0, -0.0]).tolist() == [1.0, 1.0]
    assert exp_neg([-707.0, -708.0, -1e6, -1e300, -np.inf, np.nan]).tolist() == [0.0] * 6
    assert exp_neg([np.nextafter(-707.0, 0)])[0] > 0
