"""The layer norm's launch rule (layer_norm_shape.cuh) swept over every width on
the host: the threads, registers and shared memory it asks for are those that the
kernel instances were built for."""
import ctypes
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "packr_b200" / "csrc"
# Runs the rule and returns the number of widths that break it, the first in *bad.
SWEEP = r"""
#include "layer_norm_shape.cuh"
using namespace packr::norm;
extern "C" long long sweep(long long M, long long lo, long long hi, int esize, int tensors, int bwd, long long* bad) {
  long long n = 0;
  for (long long N = lo; N <= hi; ++N) {
    if (wide(N)) continue;
    const Shape s = shape(M, N, esize, tensors, bwd != 0, 148);
    const int vw = 16 / esize;
    const long long span = N % vw ? N + vw - 1 : N;
    // instances that exist: forward 8 and 16 elements with 256 threads, 32 with 256 or 512;
    // backward 8 with 256, 16 with 256, 512 or 1024
    const int most = bwd ? (s.e == 8 ? 256 : 1024) : (s.e == 32 ? 512 : 256);
    bool ok = s.e == 8 || s.e == 16 || (s.e == 32 && !bwd);
    ok = ok && s.tmax <= most && s.nt * s.groups <= s.tmax && s.nt % 32 == 0 && s.nt >= 32;
    ok = ok && (long long)s.nt * s.e >= span && s.groups >= 1 && s.groups <= kMaxGroups && s.groups <= M;
    ok = ok && s.smem <= (size_t)kMaxSmem && (s.stages >= 1 || (bwd && s.nt > 512)) && s.grid >= 1;
    // a group's rows are a whole number of phases apart unless it has one row only
    ok = ok && (N % vw == 0 || (long long)s.grid * s.groups >= M || s.grid % vw == 0);
    if (!ok && n++ == 0) *bad = N;
  }
  return n;
}
"""


@pytest.fixture(scope="module")
def sweep(tmp_path_factory):
    d = tmp_path_factory.mktemp("norm_shape")
    (d / "sweep.cpp").write_text(SWEEP)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(d / "sweep.cpp"), "-o",
                    str(d / "sweep.so")], check=True)
    f = ctypes.CDLL(str(d / "sweep.so")).sweep
    f.restype = ctypes.c_longlong
    f.argtypes = [ctypes.c_longlong] * 3 + [ctypes.c_int] * 3 + [ctypes.POINTER(ctypes.c_longlong)]
    return f


@pytest.mark.parametrize("bwd", [0, 1])
@pytest.mark.parametrize("esize", [2, 4])
def test_every_width_gets_an_instance_that_holds_it(sweep, esize, bwd):
    bad = ctypes.c_longlong(0)
    for M in (1, 3, 100, 100000):
        for residual in (0, 1):
            n = sweep(M, 1, 16400, esize, 1 + residual + bwd, bwd, ctypes.byref(bad))
            assert n == 0, f"{n} widths, the first {bad.value}, at {M} rows"
