"""elm_quant.h's levels of a group with one reciprocal, compiled by the host compiler, against the divisions they stand for:
quotients on, beside and far from the points between two levels, scales of both signs and every magnitude."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include <cmath>
#define ELM_HOSTDEV
#include "elm_quant.h"
extern "C" void levels4(const float* v, const float* s, long groups, float* q) {
  for (long g = 0; g < groups; ++g) elm_level_group<4, -8, 7>(v + 4 * g, s[g], q + 4 * g);
}
extern "C" void levels8(const float* v, const float* s, long groups, float* q) {
  for (long g = 0; g < groups; ++g) elm_level_group<4, -127, 127>(v + 4 * g, s[g], q + 4 * g);
}
"""


@pytest.mark.parametrize("bits,lo,hi", [(4, -8, 7), (8, -127, 127)])
def test_one_reciprocal_gives_the_quotients_levels(tmp_path, bits, lo, hi):
    (tmp_path / "s.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-Wno-unknown-pragmas", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "edgelm_amd", "csrc"), str(tmp_path / "s.cpp"), "-o", str(tmp_path / "s.so")], check=True)
    lib = C.CDLL(str(tmp_path / "s.so"))
    rng = np.random.default_rng(0)
    n = 200000
    with np.errstate(all="ignore"):
        s = (rng.normal(0, 1, n) * 10.0 ** rng.integers(-44, 36, n)).astype(np.float32)
        s[(s == 0) | ~np.isfinite(s)] = 1
        top = -lo
        v = ((rng.integers(-top, top, (n, 4)) + 0.5) * s[:, None].astype(np.float64)).astype(np.float32)
        step = rng.integers(-2, 3, (n, 4))
        v = np.where(step < 0, np.nextafter(v, np.float32(-np.inf)), np.where(step > 0, np.nextafter(v, np.float32(np.inf)), v))
        v[::7] = (rng.uniform(-top, top, v[::7].shape) * s[::7, None]).astype(np.float32)
        v[::11, 0] = 0
        v[~np.isfinite(v)] = 0
        r = v / s[:, None]
        want = np.clip(np.copysign(np.floor(np.abs(r) + np.float32(0.5)), r), lo, hi).astype(np.int32)
    got, v = np.empty((n, 4), np.float32), np.ascontiguousarray(v)
    getattr(lib, f"levels{bits}")(v.ctypes.data_as(C.c_void_p), s.ctypes.data_as(C.c_void_p), C.c_long(n), got.ctypes.data_as(C.c_void_p))
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
