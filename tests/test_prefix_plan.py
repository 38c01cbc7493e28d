"""The plan of an attention behind a shared prefix: tiles and parts of a call of any accepted size fit their launches, and small calls
are split as their times were measured.  Plain host code (csrc/prefix_args.h)."""

import ctypes
import os
import shutil
import subprocess

import pytest

from helpers import PKG_DIR

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")

SHIM = """
#include "prefix_args.h"
using namespace anima;
extern "C" void t_plan(int cus, int bf, int V, int group, int Hkv, int T, int P, int longest, int* out) {
  const PrefixPlan p = prefix_plan(cus, bf, V, group, Hkv, T, P, longest);
  out[0] = p.waves; out[1] = p.nt; out[2] = p.splits; }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("prefix_plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))

    def go(bf, T, P, H, Hkv, longest, cus=256):
        out = (ctypes.c_int * 3)()
        lib.t_plan(cus, bf, T * (H // Hkv), H // Hkv, Hkv, T, P, longest, out)
        return tuple(out)

    return go


@pytest.mark.parametrize("bf", [0, 1])
@pytest.mark.parametrize("P", [0, 100, 8192, 1 << 22])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (16, 8), (32, 32), (4096, 1), (4096, 4096)])
def test_launches(plan, bf, P, H, Hkv):
    """Fewer than 2^32 threads of the tiles and of the join, for every number of rows of all heads up to 2^30; the parts' sums (520
    bytes a row) stay below 36 GB."""
    for T in [1, 3, 77, 1000] + [(1 << e) + d for e in range(11, 23) for d in (-1, 0, 1, 12345)]:
        if T > 1 << 22 or T * H > 1 << 30:
            continue
        for longest in {1, min(T, 64), T}:
            nw, nt, s = plan(bf, T, P, H, Hkv, longest)
            assert nw in (4, 8) and nt == -(-T * (H // Hkv) // (32 * nw)) and 1 <= s <= 64
            assert nt * Hkv * s * 64 * nw < 1 << 32, (T, longest, nw, nt, s)
            if s > 1:
                assert -(-T * H // 8) * 256 < 1 << 32 and s * T * H * 520 < 36e9, (T, longest, s)


def test_small_calls(plan):
    """One wave of rows behind three blocks at most: whole; few rows behind a long prefix: in parts."""
    for T, P, H, Hkv in ((2, 77, 16, 8), (1, 128, 32, 8), (5, 100, 32, 8), (2, 120, 8, 1), (30, 70, 3, 3), (8, 128, 15, 5)):
        assert plan(1, T, P, H, Hkv, T)[2] == 1
    assert plan(1, 64, 8192, 32, 8, 1)[2] > 8
