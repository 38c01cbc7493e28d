"""Products of 4-bit weights that are too large for one launch: a launch has fewer than 2^32 threads a dimension, so rows and
columns are cut into several launches."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from helpers import PKG_DIR, amd
from test_f8_launch import Large

SHIM = """
#include "q4_args.h"
using namespace anima;
extern "C" {
int64_t t_rows(int64_t M, int64_t N) { return q4_part(M, N).rows; }
int64_t t_cols(int64_t M, int64_t N) { return q4_part(M, N).cols; }
}
"""


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("q4_launch")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    for f in (lib.t_rows, lib.t_cols):
        f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64]
    return lib


SIDES = [1, 3, 5, 63, 64, 65, 1000, 2048, 4097, 1 << 14, (1 << 14) + 1, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, 1 << 26, (1 << 28) + 37, 1 << 29]


@pytest.mark.parametrize("M", SIDES)
def test_parts(parts, M):
    """Threads of every kernel that a part may take, at the part's size."""
    for N in SIDES:
        r, n = parts.t_rows(M, N), parts.t_cols(M, N)
        assert 1 <= r <= M and 1 <= n <= N
        up = lambda a, b: -(-a // b)
        threads = {"pass": 256 * (up(r, 4) + up(n, 4)), "vector": 256 * up(n, 16), "vector, one column": 256 * up(min(n, 4095), 4), "few": 512 * up(n, 32)}
        for bm, bn in ((64, 64), (64, 128), (64, 256), (128, 128), (128, 256)):
            threads[f"{bm} x {bn}"] = 256 * up(r, bm) * up(n, bn)
        assert max(threads.values()) < 1 << 32, (M, N, threads)
        # what was one launch stays one, and parts start where codes, scales and their vector loads are aligned
        assert (r, n) == (M, N) or M > 1 << 24 or N > 1 << 24 or M * N > 1 << 35
        assert n == N or n % 256 == 0


# ------------------------------------------------------------------ on the GPU


@pytest.fixture
def ctx():
    c = amd().Context(0)
    yield c
    c.close()


def around(total, cuts):
    return [8] + [c for c in cuts if c < total - 24] + [total - 8]


@pytest.mark.gpu
@pytest.mark.parametrize("mid,precision", [(False, 1), (True, 0)], ids=["sym", "mid"])
def test_rows_of_several_launches(ctx, mid, precision):
    """2^26 rows and more: the pass before them were 2^32 threads in one launch; out += gate * r."""
    import test_q4_gpu as ref

    M, N, K, g = (1 << 26) + 37, 3, 32, 32
    print(f"[case] {M} x {N} x {K}", flush=True)
    rng = np.random.default_rng(6)
    W = ref.Q4(ctx, rng, N, K, g, mid, bias=rng.normal(size=N).astype(np.float32))
    cuts = around(M, [i << 24 for i in range(1, 5)])
    x, out, add = Large(ctx, M, K, np.float32, cuts), Large(ctx, M, N, np.float32, cuts), Large(ctx, M, N, np.float32, cuts)
    xs = [rng.normal(size=(b - a, K)).astype(np.float32) for a, b in x.at]
    os_, ad = ([rng.normal(size=(b - a, N)).astype(np.float32) for a, b in x.at] for _ in range(2))
    gate = rng.normal(size=N).astype(np.float32)
    x.write(xs)
    out.write(os_)
    add.write(ad)
    ctx.linear(W.w, M, out.ptr, x=x.ptr, epilogue=2, gate=ctx.upload(gate), add=add.ptr, precision=precision)
    for x0, o0, a0, got in zip(xs, os_, ad, out.read()):
        r = x0.astype(np.float64) @ W.values.T + W.bias + a0
        want = o0 + gate * r
        more = 2.0 ** -12 * (np.abs(x0.astype(np.float64)) @ np.abs(W.values).T) if precision == 0 else 0.0  # (x to 11 bits: 2^-11 in all)
        tol = (more + ref.bound(x0.astype(np.float64), W.values, K, precision, False, want, r) + 4 * ref.BIT_EPS * (np.abs(W.bias) + np.abs(a0))) * \
            np.maximum(1, np.abs(gate)) + 4 * ref.BIT_EPS * np.abs(o0)
        assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("M,mid,N", [(1, True, (1 << 28) + 37), (5, False, (1 << 28) + 37), (5, True, (1 << 26) + 37)])
def test_columns_of_several_launches(ctx, M, mid, N):
    """2^28 columns and more were 2^32 threads of the kernels for few rows, 2^26 of them with middles of the pass before."""
    import test_q4_gpu as ref

    m = amd()
    K, g = 32, 32
    print(f"[case] {M} x {N} x {K}", flush=True)
    rng = np.random.default_rng(7)
    cuts = around(N, [i << 24 for i in range(1, 17)])
    w, s, z = Large(ctx, N, K // 2, np.uint8, cuts), Large(ctx, N, 1, np.uint16, cuts), Large(ctx, N, 1, np.uint16, cuts) if mid else None
    bias = Large(ctx, N, 1, np.float32, cuts)
    codes = [rng.integers(0, 16, (b - a, K)).astype(np.uint8) for a, b in w.at]
    sc, zc, bc = ([ref.widen(ref.bf16(f * rng.normal(size=(b - a, 1)))) for a, b in w.at] for f in (0.1, 0.1, 1.0))
    w.write([ref.pack(c) for c in codes])
    s.write([ref.bf16(v) for v in sc])
    if mid:
        z.write([ref.bf16(v) for v in zc])
    bias.write(bc)
    W = m.weight(m.W_Q4, N, K, w.ptr, group=g, group_scale=s.ptr, group_mid=z.ptr if mid else None, bias=bias.ptr)
    x = rng.normal(size=(M, K)).astype(np.float32)
    out = ctx.empty((M * N,))
    ctx.linear(W, M, out, x=ctx.upload(x), precision=m.PREC_FP32)
    x64 = x.astype(np.float64)
    for i, (a, b) in enumerate(w.at):
        v = ref.values(codes[i], sc[i], zc[i] if mid else None, g)
        want = x64 @ v.T + bc[i][:, 0]
        tol = ref.bound(x64, v, K, 1, False, want, want) + 4 * ref.BIT_EPS * np.abs(bc[i][:, 0])
        got = np.empty((M, b - a), np.float32)
        for r in range(M):
            ctx._check(m.lib().anima_d2h(ctx.h, got[r].ctypes.data, out.ptr + (r * N + a) * 4, got[r].nbytes))
        assert np.all(np.abs(got - want) <= tol), (a, (np.abs(got - want) / tol).max())
