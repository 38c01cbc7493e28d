"""Calls of the e4m3 operators that are too large for one launch: a launch has fewer than 2^32 threads a dimension, so rows
are cut into several launches, and what no launch can hold is refused with a message."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from helpers import PKG_DIR, amd
from test_f8_args import P, call, v, weight

SHIM = """
#include "f8_args.h"
using namespace anima;
extern "C" {
int64_t t_quant_part(int K) { return f8_quant_part(K); }
int64_t t_norm_part(int threads) { return f8_norm_part(threads); }
int t_wquant(const void* w, int b, int N, int K, const uint8_t* q, const float* s, char* m, size_t n) {
  return check_weight_quant_f8(w, b, N, K, q, s, F8Msg{m, n}); }
int t_linear(const anima_linear_desc* d, char* m, size_t n) { return check_linear_f8(d, F8Msg{m, n}); }
int t_glu(const anima_glu_desc* d, char* m, size_t n) { return check_linear_glu(d, F8Msg{m, n}); }
}
"""


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("f8_launch")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.t_quant_part.restype = lib.t_norm_part.restype = ctypes.c_int64
    return lib


@pytest.mark.parametrize("K", [16, 128, 144, 2048, 1 << 20, (1 << 31) - 128, (1 << 31) - 16])
def test_quant_rows(parts, K):
    """Threads of the largest launch (256 to each 16 blocks of 128 columns at the most), and its blocks in 31 bits."""
    KB, rows = -(-K // 128), parts.t_quant_part(K)
    assert rows >= 1 and rows * KB < 1 << 31
    assert -(-rows * KB // 16) * 256 < 1 << 32


@pytest.mark.parametrize("threads", [64, 128, 256, 512, 1024])
def test_residual_norm(parts, threads):
    assert 1 <= parts.t_norm_part(threads) <= ((1 << 32) - 1) // threads


@pytest.mark.parametrize("N,K,code", [(1, (1 << 31) - 16, -5), ((1 << 31) - 1, 16, -5), ((1 << 31) - 256, 16, 0),
                                      (1 << 17, 1 << 21, -5), (1 << 17, (1 << 21) - 128, 0)])
def test_weight_quant(parts, N, K, code):
    """A workgroup of 256 threads per block: 2^24 blocks are one too many."""
    rc, msg = call(parts.t_wquant, v(P), 1, N, K, v(P), v(P))
    assert rc == code and (code == 0 or "anima_weight_quant_f8" in msg)


@pytest.mark.parametrize("M,N,code", [(1, 1 << 29, 0), (1, (1 << 29) + 1, -5), (1, (1 << 31) - 1, -5), (1 << 29, 1, 0),
                                      ((1 << 29) + 1, 1, -5), ((1 << 31) - 1, 1, -5)])
def test_products(parts, M, N, code):
    """Sides of a product: at 2^29 the largest tiles (256 x 256, gated 256 x 128, of 512 threads) fit a launch, and sizes
    rounded up to a tile fit 31 bits."""
    assert code != 0 or max(-(-M // 256) * -(-N // 128), -(-M // 128) * -(-N // 256)) * 512 < 1 << 32
    m = amd()
    W = weight(N=N, K=16)
    rc, msg = call(parts.t_linear, ctypes.byref(m.LinearDesc(M=M, W=ctypes.pointer(W), x=P, out=P)))
    assert rc == code and (code == 0 or "anima_linear" in msg)
    rc, msg = call(parts.t_glu, ctypes.byref(m.GluDesc(M=M, gate=ctypes.pointer(W), up=ctypes.pointer(W), x=P, out=P)))
    assert rc == code and (code == 0 or "anima_linear_glu" in msg)


# ------------------------------------------------------------------ on the GPU


class Large:
    """A buffer of rows of which only some are written and read: around the first ones, the cuts and the end."""

    def __init__(self, ctx, rows, cols, dtype, cuts):
        self.ctx, self.rows, self.cols, self.dtype = ctx, rows, cols, np.dtype(dtype)
        self.at = [(max(0, c - 8), min(rows, c + 8)) for c in sorted(cuts)]
        assert all(b <= a for (_, b), (a, _) in zip(self.at, self.at[1:]))
        self.buf = ctx.empty((rows * cols,), dtype)
        self.ptr = self.buf.ptr

    def _step(self, a):
        return self.ptr + a * self.cols * self.dtype.itemsize

    def write(self, values):
        for (a, _), x in zip(self.at, values):
            x = np.ascontiguousarray(x, self.dtype)
            self.ctx._check(amd().lib().anima_h2d(self.ctx.h, self._step(a), x.ctypes.data, x.nbytes))

    def read(self):
        out = []
        for a, b in self.at:
            x = np.empty((b - a, self.cols), self.dtype)
            self.ctx._check(amd().lib().anima_d2h(self.ctx.h, x.ctypes.data, self._step(a), x.nbytes))
            out.append(x)
        return out


@pytest.fixture
def ctx():
    c = amd().Context(0)
    yield c
    c.close()


@pytest.mark.gpu
def test_quant_rows_of_several_launches(ctx):
    """2^29 rows of 16 and more: 2^32 threads, were they one launch."""
    import test_f8_gpu as ref

    rows, K, part = (1 << 29) + 37, 16, 1 << 27
    cuts = [8] + [i * part for i in range(1, 5)] + [rows - 8]
    print(f"[case] quant_rows_f8 of {rows} rows", flush=True)
    rng = np.random.default_rng(4)
    x, q = Large(ctx, rows, K, np.uint16, cuts), Large(ctx, rows, K, np.uint8, cuts)
    s = Large(ctx, rows, 1, np.float32, cuts)
    want = [ref.bf16(rng.normal(size=(b - a, K)).astype(np.float32)) for a, b in x.at]
    x.write([bits for bits, _ in want])
    ctx.quant_rows_f8(x.ptr, rows, K, q.ptr, s.ptr, bf16=True)
    for (_, val), gq, gs in zip(want, q.read(), s.read()):
        wq, ws = ref.quant_ref(val)
        assert np.array_equal(gq, wq) and np.array_equal(gs[:, 0], ws[0])


@pytest.mark.gpu
def test_residual_norm_of_several_launches(ctx):
    """2^26 rows and more: 2^32 threads, were they one launch; gates by group of absolute rows."""
    import test_f8_gpu as ref

    rows, C, part, group = (1 << 26) + 37, 16, 1 << 25, (1 << 24) + 31
    cuts = [8, group, part, 2 * group, 3 * group, 2 * part, rows - 8]
    print(f"[case] residual_norm of {rows} rows", flush=True)
    rng = np.random.default_rng(5)
    x, y, h = (Large(ctx, rows, C, np.float32, cuts) for _ in range(3))
    q, s = Large(ctx, rows, C, np.uint8, cuts), Large(ctx, rows, 1, np.float32, cuts)
    gate = rng.normal(size=(4, C)).astype(np.float32)
    xs, ys = ([rng.normal(size=(b - a, C)).astype(np.float32) for a, b in x.at] for _ in range(2))
    x.write(xs)
    y.write(ys)
    ctx.residual_norm(rows, C, x.ptr, y=y.ptr, gate=ctx.upload(gate), group_rows=group, h=h.ptr, q=q.ptr, s=s.ptr)
    for (a, b), x0, y0, gx, gh, gq, gs in zip(x.at, xs, ys, x.read(), h.read(), q.read(), s.read()):
        g = gate[np.arange(a, b) // group].astype(np.float64)
        x1 = x0 + g * y0
        # (two roundings of the product and the sum)
        off = np.abs(gx - x1) / (np.abs(x0) + np.abs(g * y0))
        assert off.max() <= 2 * ref.U, (a, off.max() / ref.U)
        x1 = gx.astype(np.float64)
        h1 = x1 / np.sqrt((x1 * x1).mean(1, keepdims=True) + 1e-6)
        # (the sum of squares and eps 11 roundings at the most, which the root halves; root, quotient and product one each)
        off = np.abs(gh / h1 - 1).max()
        assert off <= 16 * ref.U, (a, off / ref.U)
        wq, ws = ref.quant_ref(gh)
        assert np.array_equal(gq, wq) and np.array_equal(gs[:, 0], ws[0])
