"""Columns of a 4-bit weight whose groups' scales lie many powers of two apart, where x is zero in the groups with the large
ones: what is left has the accuracy of the small ones.

Tolerances: test_q4_gpu's of a product, with 2^-11 S for x rounded to 11 bits (half a step of a value just above a power of two).  The tiles hold a column's scales, times a power of two that brings the largest to 2^11
or more, in f16: the 8 bits of a scale are whole down to 2^-17, 2^-28 of the largest, and a smaller one is off by half of f16's last place,
2^-25, which is 2^-36 of the largest."""

import numpy as np
import pytest

import test_q4_gpu as ref
from helpers import amd, ran

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with amd().Context(0) as c:
        yield c


@pytest.mark.parametrize("apart", [20, 24, 27, 30, 34])
@pytest.mark.parametrize("precision,M,N,K,g,name", [
    (1, 40, 100, 8192, 128, "gemm.q4.64"), (1, 1025, 4092, 288, 32, "gemm.q4.128"), (1, 2049, 4092, 1056, 32, "gemm.q4.256"),
    (0, 640, 1701, 4160, 64, "gemm.q4.64"), (0, 2050, 3901, 576, 64, "gemm.q4.128"), (0, 4100, 3901, 544, 32, "gemm.q4.256"),
    (0, 64, 1300, 1024, 64, "gemm.q4.few"), (1, 20, 2700, 8224, 32, "gemm.q4.few"), (1, 4, 300, 1024, 64, "gemv.q4")])
def test_small_scales_alone(ctx, precision, M, N, K, g, name, apart):
    rng = np.random.default_rng(apart + M)
    W = ref.Q4(ctx, rng, N, K, g, False)
    codes = np.stack([W.bufs[0].numpy() & 15, W.bufs[0].numpy() >> 4], 2).reshape(N, K)
    s = rng.integers(128, 256, (N, K // g)).astype(np.float32) / 128  # (any 8 bits)
    s[:, 1::2] *= np.float32(2.0 ** -apart)
    W.bufs[1].write(ref.bf16(s))
    w = ref.values(codes, s, None, g)
    x = rng.normal(0, 1, (M, K)).astype(np.float32)
    x.reshape(M, K // g, g)[:, 0::2] = 0
    dx, out = ctx.upload(x), ctx.empty((M, N))
    assert ran(ctx, lambda: ctx.linear(W.w, M, out, x=dx, precision=precision)) == {name}
    x64 = x.astype(np.float64)
    want = x64 @ w.T
    tol = ref.bound(x64, w, K, precision, False, want, want)
    tol = tol + (2.0 ** -12 * (np.abs(x64) @ np.abs(w).T) if precision == 0 else 0.0)
    if apart > 27 and name in ("gemm.q4.64", "gemm.q4.128", "gemm.q4.256"):
        tol = tol + 2.0 ** -36 * s.max(1) * (np.abs(x64) @ np.abs(codes.astype(np.float64) - 8).T)
    err = np.abs(out.numpy() - want)
    assert np.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("M,N,K,g,name", [(40, 100, 8192, 128, "gemm.q4.64"), (40, 100, 8192, 32, "gemm.q4.64"), (640, 1701, 4160, 32, "gemm.q4.128"), (1030, 3600, 8192, 32, "gemm.q4.128"),
                                          (64, 1300, 1024, 64, "gemm.q4.few"), (4, 300, 8192, 32, "gemv.q4")])
@pytest.mark.parametrize("power", [-60, -100, -120])
def test_middles_beside_tiny_scales(ctx, M, N, K, g, name, power):
    """Constant groups (a middle, no scale) beside one group of scales 2^power: sums of like signs as large as they can be stay finite.
    The middles' part is bf16 values and three bf16 terms of a group's sum of x (2^-24 of it), so its bound is the product's."""
    rng = np.random.default_rng(M + K)
    W = ref.Q4(ctx, rng, N, K, g, True)
    codes = np.stack([W.bufs[0].numpy() & 15, W.bufs[0].numpy() >> 4], 2).reshape(N, K)
    s = np.zeros((N, K // g), np.float32)
    s[:, 0] = 2.0 ** power
    z = np.full((N, K // g), 1.9375, np.float32)
    z[:, 0] = 0
    W.bufs[1].write(ref.bf16(s))
    W.bufs[2].write(ref.bf16(z))
    w = ref.values(codes, s, z, g)
    x = np.full((M, K), 1.9375, np.float32)
    dx, out = ctx.upload(x), ctx.empty((M, N))
    assert ran(ctx, lambda: ctx.linear(W.w, M, out, x=dx, precision=1)) == {name}
    want = x.astype(np.float64) @ w.T
    err = np.abs(out.numpy() - want)
    tol = ref.bound(x.astype(np.float64), w, K, 1, False, want, want)
    assert np.all(err <= tol), (err / tol).max()
