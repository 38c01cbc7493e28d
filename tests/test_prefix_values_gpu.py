"""Attention behind a shared prefix with large finite values of v, in rows that see them: a result is a mean of values, so it is finite
where they are.  The sums before the division hold weights of up to 2^8: with n keys, values below 2^119 / n stay finite.

Tolerances: the values of v are test_prefix_gpu's times a power of two, which scales every result and its bound alike."""

import numpy as np
import pytest

from helpers import amd
from test_prefix_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with amd().Context(0) as c:
        yield c


def times(c, f):
    """The case with all its values of v times f."""
    H, Hkv = c.H, c.Hkv
    c.qkv[:, (H + Hkv) * 128: (H + 2 * Hkv) * 128] *= np.float32(f)
    c.pv = c.pv * np.float32(f)


def prepare(c):
    if c.P:
        up = [c.ctx.upload(np.ascontiguousarray(c.pk)), c.ctx.upload(np.ascontiguousarray(c.pv))]
        c.ctx.attention_prefix(k=up[0], v=up[1], lens=[c.P], H=c.H, group=c.H // c.Hkv, ldk=c.Hkv * 128, ldv=c.Hkv * 128, precision=c.precision,
                               prepare_into=c.prefix)


CASES = [([3, 1], 640, 2, 1), ([64] * 32, 640, 32, 32), ([200], 0, 2, 2), ([300, 90], 200, 2, 1), ([1], 5000, 2, 1)]


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P,H,Hkv", CASES)
@pytest.mark.parametrize("rise", [3, 30, 60, -30])
def test_large_values_where_scores_rise(ctx, lens, P, H, Hkv, precision, rise):
    """Scores that grow (or fall) by 2^rise times the weight every 64 keys, values of 2^100 (n is below 2^13): a row is finite and right."""
    c = Case(ctx, lens, P, H, Hkv, precision, normed=False, roped=False)
    sign = np.where(np.random.default_rng(1).random(128) < 0.5, -1.0, 1.0).astype(np.float32)

    def level(j):  # (q, k: powers of two, small whole numbers, signs, so that only the common factor rounds)
        return (j // 64).astype(np.float32)[:, None, None] * np.float32(0.5)

    c.pk = (level(np.arange(P)) * sign * np.ones((1, Hkv, 1))).astype(np.float32)
    at = 0
    c.qkv[:, : H * 128] = np.tile(sign, H)
    for n in lens:
        c.qkv[at: at + n, H * 128: (H + Hkv) * 128] = (level(P + np.arange(n)) * sign * np.ones((1, Hkv, 1))).reshape(n, -1)
        at += n
    c.scale = float(rise / 64 * np.log(2.0))  # a level is 128 * 0.5 * scale
    ref, _ = c.ref()
    v = max(np.abs(c.pv).max() if P else 0, np.abs(c.qkv[:, (H + Hkv) * 128:]).max())
    times(c, 2.0 ** 100)
    prepare(c)
    got = c.get().reshape(c.T, H, 128).astype(np.float64) * 2.0 ** -100
    assert np.isfinite(got).all()
    # Scores are whole levels times one factor, which is off by d = 2^-23 (bf16: q times it has 11 bits, 2^-12): the weight 2^-x of a key x
    # below the largest is off by x ln 2 d of itself, and the sum of x 2^-x ln 2 over the levels is below 1 from a rise of 3 on.  The sums of
    # a score are off by 40 2^-24 of the largest, a weight by twice that; in bf16 a weight and a value of v are rounded to 8 bits; the
    # rest are a row's sums, in steps of 16 keys, and parts.  Weights are off in the sum and in what it is divided by.
    top = abs(rise) * ((P + max(lens)) // 64) * np.log(2.0)
    tol = (2.0 ** -12 + 2 * 2.0 ** -8 if precision == 0 else 2.0 ** -23) + (80 * top + 32 + (P + max(lens)) / 16) * 2.0 ** -24
    assert np.abs(got - ref).max() <= 2 * tol * v


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P", [([9, 1, 40], 100), ([1], 2000), ([200] * 3, 1000), ([1] * 40, 0)])
def test_scaled_values(ctx, lens, P, precision):
    """Ordinary scores: values times 2^100 (or 2^-60) give the results times as much, bit for bit."""
    a = Case(ctx, lens, P, 4, 2, precision, normed=False, roped=False)
    good = a.get()
    for e in (100, -60):
        c = Case(ctx, lens, P, 4, 2, precision, normed=False, roped=False)
        times(c, 2.0 ** e)
        prepare(c)
        np.testing.assert_array_equal(c.get().astype(np.float64) * 2.0 ** -e, good)
