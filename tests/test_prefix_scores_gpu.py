"""Attention behind a shared prefix where every score of a row is a large negative number: the softmax knows differences alone."""

import numpy as np
import pytest

from helpers import amd
from test_prefix_gpu import Case
from test_prefix_values_gpu import prepare

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with amd().Context(0) as c:
        yield c


@pytest.mark.parametrize("lens,P", [([1], 0), ([3, 1], 640), ([200], 0), ([1], 5000), ([300, 90], 200)])
@pytest.mark.parametrize("power", [20, 52, 54])
def test_scores_far_below_zero(ctx, lens, P, power):
    """Every score -2^(2 power) times 1.44 * 11.3 (below -10^30 from 48 on), the same for all keys: a row is the mean of the values
    it sees, off by the roundings of its sums alone."""
    c = Case(ctx, lens, P, 2, 1, amd().PREC_FP32, normed=False, roped=False)
    f = np.float32(2.0 ** power)
    c.qkv[:, :256] = f
    c.qkv[:, 256:384] = -f
    c.pk = np.full_like(c.pk, -f)
    prepare(c)
    got = c.get().reshape(c.T, 2, 128)
    at = 0
    for n in lens:
        v = np.concatenate([c.pv[:, 0], c.qkv[at: at + n, 384:]]).astype(np.float64)
        want = np.cumsum(v, 0)[P:] / np.arange(P + 1, P + n + 1)[:, None]
        tol = (32 + (P + n) / 16) * 2.0 ** -24 * np.abs(v).max()
        for h in range(2):
            err = np.abs(got[at: at + n, h] - want)
            assert np.all(err <= tol), err.max() / tol
        at += n
