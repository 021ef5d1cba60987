"""Attention over 4-bit pages in runs that are joined: what a row gets does not depend on how many runs its pages come in."""
import numpy as np
import pytest
import torch

import plain_kv4 as P
from braidinfer_amd import kernels as K
from test_kv4_gpu import PAGE, Cache, bf16, decode, dev, prefill, step_of, tolerance

pytestmark = pytest.mark.gpu


def far_below(n, hd, bad):
    """A sequence whose last page's keys outweigh all others by 2^200 and more: q k scale = 4 * 6 * hd * 0.5 there, 384 at hd 32, and 0
    elsewhere.  Token `bad`, among the others, has a NaN in the last 32 channels of its value."""
    c = Cache([n], 1, hd)
    rng = np.random.default_rng(hd)
    k, v = np.zeros((n, 1, hd)), bf16(rng.standard_normal((n, 1, hd)))
    k[(n - 1) // PAGE * PAGE:] = 6.0
    v[bad, 0, -1] = np.nan
    for p in range(n):
        c.put(0, p, k[p], v[p])
    return c, P.held(k), P.held(v)


def check(got, want, size, most, hd, n):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert (np.abs(got - want) <= tolerance(want, size, most, hd, n))[fine].all()


@pytest.mark.parametrize("hd,nq", [(32, 4), (64, 8), (128, 4), (96, 16), (160, 3), (256, 12)])
@pytest.mark.parametrize("nsplit", [1, 3, 64])
def test_nan_of_a_run_far_below_reaches_the_token(hd, nq, nsplit):
    n = 1290
    for bad in (3, 700):
        c, k, v = far_below(n, hd, bad)
        q = np.full((1, nq, hd), 4.0)
        want, size, most = P.attention(q, k, v, 0.5, n - 1)
        assert np.isnan(want[:, :, -32:]).all() and np.isfinite(want[:, :, :-32]).all()
        check(decode(c, q, None, 0.5, nsplit), want, size, most, hd, n)


@pytest.mark.parametrize("hd,nq", [(32, 4), (64, 8), (128, 4), (160, 3), (256, 2)])
@pytest.mark.parametrize("nsplit", [1, 3, 20])
def test_nan_of_a_run_far_below_reaches_the_rows(hd, nq, nsplit):
    n, count = 1290, 9                                          # all new tokens stand in the last page
    for bad in (3, 700):
        c, k, v = far_below(n, hd, bad)
        q = np.full((count, nq, hd), 4.0)
        want, size, most = P.attention(q, k, v, 0.5, n - count)
        assert np.isnan(want[:, :, -32:]).all() and np.isfinite(want[:, :, :-32]).all()
        check(prefill(c, q, [count], None, 0.5, nsplit), want, size, most, hd, n)
