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


@pytest.mark.parametrize("nsplit", [1, 2, 9])
def test_rows_in_front_of_the_first_sequence_stay(nsplit):
    nq, nkv, hd, front, counts, behind = 4, 2, 64, 5, [7, 3], 2
    c = Cache([400, 90], nkv, hd)
    kv = c.fill()
    T = front + sum(counts) + behind
    q = bf16(np.random.default_rng(0).standard_normal((T, nq, hd)))
    table, cache = c.tensors
    out = torch.full((T, nq * hd), 9.0, device="cuda", dtype=torch.bfloat16)
    part = [torch.full((T * nq * nsplit * x,), 3.0, device="cuda") for x in (hd, 2)] if nsplit > 1 else [None, None]
    rows = torch.from_numpy(q).reshape(T, -1).bfloat16().cuda()
    K.attention_prefill_kv4(rows, nq * hd, out, step_of(counts, [0, 0])[2] + front, dev(c.slots), dev(c.lens), table, cache, 2, max(counts), nq, nkv,
                            hd, PAGE, None, 0.1, nsplit, *part)
    assert (out[:front] == 9).all() and (out[T - behind:] == 9).all()
    got, at = out.double().cpu().numpy().reshape(T, nq, hd), front
    for (k, v), n, length in zip(kv, counts, c.lens):
        want, size, most = P.attention(q[at:at + n].astype(np.float64), k, v, 0.1, length - n)
        assert (np.abs(got[at:at + n] - want) <= tolerance(want, size, most, hd, length)).all()
        at += n


@pytest.mark.parametrize("hd,nq", [(32, 4), (64, 8), (128, 4), (128, 16), (160, 3), (256, 12)])
@pytest.mark.parametrize("nsplit", [1, 2, 64])
def test_values_close_to_the_largest_number(hd, nq, nsplit):
    """One token weighs 2^7 times as much as each of the others and its value is 6 x 2^125: a product of the two, as they are, is beyond what a
    float holds, the result is not."""
    n = 5 * PAGE + 9
    c = Cache([n], 1, hd)
    k, v = np.zeros((n, 1, hd)), np.zeros((n, 1, hd))
    loud = n - 5
    k[loud], v[loud] = 1.0, 6 * 2.0 ** 125
    for p in range(n):
        c.put(0, p, k[p], v[p])
    scale = 7 * np.log(2) / hd
    q = np.ones((4, nq, hd))
    for got, first in ((decode(c, q[:1], None, scale, nsplit), n - 1), (prefill(c, q, [4], None, scale, nsplit), n - 4)):
        want, size, most = P.attention(q[:len(got)], P.held(k), P.held(v), scale, first)
        assert np.isfinite(got).all() and want.min() > 1e37
        assert (np.abs(got - want) <= tolerance(want, size, most, hd, n)).all()
