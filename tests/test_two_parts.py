"""Caches of two parts at the ends of their range: scores that are far apart, precision by
the size of a call, positions at a window's and at a table's end."""

from __future__ import annotations

import pytest
import torch

from llms_amd import harness
from llms_amd import kernels as fk
from tests.test_seg import check, exact, new_shared, new_window, randn

DEV = "cuda"
gpu = pytest.mark.gpu


# ------------------------------------------------------------- scores far apart


def along(n, D, spikes):
    """Keys [n, 1, D]: 0 but for a first channel at some positions. With q = 32 there (heads of 128) a
    channel of x is a score of 4.0806 x in powers of two."""
    k = torch.zeros(n, 1, D, dtype=torch.bfloat16)
    for p, x in spikes.items():
        k[p, 0, 0] = x
    return k


def check_apart(y, e):
    """One rounding to bf16 (2^-8), p in one bf16 part in products and in their sum (2 x 2^-8 of the weighted |v|),
    and scores of up to 2^7 powers of two: the factor log2(e) / sqrt(D) is three roundings off (2^-24 each) and the
    exponent one, so an exponential is off by 2^7 x 4 x 2^-24 x ln 2 < 2^-15, in the products and in their sum."""
    want, size, _ = e
    err = (y.to(DEV).double() - want).abs()
    tol = want.abs() * 2.0**-8 + size * (2 * 2.0**-8 + 2 * 2.0**-15) + 1e-30
    assert y.isfinite().all() and (err <= tol).all(), float((err / tol).max())


def window_apart(n, T, spikes):
    """The last T of n tokens of one head attend over all of them."""
    g = torch.Generator().manual_seed(n + T)
    c, _ = new_window(n, 0, 1, 128, 1, max_step=n)
    k, v = along(n, 128, spikes), randn(g, n, 1, 128)
    for p in spikes:
        v[p] = v[p].sign() / 2
    q = torch.zeros(T, 1, 128).bfloat16()
    q[:, :, 0] = 32
    c.write(0, k[None].to(DEV), v[None].to(DEV), 0)
    y = fk.attention_window(q[None].to(DEV), k[None, n - T :].to(DEV), v[None, n - T :].to(DEV), c, 0, n - T)
    at = torch.arange(n)
    check_apart(y[0], exact(q, k, v, at[n - T :], at))


@gpu
@pytest.mark.parametrize("late", [30.75, 31.0, 31.125, 31.25, 31.5, 40.0, 61.0, 62.25, 62.5, 80.0])
@pytest.mark.parametrize("early", [0.5, 15.0, 30.75, 31.25])
def test_a_score_far_above_those_before(early, late):
    """Of 200 keys one at position 100 counts beside a later one in the tile that the last rows see in part: sums of
    up to 2^127 meet a reference that rises by as much, or by more than an exponential can say."""
    window_apart(200, 200, {100: early, 195: late})
