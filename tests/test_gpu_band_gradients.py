"""Gradients of the banded attention where a row's D needs more digits than a bf16 output has."""
from __future__ import annotations

import math

import pytest
import torch

from tests._band_oracle import RMS, oracle
from tests.test_gpu_band_attention import _call, _tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sq,hq,hkv,d,window,buckets,max_distance,favoured", [
    (1000, 4, 4, 64, None, 8, 2048, None), (1000, 4, 4, 64, None, 8, 2048, 6), (1000, 4, 2, 128, None, 8, 2048, 5),
    (2000, 4, 4, 64, 900, 6, 2048, None), (2000, 2, 2, 128, 900, 6, 2048, 4),  # the window ends before the last bucket begins
    (1500, 8, 8, 64, None, 32, 128, 2), (1500, 4, 4, 96, 700, 32, 128, 20), (1300, 4, 4, 128, None, 2, 1000, 0)])
@pytest.mark.parametrize("seed", [0, 1])
def test_gradient_of_every_bucket(sq, hq, hkv, d, window, buckets, max_distance, favoured, seed):
    """Terms cancel in every bucket that has much of a row's weight, not in the last one only.  What is in the bf16 result
    besides its own rounding is no larger than that: sqrt(2) of it in all, since the two are independent."""
    q, k, v, table, dout = _tensors(1, sq, sq, hq, hkv, d, buckets, seed=seed)
    if favoured is not None:
        with torch.no_grad():
            table[:, favoured] = 6
    out = _call(q, k, v, table, d ** -0.5, max_distance, window=window)
    got = torch.autograd.grad(out, (q, k, v, table), dout)[3].double()
    want = oracle(q, k, v, dout, d ** -0.5, window=window, table=table, max_distance=max_distance)[0]["dtable"]
    rounding = (want.to(torch.bfloat16).double() - want).norm()
    assert (got - want).norm() <= math.sqrt(2) * rounding, f"{((got - want).norm() / rounding).item():.2f} times its rounding"


# sq, skv, start, window, sinks: few keys to a row, whichever way that comes about
@pytest.mark.parametrize("sq,skv,start,window,sinks", [
    (1000, 2, 0, 5000, 0), (1000, 2, 0, 5000, 1), (1000, 3, 0, 5000, 2), (700, 2, 300, 5000, 1), (700, 3, 4000, 100, 3),
    (900, 900, 0, 2, 0), (600, 1000, 1396, 999, 1), (700, 8, 300, 5000, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_rows_that_see_few_keys(sq, skv, start, window, sinks, d):
    """dS to bf16 and dQ, dK to bf16 are two independent roundings, and D must add nothing to speak of to them.  A rounding is off
    by U / sqrt(3) of the power of two below a value, root mean square; of the values themselves, spread evenly over the logarithm
    between two powers, that is sqrt(mean of 1 / m^2) = sqrt(3 / (8 ln 2)) = 0.736 of it.  (A tenth for the chance of a sample.)"""
    q, k, v, _, dout = _tensors(2, sq, skv, 4, 2, d)
    kw = dict(window=window, sinks=sinks)
    out = _call(q, k, v, None, d ** -0.5, 128, query_start=start, **kw)
    dq, dk = torch.autograd.grad(out, (q, k), dout)
    want = oracle(q, k, v, dout, d ** -0.5, start=start, **kw)[0]
    at = torch.arange(start, start + sq, device="cuda")
    j = torch.arange(skv, device="cuda")
    seen = ((j <= at[:, None]) & ((at[:, None] - j < window) | (j < sinks))).sum(1)
    few = ((seen >= 2) & (seen <= 8)).nonzero().flatten()  # a row that sees one key has no gradient
    off = [((dq.double() - want["dq"])[:, few].norm() / want["dq"][:, few].norm()).item()]
    if few.numel() >= sq - 1:
        off.append(((dk.double() - want["dk"]).norm() / want["dk"].norm()).item())
    assert few.numel() > 0 and max(off) <= 1.1 * math.sqrt(2 * 3 / (8 * math.log(2))) * RMS, [f"{x / RMS:.2f}" for x in off]
