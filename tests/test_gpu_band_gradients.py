"""Gradients of the banded attention where a row's D needs more digits than a bf16 output has."""
from __future__ import annotations

import math

import pytest
import torch

from tests._band_oracle import oracle
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
