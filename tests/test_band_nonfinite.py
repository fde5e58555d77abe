"""Scores that are not finite in the plain expression of the banded attention: what the kernels are held to as well."""
from __future__ import annotations

import math

import pytest
import torch

from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention


def _inputs(dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(1, 9, 2, 8, generator=g, dtype=dtype) for _ in range(3)]


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_row_with_such_a_score_is_nan(value):
    q, k, v = _inputs()
    table = torch.zeros(2, 4)
    table[1, 3] = value  # distances of 4 and more: (n / 2)^2 >= 5 / 2
    out = relative_bias_attention(q, k, v, table, 0.3, max_distance=5)
    assert out[:, 4:, 1].isnan().all() and out[:, :4].isfinite().all() and out[:, :, 0].isfinite().all()
    q[:, 4, :, 0] = 3e38
    k[:, 3, :, 0] = 3e38
    q[:, :4, :, 0] = q[:, 5:, :, 0] = 0
    out = window_attention(q, k, v, 0.3, window=4)
    assert out[:, 4].isnan().all() and out.isnan().sum() == out[:, 4].numel()


def test_a_score_of_minus_infinity_is_a_weight_of_zero():
    q, k, v = _inputs()
    q[..., 0] = 0
    q[:, [0, 6], :, 0] = 3e38
    k[..., 0] = 0
    k[:, [0, 5], :, 0] = -3e38
    out = window_attention(q, k, v, 0.3, window=3)
    assert (out[:, 0] == 0).all() and out.isfinite().all()
    x = torch.einsum("bhd,bjhd->bhj", q[:, 6], k[:, [4, 6]]) * 0.3
    torch.testing.assert_close(out[:, 6], torch.einsum("bhj,bjhd->bhd", torch.softmax(x, -1), v[:, [4, 6]]), rtol=1e-5, atol=1e-5)
