"""Scales that fp32, in which the kernels hold them, cannot: refused on every path, before a launch."""
from __future__ import annotations

import math

import pytest
import torch

from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention

SCALES = [1e-50, 2.0 ** -127, 2.0 ** 127, 1e39, 1e300, 0.0, -0.125, math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("scale", SCALES)
def test_refused(device, scale):
    q = torch.zeros(1, 4, 2, 64, device=device, dtype=torch.bfloat16)
    for _ in range(2):  # the first call on a device and a later one take different ways through the checks
        with pytest.raises(ValueError, match="scale"):
            window_attention(q, q, q, scale, window=2)
        with pytest.raises(ValueError, match="scale"):
            relative_bias_attention(q, q, q, torch.zeros(2, 8, device=device), scale)
        window_attention(q, q, q, 0.125, window=2)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("scale", [2.0 ** -126, 1e-30, 2.0 ** 100, 2.0 ** 126])
def test_extremes_that_are_held(device, scale):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 40, 2, 64, generator=g).to(torch.bfloat16) for _ in range(3))
    if scale > 1:  # scores that fit fp32 again
        q = (q.float() / scale * 0.125).to(torch.bfloat16)
    q, k, v = (t.to(device) for t in (q, k, v))
    out = window_attention(q, k, v, scale, window=30).double()
    distance = torch.arange(40, device=device)[:, None] - torch.arange(40, device=device)
    x = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * scale
    p = torch.softmax(x.masked_fill((distance < 0) | (distance >= 30), -math.inf), -1)
    want = torch.einsum("bhij,bjhd->bihd", p, v.double())
    # one rounding of each weight, one of the result
    bound = torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + 1.1 * torch.einsum("bhij,bjhd->bihd", p, v.double().abs()))
    assert ((out - want).abs() <= bound).all()
