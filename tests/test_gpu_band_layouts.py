"""Banded attention on views whose rows overlap in memory, aligned for tile loads and not."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_band_attention import _compare, _tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_overlapping_rows(offset, d):
    q, _, _, table, dout = _tensors(1, 150, 150, 4, 2, d, 12)
    base = torch.randn(20000, device="cuda").to(torch.bfloat16).requires_grad_(True)
    # each row begins 64 elements behind the one before, the second head 32 behind the first
    k = base.as_strided((1, 150, 2, d), (16000, 64, 32, 1), offset)
    v = base.as_strided((1, 150, 2, d), (16000, 32, 16, 1), 4000 + offset)
    _compare(q, k, v, None, dout, window=60)
    _compare(q, k, v, table, dout, max_distance=40)
