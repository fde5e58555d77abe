"""Banded attention at sizes where a CTA has two query tiles at a time and several items one after the other."""
from __future__ import annotations

import pytest
import torch

from tests._band_oracle import check, oracle
from tests.test_gpu_band_attention import _call, _compare, _tensors

pytestmark = pytest.mark.gpu


# b, s, hq, hkv, d, window, sinks, buckets: more than 148 query tiles times heads, so two tiles a CTA: two heads where a group is
# even, else neighbouring tiles, of which an odd number leaves the last alone; more than 296: a second item for a CTA
@pytest.mark.parametrize("b,s,hq,hkv,d,window,sinks,buckets", [
    (1, 1200, 16, 8, 64, 300, 4, 0), (1, 1200, 16, 4, 128, 500, 140, 0), (1, 1300, 16, 16, 96, 200, 0, 0), (1, 1400, 15, 5, 64, 333, 3, 0),
    (2, 1300, 16, 8, 64, 250, 3, 0), (2, 1300, 16, 2, 128, 1000, 1, 0), (3, 900, 16, 16, 128, 400, 2, 0), (3, 777, 15, 5, 96, 2000, 0, 0),
    (2, 1300, 16, 16, 64, None, 0, 32), (2, 1290, 16, 4, 128, None, 0, 20), (3, 900, 12, 4, 96, None, 0, 32), (1, 1400, 16, 8, 64, 260, 5, 16),
    (4, 700, 16, 16, 64, 130, 2, 32), (8, 300, 16, 8, 128, 90, 0, 12)])
def test_several_items_a_cta(b, s, hq, hkv, d, window, sinks, buckets):
    _compare(*_tensors(b, s, s, hq, hkv, d, buckets), window=window, sinks=sinks)


@pytest.mark.parametrize("b,s,hq,hkv,d,window,sinks,buckets", [
    (1, 1200, 16, 8, 64, 300, 4, 0), (3, 777, 15, 5, 96, 2000, 0, 0), (2, 1300, 16, 2, 128, 1000, 1, 0), (2, 1290, 16, 4, 64, None, 0, 20),
    (2, 1300, 15, 15, 128, None, 0, 32)])
def test_several_items_a_cta_without_gradients(b, s, hq, hkv, d, window, sinks, buckets):
    from nano_megatron_b200.ops import native

    q, k, v, table, dout = _tensors(b, s, s, hq, hkv, d, buckets)
    with torch.no_grad():
        out = _call(q, k, v, table, d ** -0.5, 128, window=window, sinks=sinks)
    torch.cuda.synchronize()
    native.check_status()
    values, bounds, rms = oracle(q, k, v, dout, d ** -0.5, window=window, sinks=sinks, table=table)
    check({"out": out}, values, bounds, rms)
