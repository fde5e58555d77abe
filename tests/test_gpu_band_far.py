"""Banded attention far out: positions near the largest accepted, rows whose offsets pass 32 bits."""
from __future__ import annotations

import pytest
import torch

from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention
from tests.test_gpu_band_attention import _compare, _tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 30, 0), (2 ** 30 - 10, 0), (2 ** 30 - 200, 7), (5, 300)])
@pytest.mark.parametrize("d", [64, 128])
def test_positions_near_the_limit(window, sinks, d):
    _compare(*_tensors(1, 140, 300, 4, 2, d), window=window, sinks=sinks, start=2 ** 30 - 140)


@pytest.mark.parametrize("d", [64, 128])
def test_distances_near_the_limit(d):
    """All keys are in the last bucket then, whose entry is the same for all: the table changes nothing."""
    q, k, v, table, dout = _tensors(1, 140, 300, 4, 2, d, 12)
    start = 2 ** 30 - 140
    out = relative_bias_attention(q, k, v, table, 0.125, query_start=start)
    grads = torch.autograd.grad(out, (q, k, v, table), dout)
    plain = window_attention(q, k, v, 0.125, window=2 ** 30, query_start=start)
    want = torch.autograd.grad(plain, (q, k, v), dout)
    half = torch.finfo(torch.bfloat16).eps / 2
    # both are roundings of one value, with weights to 8 and to 16 digits
    assert ((out - plain).double().abs() <= 2 * half * plain.double().abs() + half * v.double().abs().max()).all()
    for a, b in zip(grads, want):
        assert (a.double() - b.double()).norm() <= 4 * half * b.double().norm()
    assert (grads[3][:, :11] == 0).all()  # nothing falls into the other buckets


def test_rows_whose_offsets_pass_32_bits():
    rows, step = 520, 2 ** 23  # 2^32 elements: 8 GB
    store = torch.empty(rows * step, device="cuda", dtype=torch.bfloat16)
    q, k, v, _, dout = (None if t is None else t.detach() for t in _tensors(1, rows, rows, 2, 1, 64))
    views = [store.as_strided((1, rows, h, 64), (rows * step, step, 64, 1), at) for h, at in ((2, 0), (1, 256), (1, 512), (2, 1024))]
    for view, t in zip(views, (q, k, v, dout)):
        view.copy_(t)
    leaves = [t.requires_grad_(True) for t in views[:3]]
    got = window_attention(*leaves, 0.125, window=300, sinks=3)
    grads = torch.autograd.grad(got, leaves, views[3])
    near = [t.requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*near, 0.125, window=300, sinks=3)
    assert torch.equal(got, out)
    for a, b in zip(grads, torch.autograd.grad(out, near, dout)):
        assert torch.equal(a, b)
