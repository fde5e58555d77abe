"""Banded attention on the CPU: the plain expression against the definition in 64 bits, buckets, refusals."""
from __future__ import annotations

import math

import pytest
import torch

from nano_megatron_b200.ops.band_attention import (relative_bias_attention, relative_bucket_limits,
                                                   relative_position_buckets, window_attention)
from tests._band_oracle import bucket, oracle


def _inputs(b, sq, skv, hq, hkv, d, buckets=0, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(b, s, h, d, generator=g, dtype=dtype) for s, h in ((sq, hq), (skv, hkv), (skv, hkv)))
    dout = torch.randn(b, sq, hq, d, generator=g, dtype=dtype)
    table = torch.randn(hq, buckets, generator=g, dtype=dtype) if buckets else None
    return [t if t is None else t.requires_grad_(True) for t in (q, k, v, table)] + [dout]


@pytest.mark.parametrize("buckets,distance", [(2, 2), (2, 128), (3, 2), (5, 9), (32, 128), (32, 17), (64, 2048), (128, 65), (128, 2048)])
def test_buckets_are_those_of_the_definition(buckets, distance):
    n = min(2 * distance, 2400)
    want = [bucket(i, buckets, distance) for i in range(n)]
    got = relative_position_buckets(torch.arange(n), buckets, distance)
    assert got.tolist() == want
    limits = relative_bucket_limits(buckets, distance)
    assert len(limits) == buckets - 1 and list(limits) == sorted(limits) and limits[-1] <= distance


def test_buckets_on_borders_of_the_logarithm():
    # 4 exact ones, then one border every factor of 4^(1/4): 8 = 4 * 4^(2/4) begins bucket 6, which a rounded logarithm may miss
    assert relative_bucket_limits(8, 16) == (1, 2, 3, 4, 6, 8, 12)


@pytest.mark.parametrize("sq,skv,window,sinks,start", [(7, 7, 3, 0, 0), (7, 7, 3, 2, 0), (1, 9, 4, 1, 8), (5, 9, 100, 0, 4),
                                                       (6, 4, 2, 0, 1), (6, 4, 2, 1, 3), (3, 4, 1, 0, 0), (4, 6, 2, 99, 2)])
@pytest.mark.parametrize("buckets", [0, 5])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (3, 1)])
def test_expression_and_its_gradients(sq, skv, window, sinks, start, buckets, hq, hkv):
    q, k, v, table, dout = _inputs(2, sq, skv, hq, hkv, 8, buckets)
    kw = dict(window=window, sinks=sinks, query_start=start)
    if table is None:
        out = window_attention(q, k, v, 0.3, **kw)
    else:
        out = relative_bias_attention(q, k, v, table, 0.3, max_distance=6, **kw)
    leaves = [t for t in (q, k, v, table) if t is not None]
    grads = torch.autograd.grad(out, leaves, dout)
    values, _, _ = oracle(q, k, v, dout, 0.3, window=window, sinks=sinks, start=start, table=table, max_distance=6)
    for name, t in zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)):
        torch.testing.assert_close(t, values[name], rtol=1e-10, atol=1e-12, msg=lambda m, n=name: f"{n}: {m}")


def test_expression_against_differences():
    q, k, v, table, _ = _inputs(1, 5, 6, 2, 1, 4, 4)
    assert torch.autograd.gradcheck(
        lambda q, k, v, t: relative_bias_attention(q, k, v, t, 0.5, max_distance=5, window=3, sinks=1, query_start=1), (q, k, v, table))
    assert torch.autograd.gradcheck(lambda q, k, v: window_attention(q, k, v, 0.5, window=2, query_start=4), (q, k, v))


def test_masked_buckets_and_rows_that_see_nothing():
    q, k, v, table, dout = _inputs(1, 6, 6, 2, 2, 4, 4)
    with torch.no_grad():
        table[0, 0] = -math.inf      # head 0 never sees the own position: its first row sees nothing
        table[1, 2] = torch.finfo(table.dtype).min
    out = relative_bias_attention(q, k, v, table, 0.5, max_distance=5)
    assert torch.isfinite(out).all() and (out[:, 0, 0] == 0).all() and (out[:, 0, 1] == v[:, 0, 1]).all()
    for g in torch.autograd.grad(out, (q, k, v, table), dout):
        assert torch.isfinite(g).all()


def test_a_window_as_long_as_the_sequence_is_causal_attention():
    from nano_megatron_b200.parallel.attention_backend import unfused_causal_attention

    q, k, v, _, _ = _inputs(2, 9, 9, 3, 3, 8)
    want = unfused_causal_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), scale=0.4).transpose(1, 2)
    torch.testing.assert_close(window_attention(q, k, v, 0.4, window=9), want, rtol=1e-12, atol=1e-12)


def test_empty_inputs():
    q, k, v, _, _ = _inputs(2, 0, 3, 2, 2, 8)
    assert window_attention(q, k, v, 1.0, window=2).shape == (2, 0, 2, 8)
    q, k, v, table, _ = _inputs(2, 3, 0, 2, 2, 8, 4)
    out = relative_bias_attention(q, k, v, table, 1.0)
    assert out.shape == (2, 3, 2, 8) and (out == 0).all()


def _good():
    q, k, v, table, _ = _inputs(1, 4, 4, 4, 2, 8, 4)
    return q, k, v, table


@pytest.mark.parametrize("change,error", [
    (dict(window=0), ValueError), (dict(window=-1), ValueError), (dict(window=2.0), TypeError), (dict(window=True), TypeError),
    (dict(window=None), TypeError), (dict(sinks=-1), ValueError), (dict(sinks=1.5), TypeError), (dict(query_start=-1), ValueError),
    (dict(query_start=2 ** 30), ValueError), (dict(window=2 ** 40), ValueError), (dict(sinks=2 ** 31), ValueError), (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError),
    (dict(scale=float("nan")), ValueError), (dict(scale=float("inf")), ValueError)])
def test_refused_numbers(change, error):
    q, k, v, _ = _good()
    kw = {"window": 2, "sinks": 0, "query_start": 0, **change}
    scale = kw.pop("scale", 1.0)
    with pytest.raises(error):
        window_attention(q, k, v, scale, **kw)


def test_refused_tensors():
    q, k, v, table = _good()
    for bad in ((q[0], k, v), (q, k, v[:, :3]), (q[..., :4], k, v), (q[:, :, :3], k, v), (q.float(), k, v), (q.long(), k.long(), v.long()),
                (q.expand(2, -1, -1, -1), k, v), (q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(ValueError):
            window_attention(*bad, 1.0, window=2)
    for bad in (table[:2], table[0], table[:, :1], torch.zeros(4, 129)):
        with pytest.raises(ValueError):
            relative_bias_attention(q, k, v, bad, 1.0)
    for distance in (2, 0, -1, 2049):
        with pytest.raises(ValueError):
            relative_bias_attention(q, k, v, table, 1.0, max_distance=distance)
    with pytest.raises(TypeError):
        relative_bias_attention(q, k, v, table, 1.0, max_distance=8.0)
