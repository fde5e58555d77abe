"""Entries of the bias table that mask their bucket, in the unfused path and in the oracle's attention: hidden keys stay hidden."""
from __future__ import annotations

import math

import pytest
import torch

from nano_megatron_b200.parallel import unfused_banded_attention
from nano_megatron_b200.reference import ReferenceGPT, ReferenceGPTConfig

from ._band_oracle import oracle


@pytest.mark.parametrize("mask", [-math.inf, torch.finfo(torch.float64).min])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 0), (3, 1)])
def test_unfused_entry_point(mask, window, sinks):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 3, 7, 8, generator=g, dtype=torch.float64) for _ in range(3))
    table = torch.randn(3, 5, generator=g, dtype=torch.float64)
    table[0, 0] = table[1, 4] = mask   # the own position; all from some distance on
    table[2] = -math.inf               # a head that sees nothing
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    out = unfused_banded_attention(q, k, v, scale=0.3, window=window, sinks=sinks, table=table, max_distance=6)
    dout = torch.randn(out.shape, generator=g, dtype=torch.float64)
    grads = torch.autograd.grad(out, leaves, dout)
    values, _, _ = oracle(*(t.transpose(1, 2) for t in (q, k, v, dout)), 0.3, window=window, sinks=sinks, table=table, max_distance=6)
    torch.testing.assert_close(out.transpose(1, 2), values["out"], rtol=1e-10, atol=1e-12)
    for name, got in zip(("dq", "dk", "dv"), grads):
        torch.testing.assert_close(got.transpose(1, 2), values[name], rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(grads[3], values["dtable"], rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("mask", [-math.inf, torch.finfo(torch.float32).min])
def test_the_model_does_not_see_the_future(mask):
    torch.manual_seed(0)
    model = ReferenceGPT(ReferenceGPTConfig(vocab_size=32, max_seq_len=12, hidden_size=32, num_layers=2, num_heads=4,
                                            position_embedding_type="relative", relative_buckets=6, relative_max_distance=8))
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("rel_bias"):
                p[:, :2] = mask   # neither the own position nor the one before
    ids = torch.randint(0, 32, (1, 12))
    other = ids.clone()
    other[0, 6:] = (ids[0, 6:] + 1) % 32
    a, b = model(ids), model(other)
    assert a.isfinite().all() and torch.equal(a[:, :6], b[:, :6])
