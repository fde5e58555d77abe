"""What a configuration accepts of windows and relative positions is what the operators accept."""
from __future__ import annotations

from dataclasses import asdict
from types import SimpleNamespace

import pytest
import torch

from nano_megatron_b200.models import build_tp_gpt_from_reference
from nano_megatron_b200.parallel import unfused_banded_attention
from nano_megatron_b200.reference import ReferenceGPT, ReferenceGPTConfig

from ._thread_ranks import run_ranks, thread_context


def _config(**knobs):
    return ReferenceGPTConfig(vocab_size=32, max_seq_len=8, hidden_size=32, num_layers=1, num_heads=4, **knobs)


@pytest.mark.parametrize("buckets,distance", [(32, 16), (33, 16), (200, 300), (129, 300), (32, 4096), (32, 2049), (1, 8), (0, 8)])
def test_refused_buckets(buckets, distance):
    with pytest.raises(ValueError):
        _config(position_embedding_type="relative", relative_buckets=buckets, relative_max_distance=distance)


@pytest.mark.parametrize("buckets,distance", [(32, 17), (33, 17), (128, 65), (128, 2048), (2, 2)])
def test_accepted_buckets_run(buckets, distance):
    model = ReferenceGPT(_config(position_embedding_type="relative", relative_buckets=buckets, relative_max_distance=distance))
    assert model(torch.zeros(1, 8, dtype=torch.long)).isfinite().all()


@pytest.mark.parametrize("knobs", [dict(attention_window=2.5), dict(attention_window=True), dict(attention_window=4, attention_sinks=1.0),
                                   dict(position_embedding_type="relative", relative_buckets=8.0),
                                   dict(position_embedding_type="relative", relative_max_distance=64.5)])
def test_numbers_that_are_not_whole(knobs):
    with pytest.raises(TypeError):
        _config(**knobs)


def test_unused_knobs_are_not_looked_at():
    assert _config(relative_buckets=1000).relative_buckets == 1000


@pytest.mark.parametrize("kw,error", [(dict(window=2.5), TypeError), (dict(window=0), ValueError), (dict(window=2, sinks=-1), ValueError),
                                      (dict(window=2, sinks=0.5), TypeError), (dict(table=torch.zeros(2, 1)), ValueError),
                                      (dict(table=torch.zeros(2, 8), max_distance=4), ValueError)])
def test_the_unfused_entry_point_refuses_the_same(kw, error):
    q = torch.zeros(1, 2, 4, 8)
    with pytest.raises(error):
        unfused_banded_attention(q, q, q, scale=1.0, **kw)


def test_a_configuration_without_these_fields():
    """The reference project's own object, which knows neither windows nor relative positions."""
    fields = {n: v for n, v in asdict(_config()).items() if not n.startswith(("attention_window", "attention_sinks", "relative_"))}
    torch.manual_seed(0)
    ref = ReferenceGPT(SimpleNamespace(**fields))
    ids = torch.randint(0, 32, (1, 8))

    def rank_fn(rank, be, model):
        return model(ids)

    got = run_ranks(1, rank_fn, lambda rank, be: build_tp_gpt_from_reference(ref, thread_context(rank, be, tp=1)))[0]
    torch.testing.assert_close(got, ref(ids), rtol=1e-5, atol=1e-5)
