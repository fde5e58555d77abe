"""Banded attention in the models: the oracle against the definition, the parallel GPT on simulated ranks against the oracle,
checkpoints, configuration, command line."""
from __future__ import annotations

import pytest
import torch

from nano_megatron_b200.distributed import DistributedDataParallel
from nano_megatron_b200.models import build_tp_gpt_from_reference
from nano_megatron_b200.parallel import flash_banded_attention, unfused_banded_attention
from nano_megatron_b200.reference import ReferenceGPT, ReferenceGPTConfig

from ._band_oracle import oracle
from ._thread_ranks import run_ranks, thread_context
from .test_distributed_gloo import _close, _model_cfg, _reference

KNOBS = {
    "window": dict(attention_window=5),
    "window_sinks_gqa": dict(attention_window=3, attention_sinks=2, num_query_groups=4, use_fused_qkv=True),
    "relative": dict(position_embedding_type="relative", relative_buckets=8, relative_max_distance=12),
    "relative_window": dict(position_embedding_type="relative", relative_buckets=6, relative_max_distance=7, attention_window=6,
                            attention_sinks=1, use_fused_qkv=True),
}


def _check_grads(model, ref, ctx, cfg):
    """Every gradient against this rank's slice of the oracle's."""
    from nano_megatron_b200.utils.checkpoint import shard_tensor

    want = dict(ref.named_parameters())
    for n, p in model.named_parameters():
        if p.grad is not None:
            _close(p.grad, shard_tensor(n, want[n].grad, cfg, ctx.tensor_parallel_rank, ctx.tensor_parallel_size), f"grad {n}")
        if n.endswith("rel_bias"):
            assert p.grad is not None and p.grad.abs().max() > 0


def _cfg(name):
    return _model_cfg(**KNOBS[name])


def _spread_bias(model):
    """Relative tables start at zero; give them something to do."""
    gen = torch.Generator().manual_seed(9)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("rel_bias"):
                p.copy_(torch.randn(p.shape, generator=gen))


def _run_reference(cfg, ids, labels=None):
    made = ReferenceGPT.__init__

    def init(self, config):
        made(self, config)
        _spread_bias(self)

    with pytest.MonkeyPatch.context() as m:
        m.setattr(ReferenceGPT, "__init__", init)
        return _reference(cfg, ids, labels) if labels is not None else _reference(cfg, ids)


@pytest.mark.parametrize("window,sinks,buckets,start", [(3, 0, 0, 0), (4, 2, 0, 3), (None, 0, 6, 0), (5, 1, 6, 2)])
def test_unfused_entry_point(window, sinks, buckets, start):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 3, n, 8, generator=g, dtype=torch.float64) for n in (6, 6 + start, 6 + start))
    table = torch.randn(3, buckets, generator=g, dtype=torch.float64) if buckets else None
    out = unfused_banded_attention(q, k, v, scale=0.3, window=window, sinks=sinks, table=table, max_distance=9, query_start=start)
    values, _, _ = oracle(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), torch.zeros(2, 6, 3, 8), 0.3, window=window, sinks=sinks,
                          start=start, table=table, max_distance=9)
    torch.testing.assert_close(out.transpose(1, 2), values["out"], rtol=1e-10, atol=1e-12)
    with pytest.raises(ValueError):
        unfused_banded_attention(q, k, v, scale=0.3, window=3, query_start=start + 1)
    with pytest.raises(ValueError):
        unfused_banded_attention(q, k[:, :1], v[:, :1], scale=0.3, window=3)
    with pytest.raises(RuntimeError):
        flash_banded_attention(q, k, v, scale=0.3, window=3)  # no GPU tensors


def test_a_wide_window_changes_nothing_and_a_narrow_one_does():
    ids = torch.randint(0, _model_cfg().vocab_size, (2, 16), generator=torch.Generator().manual_seed(1))
    torch.manual_seed(0)
    plain = ReferenceGPT(_model_cfg())
    for window, same in ((16, True), (15, False), (2, False)):
        torch.manual_seed(0)
        model = ReferenceGPT(_model_cfg(attention_window=window))
        off = (model(ids) - plain(ids)).abs().max()
        assert (off < 1e-6) if same else (off > 0)
        acts = model.forward_with_activations(ids)[1]["layers"][0]["attn"]
        assert acts["probs"].shape[-1] == 16 and (acts["probs"][0, 0, 15] > 0).sum() == min(window, 16)


@pytest.mark.parametrize("tp,sp,name", [(1, False, "relative_window"), (2, False, "window"), (4, True, "window_sinks_gqa"),
                                        (2, True, "relative"), (4, False, "relative_window")])
def test_tensor_parallel_gpt(tp, sp, name):
    cfg = _cfg(name)
    torch.manual_seed(1234)
    ids = torch.randint(0, cfg.vocab_size, (2, 16))
    ref, ref_logits, ref_loss = _run_reference(cfg, ids)

    def prepare(rank, be):
        ctx = thread_context(rank, be, tp=tp, sequence_parallel=sp)
        return ctx, build_tp_gpt_from_reference(ref, ctx)

    def rank_fn(rank, be, prepared):
        ctx, model = prepared
        logits = model(ids)
        loss = model.shifted_cross_entropy(logits, ids)
        loss.backward()
        _close(loss.detach(), ref_loss, "loss")
        _check_grads(model, ref, ctx, cfg)
        return logits.detach()

    _close(torch.cat(run_ranks(tp, rank_fn, prepare), dim=-1), ref_logits, "logits")


@pytest.mark.parametrize("tp,cp,name", [(1, 4, "window_sinks_gqa"), (1, 2, "relative"), (2, 2, "relative_window")])
def test_context_parallel_gpt(tp, cp, name):
    cfg = _cfg(name)
    torch.manual_seed(1234)
    ids = torch.randint(0, cfg.vocab_size, (2, 16))
    ref, ref_logits, ref_loss = _run_reference(cfg, ids, ids.clone())

    def prepare(rank, be):
        ctx = thread_context(rank, be, tp=tp, cp=cp)
        return ctx, build_tp_gpt_from_reference(ref, ctx)

    def rank_fn(rank, be, prepared):
        ctx, model = prepared
        ddp = DistributedDataParallel(model, ctx)
        logits = ddp(ids)
        loss = model.shifted_cross_entropy(logits, ids)
        loss.backward()
        ddp.finish_grad_sync()
        _check_grads(model, ref, ctx, cfg)
        return ctx.tensor_parallel_rank, ctx.context_parallel_rank, logits.detach(), loss.detach()

    results = run_ranks(tp * cp, rank_fn, prepare)
    rows = []
    for c in range(cp):
        parts = sorted((r for r in results if r[1] == c), key=lambda r: r[0])
        rows.append(torch.cat([p[2] for p in parts], dim=-1))
    _close(torch.cat(rows, dim=1), ref_logits, "logits")
    _close(torch.stack([r[3] for r in results if r[0] == 0]).mean(), ref_loss, "loss")


def test_relative_table_in_checkpoints():
    from nano_megatron_b200.utils.checkpoint import shard_tensor, unshard_tensor

    cfg = _cfg("relative")
    full = torch.randn(cfg.num_heads, cfg.relative_buckets)
    name = "blocks.0.attn.rel_bias"
    shards = [shard_tensor(name, full, cfg, r, 2) for r in range(2)]
    assert shards[0].shape[0] == cfg.num_heads // 2 and torch.equal(unshard_tensor(name, shards, cfg), full)


def test_pipeline_graphs_leave_the_table_to_autograd():
    from types import SimpleNamespace

    from nano_megatron_b200.engine.pipeline_trainer import PipelineTrainer

    cfg = _cfg("relative")

    def prepare(rank, be):
        return build_tp_gpt_from_reference(ReferenceGPT(cfg), thread_context(rank, be, tp=1))

    def rank_fn(rank, be, model):
        for p in model.parameters():
            p.main_grad = torch.zeros_like(p)
        trainer = SimpleNamespace(stage=model)
        assert not PipelineTrainer._parameters_write_directly(trainer)
        for block in model.blocks:
            block.attn.rel_bias = None
        assert PipelineTrainer._parameters_write_directly(trainer)

    run_ranks(1, rank_fn, prepare)


@pytest.mark.parametrize("bad", [dict(attention_window=0), dict(attention_sinks=2), dict(attention_window=4, attention_sinks=-1),
                                 dict(position_embedding_type="relative", relative_buckets=1),
                                 dict(position_embedding_type="relative", relative_buckets=32, relative_max_distance=15)])
def test_refused_configurations(bad):
    with pytest.raises(ValueError):
        ReferenceGPTConfig(num_heads=4, hidden_size=64, **bad)


def test_command_line(tmp_path, capsys):
    from nano_megatron_b200.cli import run_reference_gpt

    for extra in (["--window", "4", "--sinks", "1"], ["--relative-pos"]):
        assert run_reference_gpt.main(["--steps", "2", "--seq", "16", *extra]) == 0
    assert "step 1: loss" in capsys.readouterr().out


def test_parameter_count():
    from nano_megatron_b200.cli.verify_architecture import count_parameters, expected_parameter_count

    cfg = _cfg("relative")
    assert count_parameters(cfg) == expected_parameter_count(cfg)
