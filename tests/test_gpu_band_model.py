"""Banded attention in the bf16 GPU model: against the fp32 oracle, and under the trainer's captured step."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_model import ctx  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu

KNOBS = {
    "window_packed": dict(attention_window=70, attention_sinks=3, use_fused_qkv=True, position_embedding_type="learned_absolute"),
    "window_rope_gqa": dict(attention_window=100, num_query_groups=2, use_fused_qkv=True),
    "relative": dict(position_embedding_type="relative", use_fused_qkv=True),
    "relative_window_separate": dict(position_embedding_type="relative", relative_buckets=16, relative_max_distance=60,
                                     attention_window=90, attention_sinks=2, num_query_groups=2, normalization="rmsnorm"),
}


def _pair(ctx, name, seed=0):
    from nano_megatron_b200.models import build_tp_gpt_from_reference
    from nano_megatron_b200.reference import ReferenceGPT, ReferenceGPTConfig, seed_all

    seed_all(seed)
    cfg = ReferenceGPTConfig(num_layers=2, hidden_size=256, num_heads=4, vocab_size=512, max_seq_len=256, **KNOBS[name])
    ref = ReferenceGPT(cfg)
    with torch.no_grad():
        for n, p in ref.named_parameters():
            if n.endswith("rel_bias"):
                p.normal_()
            elif p.dim() > 1:
                p.mul_(0.5)
    return cfg, ref, build_tp_gpt_from_reference(ref, ctx).to("cuda", dtype=torch.bfloat16)


@pytest.mark.parametrize("name", list(KNOBS))
def test_model_tracks_the_oracle(ctx, name):  # noqa: F811
    from nano_megatron_b200.ops import native
    from nano_megatron_b200.reference import shifted_cross_entropy

    cfg, ref, model = _pair(ctx, name)
    ids = torch.randint(0, cfg.vocab_size, (2, 256))
    before = native.lib().nmb_band_launches()
    logits = model(ids.cuda())
    loss = model.shifted_cross_entropy(logits, ids.cuda())
    loss.backward()
    torch.cuda.synchronize()
    native.check_status()
    assert native.lib().nmb_band_launches() >= before + 8  # two layers, forward and backward
    ref_logits = ref(ids)
    ref_loss = shifted_cross_entropy(ref_logits, ids)
    ref_loss.backward()
    # the bounds that the models with causal attention are held to
    assert (logits.float().cpu() - ref_logits).abs().max().item() < 4e-2 * ref_logits.abs().max().item()
    assert abs(loss.item() - ref_loss.item()) < 3e-2 * abs(ref_loss.item())
    want = dict(ref.named_parameters())
    for n, p in model.named_parameters():
        if want[n].grad is None:
            assert p.grad is None or not p.grad.any(), n
            continue
        rel = (p.grad.float().cpu() - want[n].grad).norm().item() / (want[n].grad.norm().item() + 1e-6)
        assert rel < 8e-2, (n, rel)


@pytest.mark.parametrize("name", ["window_packed", "relative_window_separate"])
def test_trainer_captures_the_step(ctx, name):  # noqa: F811
    """Eager steps, then a captured one: the same losses as forward, backward and update written out."""
    from nano_megatron_b200.engine import Trainer
    from nano_megatron_b200.ops import native
    from nano_megatron_b200.reference import AdamW

    cfg, _, model = _pair(ctx, name)
    _, _, twin = _pair(ctx, name)
    trainer = Trainer(model, ctx, lr=1e-3, weight_decay=0.01, bucket_cap_mb=0.5)
    opt = AdamW(twin.named_parameters(), lr=1e-3, weight_decay=0.01)
    gen = torch.Generator().manual_seed(7)
    for step in range(6):
        ids = torch.randint(0, cfg.vocab_size, (4, 256), generator=gen).cuda()
        got = trainer.step(ids).item()
        opt.zero_grad()
        loss = twin.shifted_cross_entropy(twin(ids), ids)
        loss.backward()
        opt.step()
        # the bound of the trainer's own test: the embedding's bf16 atomics differ from run to run
        assert abs(got - loss.item()) <= 1e-2 * abs(loss.item()), (step, got, loss.item())
    torch.cuda.synchronize()
    native.check_status()
    assert trainer.graphed, trainer.graph_error
    for (n, p), q in zip(model.named_parameters(), twin.parameters()):
        if n.endswith("rel_bias"):
            assert (p - q).float().norm() <= 2e-2 * q.float().norm(), n
    trainer.close()


def test_context_parallel_shards_make_up_the_whole(ctx):  # noqa: F811
    """The rows of four shards, each against all keys, are the rows of the whole call; their key gradients add up."""
    from nano_megatron_b200.ops.band_attention import relative_bias_attention

    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, dout = (torch.randn(2, 512, h, 64, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 2, 4))
    table = torch.randn(4, 32, generator=g, device="cuda").to(torch.bfloat16).requires_grad_(True)
    leaves = [t.requires_grad_(True) for t in (q, k, v)] + [table]
    kw = dict(window=300, sinks=5)
    whole = relative_bias_attention(q, k, v, table, 0.125, **kw)
    want = torch.autograd.grad(whole, leaves, dout)
    parts, grads = [], []
    for r in range(4):
        rows = slice(128 * r, 128 * (r + 1))
        part = relative_bias_attention(q[:, rows], k, v, table, 0.125, query_start=128 * r, **kw)
        grads.append(torch.autograd.grad(part, leaves, dout[:, rows]))
        parts.append(part)
    assert torch.equal(torch.cat(parts, dim=1), whole)          # the same tiles in the same order
    assert torch.equal(sum(t[0] for t in grads), want[0])        # each row's gradient comes from one shard
    for i in (1, 2, 3):
        total = sum(t[i].float() for t in grads)
        # four results rounded to bf16 and one: five roundings of at most eps / 2 of parts of about the whole's size
        assert (total - want[i].float()).norm() <= 5 * torch.finfo(torch.bfloat16).eps / 2 * want[i].float().norm()
