"""The bias table under the trainer's captured step: its gradient buffer after a replay, and what the steps make of it."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_band_model import _pair
from tests.test_gpu_model import ctx  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def _tables(model):
    return [p for n, p in model.named_parameters() if n.endswith("rel_bias")]


@pytest.mark.parametrize("name", ["relative", "relative_window_separate"])
def test_gradient_after_a_replay(ctx, name):  # noqa: F811
    """After every captured step the table's buffer holds the gradient of that step's tokens, as an eager backward pass of the
    same weights gives it: the same kernels on the same values, so that at most one rounding to bf16 lies between them."""
    from nano_megatron_b200.engine import Trainer

    cfg, _, model = _pair(ctx, name)
    _, _, twin = _pair(ctx, name)
    trainer = Trainer(model, ctx, lr=1e-3, weight_decay=0.01, bucket_cap_mb=0.5)
    gen = torch.Generator().manual_seed(7)
    seen = []
    for step in range(8):
        ids = torch.randint(0, cfg.vocab_size, (4, 256), generator=gen).cuda()
        with torch.no_grad():
            for p, q in zip(model.parameters(), twin.parameters()):
                q.copy_(p)
                q.grad = None
        twin.shifted_cross_entropy(twin(ids), ids).backward()
        trainer.step(ids)
        torch.cuda.synchronize()
        if not trainer.graphed:
            continue
        for p, q in zip(_tables(model), _tables(twin)):
            want = q.grad.float()
            assert want.norm() > 0
            assert ((p.main_grad.float() - want).abs() <= torch.finfo(torch.bfloat16).eps * want.abs()).all()
        seen.append(_tables(model)[0].main_grad.clone())
    assert len(seen) >= 3, trainer.graph_error
    assert all((a - b).norm() > 0.1 * a.norm() for a, b in zip(seen, seen[1:]))  # other tokens, another gradient
    trainer.close()


def test_the_table_moves_as_written_out(ctx):  # noqa: F811
    """From zero on, so that what a step adds is neither rounded away nor small beside the table."""
    from nano_megatron_b200.engine import Trainer
    from nano_megatron_b200.reference import AdamW

    cfg, _, model = _pair(ctx, "relative")
    _, _, twin = _pair(ctx, "relative")
    with torch.no_grad():
        for p in _tables(model) + _tables(twin):
            p.zero_()
    trainer = Trainer(model, ctx, lr=1e-2, weight_decay=0.0, bucket_cap_mb=0.5)
    opt = AdamW(twin.named_parameters(), lr=1e-2, weight_decay=0.0)
    gen = torch.Generator().manual_seed(7)
    for _ in range(8):
        ids = torch.randint(0, cfg.vocab_size, (4, 256), generator=gen).cuda()
        trainer.step(ids)
        opt.zero_grad()
        twin.shifted_cross_entropy(twin(ids), ids).backward()
        opt.step()
    assert trainer.graphed, trainer.graph_error
    for p, q in zip(_tables(model), _tables(twin)):
        # a first step of the optimizer is lr for every element, whatever its gradient's size
        assert q.float().norm() > 1e-2 * q.numel() ** 0.5
        # a table that is not trained is 1 away, one trained the other way 2; the twins' own runs drift apart by the embedding's
        # atomic sums, which an optimizer that divides by the gradient's size blows up where a gradient is near zero
        assert (p - q).float().norm() <= 0.5 * q.float().norm()
    trainer.close()
