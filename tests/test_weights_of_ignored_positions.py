"""Weighted losses: what stands at ignored positions does not count."""
import math

import pytest
import torch

TINY = dict(layers=1, hidden=256, ffn=512, heads=2, sequence=256, micro_batch=1,
            accumulation_steps=1, vocab=512, chunk_rows=128)


@pytest.mark.parametrize("filler", [math.nan, math.inf, -math.inf])
def test_weights_of_ignored_positions_do_not_count(filler):
    from tempname_5090_b200.models.gpt import GPT
    from tempname_5090_b200.models.train import Trainer
    model = GPT(TINY, device="cpu", seed=7)
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 512, (256,), generator=g)
    targets = torch.randint(0, 512, (256,), generator=g)
    targets[::5] = -100
    weights = torch.rand(256, generator=g)
    want = model.forward_backward(tokens, targets, weights=weights, entropy_bonus=0.01)
    grad = model.store.grad.clone()
    spoilt = torch.where(targets < 0, torch.full((), filler), weights)
    got = model.forward_backward(tokens, targets, weights=spoilt, entropy_bonus=0.01)
    assert torch.equal(got, want) and bool(want.isfinite())
    assert torch.equal(model.store.grad, grad)
    loss, _ = Trainer(model).train_step([(tokens, targets, spoilt)])
    assert math.isfinite(loss)
