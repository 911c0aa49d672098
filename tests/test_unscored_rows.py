"""Rows that are not scored pass no gradient on, whatever their logits hold."""
import pytest
import torch

from tempname_5090_b200.ops import loss

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [40, 1003, 33792])
def test_unscored_rows_of_a_padded_batch(V, dtype, device):
    z = torch.randn(9, V, generator=torch.Generator().manual_seed(V)).to(dtype)
    z[1], z[3, V // 2], z[4, 0], z[5, V - 1] = torch.nan, torch.nan, torch.inf, -torch.inf
    z[7], z[8, 3] = -torch.inf, torch.nan
    t = torch.tensor([0, -100, 1, -1, -100, -100, V - 1, -1, 3])
    a = torch.linspace(-1, 2, 9)
    b = torch.tensor([0.5, 0.0, -1.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0])
    z, t, a, b = (x.to(device) for x in (z, t, a, b))
    scores, state = loss.token_logprobs(z, t)
    unscored = t < 0
    assert bool((scores.logprob[unscored] == 0).all())
    for up in (None, b):
        g = loss.token_logprobs_backward(z, t, state, a, up)
        assert bool((g[unscored] == 0).all())
        assert bool(g[8].isnan().all()) and bool(g[[0, 2, 6]].isfinite().all())
        assert bool((g[[0, 2, 6]] != 0).any(1).all())
    # the entropy of an unscored row still has its gradient, and a row with NaN none of its own
    g = loss.token_logprobs_backward(z, t, state, a, torch.ones(9, device=device))
    assert bool((g[5] != 0).any()) and bool(g[5].isfinite().all()) and bool(g[[1, 3, 4]].isnan().all())
