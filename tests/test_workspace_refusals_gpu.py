"""Workspaces that the row operators' gradients do not take."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape, std=1.0, to=BF16):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(to)


def ops():
    from tempname_5090_b200.ops import actpack, loss, norm
    return actpack, loss, norm


def test_refusals_of_workspaces():
    """A workspace that is large enough to be used has to be contiguous FP32 on the same device."""
    actpack, _, norm = ops()
    rows, H = 4, 64
    x, vec = randn(2, rows, H), randn(3, H)
    x_out, h, stats = norm.block_join_fwd(x, x, *[vec] * 5, 1e-5)
    p = actpack.pack(x_out)
    size = 4 * rows * H
    want = norm.block_join_bwd(h, None, x_out, x, stats, *[vec] * 4)
    fine = torch.empty(size, device="cuda")
    for spare in (fine, fine[:5], torch.empty(2 * size + 1, device="cuda")[1:]):  # too small: not used
        got = norm.block_join_bwd(h, None, x_out, x, stats, *[vec] * 4, workspace=spare)
        for a, b in zip(got[:2], want[:2]):
            # off the 16-byte boundary the row's sums have another order: two roundings to BF16, 2^-8 each
            assert (a.double() - b.double()).abs().max() <= 2.0 ** -7 * b.double().abs().max()
    for spare in (fine.double(), fine.cpu(), torch.empty(2 * size, device="cuda")[::2]):
        with pytest.raises(ValueError):
            norm.block_join_bwd(h, None, x_out, x, stats, *[vec] * 4, workspace=spare)
        with pytest.raises(ValueError):
            norm.layer_norm_bwd_packed(h, p, vec, stats[2], stats[3], workspace=spare)
