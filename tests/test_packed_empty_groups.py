"""Packed groups without values: zeros, infinities and NaN alone."""
import pytest
import torch

from tempname_5090_b200.ops import actpack


def test_unit_of_a_group_without_values():
    """The smallest power of two holds a group whose values are zero, infinite or NaN."""
    for cols in (128, 200):
        x = torch.zeros(4, cols)
        x[1], x[2], x[3, :5] = torch.inf, torch.nan, -torch.inf
        p = actpack.pack(x)
        first = (cols + 15) // 16 * 16
        groups = (cols + 127) // 128
        assert bool((p.data[:, first:first + groups] == 1).all())  # 2^-126
        assert bool((p.data[:, first + groups:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packed_bytes_of_groups_without_values(dtype):
    """Zeros, infinities, NaN and the smallest numbers: the CPU statement's bytes."""
    for cols in (256, 301):
        x = torch.randn(8, cols, generator=torch.Generator().manual_seed(4)).to("cuda", dtype)
        x[0], x[1] = 0.0, -0.0
        x[2, :128] = torch.inf
        x[3] = torch.nan
        x[4] = torch.finfo(dtype).smallest_normal / 2
        x[5] = 2.0 ** -120
        x[6, :256] = 0.0
        x[7, 5] = -torch.inf
        assert torch.equal(actpack.pack(x).data.cpu(), actpack.pack(x.cpu()).data)
