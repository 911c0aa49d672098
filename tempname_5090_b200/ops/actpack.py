"""Activations kept in 8 bits between the forward and the backward pass.

`pack` keeps a [rows, cols] matrix as E4M3 codes with one power of two for each
group of 128 columns (the smallest 2^e with max|x| <= 448 * 2^e): 1.008 bytes a
value against BF16's 2, off by at most half a code's step (2^-4 relative, and
2^-10 of the group's power of two for values near zero).  Infinities and NaN become
NaN and do not count in their group's maximum; magnitudes above 240 * 2^120 become
that (the next code up is 2^128).  `unpack` gives the kept values
back, `unpack_gelu` those of an MLP's pre-activation together with their GeLU
(what the MLP's backward pass multiplies with), and
`norm.layer_norm_bwd_packed` / `norm.block_join_bwd` read packed rows directly.

CUDA tensors run the native sm_100a kernels on the current stream; CPU tensors a
torch statement of the same arithmetic.  This is for one GPU's own memory and
exact to the bit; the TACO codec (ops/taco.py) is the one for packets between
GPUs.
"""
from __future__ import annotations

import torch

from .._native import count_launch, lib

GROUP = 128
DTYPES = (torch.bfloat16, torch.float32)


def _align(n: int) -> int:
    return (n + 15) // 16 * 16


def row_bytes(cols: int) -> int:
    """Bytes of a packed row: codes, then exponent bytes, each padded to 16."""
    return _align(cols) + _align((cols + GROUP - 1) // GROUP)


class Packed8:
    """A [rows, cols] matrix in 8 bits: `data` is uint8 [rows, row_bytes(cols)], and
    `dtype` the type its values are given back in."""

    __slots__ = ("data", "cols", "dtype")

    def __init__(self, data: torch.Tensor, cols: int, dtype: torch.dtype = torch.bfloat16):
        if dtype not in DTYPES:
            raise ValueError("packed activations are BF16 or FP32")
        if data.dtype != torch.uint8 or data.dim() != 2 or data.shape[1] != row_bytes(cols) \
                or not data.is_contiguous():
            raise ValueError("packed data must be contiguous uint8 [rows, row_bytes(cols)]")
        if data.is_cuda and data.data_ptr() % 16:
            raise ValueError("packed data must start on a 16-byte boundary")
        self.data, self.cols, self.dtype = data, cols, dtype

    @classmethod
    def _of(cls, data, cols, dtype):
        """`pack`'s own result, which needs no checks."""
        p = cls.__new__(cls)
        p.data, p.cols, p.dtype = data, cols, dtype
        return p

    @property
    def shape(self):
        return torch.Size((self.data.shape[0], self.cols))

    @property
    def device(self):
        return self.data.device

    @property
    def is_cuda(self):
        return self.data.is_cuda

    def nbytes(self) -> int:
        return self.data.numel()


def pack(x: torch.Tensor) -> Packed8:
    """Keep x [rows, cols] (BF16 or FP32, any row stride) in 8 bits."""
    if x.is_cuda:
        try:
            data = lib().pack(x)
        except (RuntimeError, TypeError):
            _check_packable(x)
            raise
        count_launch()
        return Packed8._of(data, x.shape[1], x.dtype)
    _check_packable(x)
    return _pack_cpu(x)


def _check_packable(x):
    if x.dim() != 2 or x.dtype not in DTYPES:
        raise ValueError("pack takes a BF16 or FP32 matrix")
    if x.shape[1] == 0:
        raise ValueError("pack needs at least one column")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError("pack needs contiguous rows")


@torch.no_grad()
def _pack_cpu(x):
    rows, cols = x.shape
    if not rows:
        return Packed8(torch.empty((0, row_bytes(cols)), dtype=torch.uint8), cols, x.dtype)
    groups = torch.nn.functional.pad(x.float(), (0, -cols % GROUP)).view(rows, -1, GROUP)
    finite = torch.where(groups.isfinite(), groups.abs(), torch.zeros(()))
    fraction, exponent = torch.frexp(finite.amax(2))
    exponent = torch.where(fraction > 0.875, exponent - 8, exponent - 9).clamp(min=-126)
    exponent = torch.where(fraction > 0, exponent, -126)  # zero has no exponent of its own
    scaled = torch.ldexp(groups, -exponent[:, :, None])
    top = torch.where(exponent == 120, 240.0, 448.0)[:, :, None]
    scaled = torch.where(scaled.isfinite(), torch.minimum(scaled.abs(), top).copysign(scaled), torch.full((), float("nan")))
    codes = scaled.to(torch.float8_e4m3fn).view(torch.uint8).reshape(rows, groups.shape[1] * GROUP)
    data = torch.zeros((rows, row_bytes(cols)), dtype=torch.uint8)
    data[:, :cols] = codes[:, :cols]
    data[:, _align(cols):_align(cols) + exponent.shape[1]] = (exponent + 127).to(torch.uint8)
    return Packed8(data, cols, x.dtype)


def _values(p: Packed8) -> torch.Tensor:
    """FP32 values (CPU statement; exact)."""
    rows, cols = p.shape
    units = p.data[:, _align(cols):_align(cols) + (cols + GROUP - 1) // GROUP].to(torch.int32) - 127
    codes = p.data[:, :cols].contiguous().view(torch.float8_e4m3fn).float()
    return torch.ldexp(codes, units.repeat_interleave(GROUP, 1)[:, :cols])


def _check(p) -> None:
    if not isinstance(p, Packed8):
        raise ValueError("expected a Packed8")


def unpack(p: Packed8) -> torch.Tensor:
    """The kept values, [rows, cols] of p.dtype."""
    _check(p)
    if p.is_cuda:
        count_launch()
        return lib().unpack(p.data, p.cols, p.dtype == torch.float32, False)[0]
    return _values(p).to(p.dtype)


def unpack_gelu(p: Packed8):
    """(x, GeLU(x)) of the kept pre-activation x, both [rows, cols] of p.dtype."""
    _check(p)
    if p.is_cuda:
        count_launch()
        x, act = lib().unpack(p.data, p.cols, p.dtype == torch.float32, True)
        return x, act
    x = _values(p)
    return x.to(p.dtype), torch.nn.functional.gelu(x).to(p.dtype)
