"""LayerNorm forward/backward, the joint of two blocks, GeLU backward and column sums.

CUDA tensors: native sm_100a kernels.  CPU tensors: the same math in torch
(test oracle path).  Semantics: F.layer_norm in FP32 on BF16 storage.

The joint (`block_join_fwd`) is what stands between two branches of a network
that normalises before and after each of them: the norm of the branch's output,
its gate, the scaled residual and the norm of the next branch's input, in one
pass.  Its gradient (`block_join_bwd`) and LayerNorm's (`layer_norm_bwd_packed`)
also read inputs kept in 8 bits (ops/actpack.py).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F

from .._native import count_launch, lib
from .actpack import Packed8, _values


def layer_norm_fwd(x, weight, bias, eps, out=None):
    """Returns (y, mean, rstd); y may be written into `out` (row-strided view allowed)."""
    rows, H = x.shape
    if x.is_cuda:
        y = torch.empty((rows, H), dtype=torch.bfloat16, device=x.device) if out is None else out
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        lib().layernorm_fwd(x, weight, bias, y, mean, rstd, float(eps))
        count_launch()
        return y, mean, rstd
    xf = x.float()
    mean = xf.mean(1)
    var = xf.var(1, unbiased=False)
    rstd = torch.rsqrt(var + eps)
    y = ((xf - mean[:, None]) * rstd[:, None] * weight.float() + bias.float()).to(x.dtype)
    if out is not None:
        out.copy_(y)
        y = out
    return y, mean, rstd


def layer_norm_bwd(dy, x, weight, mean, rstd, dres=None, workspace=None, out=None):
    """Returns (dx, dweight, dbias); dx = bf16(bf16(ln_dx) + dres) when dres is given,
    written into `out` (contiguous [rows, H]) when given."""
    rows, H = x.shape
    if x.is_cuda:
        dx = torch.empty_like(x) if out is None else out
        dw = torch.empty(H, dtype=torch.bfloat16, device=x.device)
        db = torch.empty(H, dtype=torch.bfloat16, device=x.device)
        need = lib().layernorm_bwd_workspace(rows, H)
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(need, dtype=torch.float32, device=x.device)
        lib().layernorm_bwd(dy.contiguous(), x.contiguous(), weight, mean, rstd, dx, dw, db, workspace, dres)
        count_launch(4)
        return dx, dw, db
    xf, g = x.float(), dy.float()
    xhat = (xf - mean[:, None]) * rstd[:, None]
    gw = g * weight.float()
    s1 = gw.mean(1, keepdim=True)
    s2 = (gw * xhat).mean(1, keepdim=True)
    dx = rstd[:, None] * (gw - s1 - xhat * s2)
    if dres is not None:
        dx = dx.to(torch.bfloat16).float() + dres.float()
    dx = dx.to(x.dtype)
    if out is not None:
        out.copy_(dx)
        dx = out
    return (dx, (g * xhat).sum(0).to(x.dtype), g.sum(0).to(x.dtype))


def gelu_bwd(dy, pre):
    if dy.is_cuda:
        dx = torch.empty_like(dy)
        lib().gelu_bwd(dy.contiguous(), pre.contiguous(), dx)
        count_launch()
        return dx
    z = pre.float()
    cdf = 0.5 * (1 + torch.erf(z * 0.7071067811865476))
    pdf = 0.3989422804014327 * torch.exp(-0.5 * z * z)
    return (dy.float() * (cdf + z * pdf)).to(dy.dtype)


def column_sum(g, out=None, workspace=None):
    """bf16 column sums of a [rows, cols] bf16 matrix (bias gradients), deterministic."""
    rows, cols = g.shape
    if g.is_cuda:
        out = torch.empty(cols, dtype=torch.bfloat16, device=g.device) if out is None else out
        parts = 64 if rows >= 4096 else (32 if rows >= 512 else 1)
        if workspace is None or workspace.numel() < parts * cols:
            workspace = torch.empty(parts * cols, dtype=torch.float32, device=g.device)
        lib().column_sum(g, out, workspace)
        count_launch(2)
        return out
    s = g.float().sum(0).to(g.dtype)
    if out is not None:
        out.copy_(s)
        return out
    return s


# ------------------------------------------------------------------ block joint
JOIN_DTYPES = (torch.bfloat16, torch.float32)
JOIN_MAX_COLS = 8192


class JoinGrads(NamedTuple):
    dx: torch.Tensor            # [rows, H], of the residual stream's input
    dy: torch.Tensor            # [rows, H], of the branch's output
    dpost_weight: torch.Tensor  # [H] each
    dpost_bias: torch.Tensor
    dgate: torch.Tensor
    dpre_weight: torch.Tensor
    dpre_bias: torch.Tensor
    h: torch.Tensor | None      # the next branch's input again, where it was asked for


def _check_matrix(name, t, like, shape, own_rows=False):
    if t.dtype != like.dtype or t.device != like.device or t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)} of {like.dtype} on {like.device}")
    if shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} needs contiguous rows")
    if own_rows and shape[0] > 1 and t.stride(0) < shape[1]:
        raise ValueError(f"{name} needs rows of its own")


def _check_vectors(like, cols, **vectors):
    for name, t in vectors.items():
        if t.dtype != like.dtype or t.device != like.device or t.shape != (cols,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous ({cols},) of {like.dtype} on {like.device}")


def _check_stats(like, shape, **stats):
    for name, t in stats.items():
        if t.dtype != torch.float32 or t.device != like.device or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous FP32 {tuple(shape)} on {like.device}")


def _check_workspace(like, workspace):
    if workspace is not None and (workspace.dtype != torch.float32 or workspace.device != like.device
                                  or not workspace.is_contiguous()):
        raise ValueError(f"workspace must be contiguous FP32 on {like.device}")


def _check_first(name, t):
    if t.dim() != 2 or t.dtype not in JOIN_DTYPES:
        raise ValueError(f"{name} must be a BF16 or FP32 matrix")
    if not 1 <= t.shape[1] <= JOIN_MAX_COLS:
        raise ValueError(f"the hidden size must be between 1 and {JOIN_MAX_COLS}")


def _check_kept(name, t, like, shape):
    if isinstance(t, Packed8):
        if t.shape != shape or t.device != like.device:
            raise ValueError(f"{name} must be the packed form of {tuple(shape)} on {like.device}")
    else:
        _check_matrix(name, t, like, shape)


def _check_kept_width(p, like):
    if p.cols != like.shape[-1]:
        raise ValueError(f"packed rows of {p.cols} columns where {like.shape[-1]} are needed")


def block_join_fwd(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, eps, residual_scale=1.0, out=None):
    """Returns (x_out, h, stats) for the residual stream x and a branch's output y, [rows, H]:

        x_out = residual_scale * x + gate * LayerNorm(y; post_weight, post_bias)
        h     = LayerNorm(x_out; pre_weight, pre_bias)

    gate and the norms' parameters are [H].  BF16 or FP32, H up to 8192, any row
    strides; h may be written into `out` (a row-strided view is allowed).  h is
    computed from x_out before its rounding to the storage type.  `stats` (FP32
    [4, rows]: mean and reciprocal deviation of y, then of x_out) is for the gradient.
    """
    if x.is_cuda:
        try:
            x_out, h, stats = lib().block_join_fwd(x, y, post_weight, post_bias, gate, pre_weight, pre_bias,
                                                   residual_scale, eps, out)
        except (RuntimeError, TypeError):
            _check_join_fwd(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, out)
            raise
        count_launch()
        return x_out, h, stats
    _check_join_fwd(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, out)
    return _join_fwd_cpu(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, eps, residual_scale, out)


def _check_join_fwd(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, out):
    _check_first("x", x)
    _check_matrix("x", x, x, x.shape)
    _check_matrix("y", y, x, x.shape)
    _check_vectors(x, x.shape[1], post_weight=post_weight, post_bias=post_bias, gate=gate, pre_weight=pre_weight,
                   pre_bias=pre_bias)
    if out is not None:
        _check_matrix("out", out, x, x.shape, own_rows=True)


@torch.no_grad()
def _join_fwd_cpu(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, eps, residual_scale, out):
    yhat, mean_y, rstd_y = _normed(y.float(), eps)
    u = residual_scale * x.float() + gate.float() * (yhat * post_weight.float() + post_bias.float())
    uhat, mean_u, rstd_u = _normed(u, eps)
    h = (uhat * pre_weight.float() + pre_bias.float()).to(x.dtype)
    if out is not None:
        out.copy_(h)
        h = out
    return u.to(x.dtype), h, torch.stack([mean_y, rstd_y, mean_u, rstd_u])


def _normed(v, eps):
    mean = v.mean(1)
    rstd = torch.rsqrt(v.var(1, unbiased=False) + eps)
    return (v - mean[:, None]) * rstd[:, None], mean, rstd


def _kept_float(t):
    return _values(t) if isinstance(t, Packed8) else t.float()


def _norm_input_grad(g, hat, rstd):
    return rstd[:, None] * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))


def block_join_bwd(dh, dx_out, x_out, y, stats, post_weight, post_bias, gate, pre_weight, residual_scale=1.0,
                   pre_bias=None, workspace=None, out=None) -> JoinGrads:
    """Gradients of `block_join_fwd` from that of h and (or None) of x_out.

    x_out and y are the forward's tensors, or both their packed 8-bit forms.  dy may
    be written into `out` (a row-strided view is allowed).  With `pre_bias` given, h is
    computed again from x_out and returned too.  `workspace` (FP32) is used where it
    is large enough.  Gradients of x_out and h join in FP32; parameter gradients are
    sums over the rows in a fixed order.
    """
    if dh.is_cuda:
        try:
            kept = isinstance(x_out, Packed8)
            if kept != isinstance(y, Packed8):
                raise ValueError("x_out and y are kept in the same form")
            if kept:  # rows of another width may take as many bytes
                _check_kept_width(x_out, dh)
                _check_kept_width(y, dh)
            elif x_out.dtype == torch.uint8:
                raise ValueError("packed rows are given as a Packed8")
            grads = lib().block_join_bwd(dh, dx_out, x_out.data if kept else x_out, y.data if kept else y, stats,
                                         post_weight, post_bias, gate, pre_weight, pre_bias, out, workspace,
                                         residual_scale)
        except (RuntimeError, TypeError):
            _check_join_bwd(dh, dx_out, x_out, y, stats, post_weight, post_bias, gate, pre_weight, pre_bias, out)
            _check_workspace(dh, workspace)
            raise
        count_launch(2)
        return JoinGrads(*grads)
    _check_join_bwd(dh, dx_out, x_out, y, stats, post_weight, post_bias, gate, pre_weight, pre_bias, out)
    return _join_bwd_cpu(dh, dx_out, x_out, y, stats, post_weight, post_bias, gate, pre_weight, residual_scale,
                         pre_bias, out)


def _check_join_bwd(dh, dx_out, x_out, y, stats, post_weight, post_bias, gate, pre_weight, pre_bias, out):
    _check_first("dh", dh)
    rows, H = dh.shape
    _check_matrix("dh", dh, dh, dh.shape)
    if dx_out is not None:
        _check_matrix("dx_out", dx_out, dh, dh.shape)
    if isinstance(x_out, Packed8) != isinstance(y, Packed8):
        raise ValueError("x_out and y are kept in the same form")
    _check_kept("x_out", x_out, dh, dh.shape)
    _check_kept("y", y, dh, dh.shape)
    _check_stats(dh, (4, rows), stats=stats)
    _check_vectors(dh, H, post_weight=post_weight, post_bias=post_bias, gate=gate, pre_weight=pre_weight)
    if pre_bias is not None:
        _check_vectors(dh, H, pre_bias=pre_bias)
    if out is not None:
        _check_matrix("out", out, dh, dh.shape, own_rows=True)


@torch.no_grad()
def _join_bwd_cpu(dh, dx_out, x_out, y, stats, post_weight, post_bias, gate, pre_weight, residual_scale, pre_bias, out):
    mean_y, rstd_y, mean_u, rstd_u = stats
    uhat = (_kept_float(x_out) - mean_u[:, None]) * rstd_u[:, None]
    yhat = (_kept_float(y) - mean_y[:, None]) * rstd_y[:, None]
    dhf, pw, g = dh.float(), post_weight.float(), gate.float()
    dt = _norm_input_grad(dhf * pre_weight.float(), uhat, rstd_u)
    if dx_out is not None:
        dt = dt + dx_out.float()
    dn = dt * g
    dy = _norm_input_grad(dn * pw, yhat, rstd_y).to(dh.dtype)
    if out is not None:
        out.copy_(dy)
        dy = out
    h = None if pre_bias is None else (uhat * pre_weight.float() + pre_bias.float()).to(dh.dtype)
    return JoinGrads((residual_scale * dt).to(dh.dtype), dy, (dn * yhat).sum(0).to(dh.dtype), dn.sum(0).to(dh.dtype),
                     (dt * (yhat * pw + post_bias.float())).sum(0).to(dh.dtype),
                     (dhf * uhat).sum(0).to(dh.dtype), dhf.sum(0).to(dh.dtype), h)


def layer_norm_bwd_packed(dy, x, weight, mean, rstd, dres=None, bias=None, workspace=None, out=None):
    """LayerNorm's gradient from its input kept in 8 bits (x: Packed8) and the
    statistics of the forward pass.  Returns (dx, dweight, dbias, y): dx includes
    dres when given (joined in FP32) and is written into `out` when given; y is the
    norm's output again when `bias` is given (the weight gradient of the product that
    follows reads it), else None.
    """
    if dy.is_cuda:
        if not isinstance(x, Packed8):
            raise ValueError("x must be a Packed8")
        try:
            _check_kept_width(x, dy)
            dx, dw, db, y = lib().layer_norm_bwd_packed(dy, dres, x.data, mean, rstd, weight, bias, out, workspace)
        except (RuntimeError, TypeError):
            _check_packed_norm(dy, x, weight, mean, rstd, dres, bias, out)
            _check_workspace(dy, workspace)
            raise
        count_launch(2)
        return dx, dw, db, y
    _check_packed_norm(dy, x, weight, mean, rstd, dres, bias, out)
    return _packed_norm_cpu(dy, x, weight, mean, rstd, dres, bias, out)


def _check_packed_norm(dy, x, weight, mean, rstd, dres, bias, out):
    _check_first("dy", dy)
    rows, H = dy.shape
    _check_matrix("dy", dy, dy, dy.shape)
    if not isinstance(x, Packed8):
        raise ValueError("x must be a Packed8")
    _check_kept("x", x, dy, dy.shape)
    _check_stats(dy, (rows,), mean=mean, rstd=rstd)
    _check_vectors(dy, H, weight=weight)
    if bias is not None:
        _check_vectors(dy, H, bias=bias)
    if dres is not None:
        _check_matrix("dres", dres, dy, dy.shape)
    if out is not None:
        _check_matrix("out", out, dy, dy.shape, own_rows=True)


@torch.no_grad()
def _packed_norm_cpu(dy, x, weight, mean, rstd, dres, bias, out):
    hat = (_values(x) - mean[:, None]) * rstd[:, None]
    g = dy.float()
    dx = _norm_input_grad(g * weight.float(), hat, rstd)
    if dres is not None:
        dx = dx + dres.float()
    dx = dx.to(dy.dtype)
    if out is not None:
        out.copy_(dx)
        dx = out
    y = None if bias is None else (hat * weight.float() + bias.float()).to(dy.dtype)
    return dx, (g * hat).sum(0).to(dy.dtype), g.sum(0).to(dy.dtype), y
