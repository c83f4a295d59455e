"""Normalisation and dropout for U-Net blocks, as functions with gradients and as modules.

They work on the library's activations: contiguous NHWC ``(B, H, W, pad_ch(channels))``, fp32 or bf16.  (A
channels-last torch tensor of 32, 48, 64, ... channels is one: ``t.permute(0, 2, 3, 1)``.)  Each call is one operator
of ``ops`` in forward and one in backward; between the two, x and the (B, groups) statistics are kept, and no mask."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops


def _grad(dy: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return dy.to(like.dtype).contiguous()


def _widened(d: torch.Tensor, width: int) -> torch.Tensor:
    """The gradient of a tensor wider than its channels: what lies behind them has none."""
    return d if d.shape[3] == width else torch.nn.functional.pad(d, (0, width - d.shape[3]))


def _counter(drop: Optional[ops.Drop]) -> Optional[torch.Tensor]:
    """What a drop reads on the device when a kernel runs.  Saved for backward: autograd then reports a counter that was
    changed between the two passes, whose masks would differ."""
    return drop.offset_dev if drop is not None else None


class _GroupNormActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, channels, groups, act, eps, drop):
        y, mean, rstd = ops.group_norm_act_fwd(x, channels, groups, weight, bias, act=act, eps=eps, drop=drop)
        ctx.save_for_backward(x, weight, bias, mean, rstd, _counter(drop))
        ctx.spec = channels, groups, act, drop
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd, _ = ctx.saved_tensors
        channels, groups, act, drop = ctx.spec
        dx, dweight, dbias = ops.group_norm_act_bwd(x, _grad(dy, x), mean, rstd, channels, groups, weight, bias, act=act, drop=drop,
                                                    want_dweight=ctx.needs_input_grad[1], want_dbias=ctx.needs_input_grad[2])
        return _widened(dx, x.shape[3]), dweight, dbias, None, None, None, None, None


class _DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, channels, drop):
        if _counter(drop) is not None:             # nothing else is saved: without one, backward may run as often as it likes
            ctx.save_for_backward(drop.offset_dev)
        ctx.spec, ctx.width = (channels, drop), x.shape[3]
        ctx.residual_width = residual.shape[3] if residual is not None else 0
        return ops.dropout_fwd(x, channels, drop, residual=residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        channels, drop = ctx.spec
        if _counter(drop) is not None:
            _ = ctx.saved_tensors                  # raises where the counter was changed
        dy = dy.contiguous()
        dx = _widened(ops.dropout_bwd(dy, channels, drop), ctx.width) if ctx.needs_input_grad[0] else None
        dr = None
        if ctx.needs_input_grad[1]:                # dy itself, but for padding channels, whose output is a constant
            dr = _widened(dy if dy.shape[3] == channels else ops.dropout_fwd(dy, channels, None), ctx.residual_width)
        return dx, dr, None, None


def group_norm_act(x, channels: int, groups: int, weight=None, bias=None, act: str = "none", eps: float = 1e-5,
                   drop: Optional[ops.Drop] = None) -> torch.Tensor:
    """``dropout(act(group_norm(x)))``, differentiable in x, weight and bias."""
    return _GroupNormActFunction.apply(x, weight, bias, channels, groups, act, eps, drop)


def dropout(x, channels: int, drop: Optional[ops.Drop], residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + dropout(x)``, differentiable in both; without a ``drop`` nothing is dropped."""
    return _DropoutFunction.apply(x, residual, channels, drop)


def fresh_drop(p: float, per_channel: bool = False, offset_dev: Optional[torch.Tensor] = None) -> ops.Drop:
    """A ``Drop`` seeded from torch's default CPU generator: ``torch.manual_seed`` makes it repeat, and a
    checkpointed forward pass, which restores that generator, drops the same units again."""
    return ops.Drop(p, int(torch.empty((), dtype=torch.int64).random_()), 0, offset_dev, per_channel)


class Dropout(nn.Module):
    """``residual + dropout(x)`` in training mode, ``residual + x`` in evaluation mode and where ``p`` is 0: by the same
    operator, so inputs may be wider than the channels in both, and differently wide.

    ``offset_dev``: a one-element int64 GPU tensor for steps captured into a graph, whose seed is fixed by the capture;
    the caller counts it up once per step, after the backward pass."""

    def __init__(self, channels: int, p: float = 0.5, per_channel: bool = False, offset_dev: Optional[torch.Tensor] = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout: p must be between 0 and 1, got {p}")
        self.channels, self.p, self.per_channel, self.offset_dev = int(channels), float(p), bool(per_channel), offset_dev

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.training and self.p > 0.0:
            return dropout(x, self.channels, fresh_drop(self.p, self.per_channel, self.offset_dev), residual)
        if residual is None and x.shape[-1] == ops.pad_ch(self.channels):
            return x
        if residual is not None and not x.is_cuda and x.shape == residual.shape:       # nothing is dropped, and there are no kernels
            return x + residual
        return dropout(x, self.channels, None, residual)

    def extra_repr(self) -> str:
        return f"{self.channels}, p={self.p}, per_channel={self.per_channel}"


class GroupNormAct(nn.Module):
    """Group norm, an activation ("none", "relu", "silu", "gelu") and, in training mode, dropout with probability
    ``p``, in one operator.  Parameters are those of ``nn.GroupNorm(groups, channels, eps)``."""

    def __init__(self, groups: int, channels: int, act: str = "relu", eps: float = 1e-5, p: float = 0.0,
                 per_channel: bool = False, affine: bool = True, offset_dev: Optional[torch.Tensor] = None):
        super().__init__()
        if groups < 1 or channels < 1 or channels % groups:
            raise ValueError(f"group_norm_act: {channels} channels do not split into {groups} groups")
        if act not in ops.ACTIVATIONS:
            raise ValueError(f"unknown activation {act!r} ({', '.join(ops.ACTIVATIONS)})")
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout: p must be between 0 and 1, got {p}")
        self.groups, self.channels, self.act, self.eps = int(groups), int(channels), act, float(eps)
        self.p, self.per_channel, self.offset_dev = float(p), bool(per_channel), offset_dev
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        drop = fresh_drop(self.p, self.per_channel, self.offset_dev) if self.training and self.p > 0.0 else None
        return group_norm_act(x, self.channels, self.groups, self.weight, self.bias, self.act, self.eps, drop)

    def extra_repr(self) -> str:
        return f"{self.groups}, {self.channels}, act={self.act}, eps={self.eps}, p={self.p}, per_channel={self.per_channel}"
