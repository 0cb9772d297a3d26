"""Group normalisation with an affine map and an activation, in one kernel each way.

``GroupNormAct`` is ``torch.nn.GroupNorm`` followed by an activation, for channels-last images;
``HeadNormAct`` normalises every head of every token on its own. Their backward pass leaves the
per-sample weight and bias gradients (reference: opacus/grad_sample/group_norm.py:26-47, a pass of
its own over activations and backprops) as a by-product of the input gradient.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from .. import _lib, kernels
from .param_rows import first_derivative_only, forget_rows, parameter_rows, rows_dim


class _NormActFn(torch.autograd.Function):
    """``x`` ``[n, *, C]``; ``rows`` ``[n, 2, C]`` stands for weight and bias per sample (None: no
    affine map) and only receives their gradient, the values come from ``weight`` and ``bias``."""

    @staticmethod
    def forward(ctx, x, rows, weight, bias, num_groups, eps, activation, per_position):
        x = x.contiguous()
        y, stats = kernels.group_norm_act(x, num_groups, weight, bias, eps, activation, per_position)
        ctx.save_for_backward(x, stats, weight, bias)
        ctx.settings = (num_groups, eps, activation, per_position)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        first_derivative_only("group norm with an activation")
        x, stats, weight, bias = ctx.saved_tensors
        num_groups, eps, activation, per_position = ctx.settings
        dx, dw, db = kernels.group_norm_act_backward(
            x, grad_y, stats, num_groups, weight, bias, eps, activation, per_position
        )
        rows = torch.stack((dw, db), dim=1).to(weight.dtype) if ctx.needs_input_grad[1] else None
        return (dx if ctx.needs_input_grad[0] else None), rows, None, None, None, None, None, None


class _NormAct(nn.Module):
    # the grad-sample hooks listen to the parameters' per-sample rows
    per_sample_rows = True
    per_position: bool

    def __init__(
        self,
        num_groups: int,
        num_channels: int,
        eps: float = 1e-5,
        affine: bool = True,
        activation: str = "silu",
        device=None,
        dtype=None,
    ) -> None:
        super().__init__()
        if num_groups < 1 or num_channels % num_groups != 0:
            raise ValueError("num_channels must be divisible by num_groups")
        if activation not in _lib.DPK_ACT:
            raise ValueError(f"activation must be one of {sorted(_lib.DPK_ACT)}, got {activation!r}")
        self.num_groups, self.num_channels, self.eps, self.affine = num_groups, num_channels, eps, affine
        self.activation = activation
        if affine:
            self.weight = nn.Parameter(torch.empty(num_channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.empty(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        if self.affine:
            nn.init.ones_(self.weight)
            nn.init.zeros_(self.bias)

    def extra_repr(self) -> str:
        return (
            f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, activation={self.activation}"
        )

    def _apply_to(self, x: Tensor) -> Tensor:
        """``x`` ``[n, *, C]``."""
        if x.shape[-1] != self.num_channels:
            raise ValueError(f"expected {self.num_channels} channels, got {x.shape[-1]}")
        wide = kernels.widen(x)  # float16 runs on the float32 kernels
        rows = None
        if self.affine and torch.is_grad_enabled() and (self.weight.requires_grad or self.bias.requires_grad):
            rows = parameter_rows(self, (self.weight, self.bias), x.shape[0])
        weight, bias = (None, None) if not self.affine else (kernels.widen(self.weight.detach()), kernels.widen(self.bias.detach()))
        try:
            y = _NormActFn.apply(wide, rows, weight, bias, self.num_groups, self.eps, self.activation, self.per_position)
        except BaseException:
            forget_rows(self)
            raise
        return y if y.dtype == x.dtype else y.to(x.dtype)


class GroupNormAct(_NormAct):
    """``activation(GroupNorm(x))`` of ``[n, C, *]`` tensors; the arguments of ``torch.nn.GroupNorm``
    plus ``activation`` (``none``, ``relu``, ``silu`` or ``gelu`` in its erf form). Works on
    channels-last memory and returns it: an image in ``torch.channels_last`` format is read as it
    is, any other layout is copied into it first."""

    per_position = False

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() < 2:
            raise ValueError(f"expected [n, C, *], got {tuple(x.shape)}")
        return self._apply_to(x.movedim(1, -1)).movedim(-1, 1)


class HeadNormAct(_NormAct):
    """``activation`` of the group norm of every position on its own: ``[n, *, C]`` with the channels
    last, ``num_groups`` heads of ``C / num_groups`` neighbouring channels, statistics over one head
    of one position. The norm of the heads of an attention or recurrence output; causal, since no
    position sees another. In a model wrapped with ``batch_first=False`` the samples lie along the
    second dimension, as they do for ``nn.LayerNorm`` there."""

    per_position = True
    follows_layout = True

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() < 2:
            raise ValueError(f"expected [n, *, C], got {tuple(x.shape)}")
        if rows_dim(self) == 0:
            return self._apply_to(x)
        if x.dim() < 3:
            raise ValueError(f"expected [T, n, *, C] in a model with batch_first=False, got {tuple(x.shape)}")
        return self._apply_to(x.transpose(0, 1)).transpose(0, 1)
