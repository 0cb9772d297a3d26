"""Samplers of the layers whose backward kernels leave per-sample parameter gradients.

For these (``per_sample_rows = True`` on the module) the hooks hand a sampler the gradient of the
parameters' per-sample rows (``layers/param_rows.py``) in the place of the output's, so what is
left to do is the factor that turns a mean-reduced loss's gradients into a sum-reduced one's
(opacus/grad_sample/grad_sample_module.py:402-406).
"""

from __future__ import annotations

from typing import Dict, List

import torch
import torch.nn as nn

from ..layers.gated_rnn import GatedScan
from ..layers.norm_act import GroupNormAct, HeadNormAct
from .grad_sample_module import fused_scale, owns_output
from .utils import register_grad_sampler


@register_grad_sampler(GatedScan)
@owns_output
@fused_scale
def compute_gated_scan_grad_sample(
    layer: GatedScan, activations: List[torch.Tensor], backprops: torch.Tensor, scale: float = 1.0
) -> Dict[nn.Parameter, torch.Tensor]:
    """``backprops`` ``[n, D]``: the per-sample gradient of ``decay``."""
    return {layer.decay: backprops * scale} if layer.decay.requires_grad else {}


@register_grad_sampler([GroupNormAct, HeadNormAct])
@owns_output
@fused_scale
def compute_norm_act_grad_sample(
    layer: nn.Module, activations: List[torch.Tensor], backprops: torch.Tensor, scale: float = 1.0
) -> Dict[nn.Parameter, torch.Tensor]:
    """``backprops`` ``[n, 2, C]``: the per-sample gradients of weight and bias."""
    return {p: backprops[:, k] * scale for k, p in enumerate((layer.weight, layer.bias)) if p.requires_grad}
