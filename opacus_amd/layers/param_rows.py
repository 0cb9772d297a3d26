"""Parameters that enter a layer as one row per sample.

A layer whose backward kernel has the per-sample gradient of a parameter on the way (the sums over
a sample's positions that the input gradient needs, or that come with it) hands autograd the
parameter expanded to ``[n, *shape]``: the gradient that arrives at those rows IS the
per-sample gradient, and autograd's reduction of the expansion gives the ordinary one. The
grad-sample hooks listen to the rows instead of the layer's output (``per_sample_rows = True`` on
the module), so no sampler reads activations and backprops a second time.
"""

from __future__ import annotations

from typing import Sequence

import torch
import torch.nn as nn


def parameter_rows(module: nn.Module, params: Sequence[nn.Parameter], n: int) -> torch.Tensor:
    """``[n, *shape]`` (several parameters of one shape: ``[n, len(params), *shape]``) for the layer's
    autograd function to return per-sample gradients to. Where grad-sample hooks are installed on
    ``module`` they pick the tensor up right after this call of its forward."""
    stacked = params[0] if len(params) == 1 else torch.stack(list(params))
    rows = stacked.expand(n, *stacked.shape)
    if "_dpk_rows_hooked" in module.__dict__:
        module.__dict__["_dpk_param_rows"] = rows
    return rows


def forget_rows(module: nn.Module) -> None:
    """For a forward pass that raises after :func:`parameter_rows`: no hook picks its rows up, and a tensor
    that is left on the module keeps it from being copied."""
    module.__dict__.pop("_dpk_param_rows", None)


def rows_dim(module: nn.Module) -> int:
    """The dimension of ``module``'s input that the samples lie along: 0, or 1 where the grad-sample hooks
    of a model with ``batch_first=False`` are installed on a layer that follows the model's layout
    (``follows_layout = True``). The rows themselves are samples first in either case."""
    return module.__dict__.get("_dpk_rows_hooked", 0)


def first_derivative_only(what: str) -> None:
    """Called inside a backward pass, where grad mode is on only under ``create_graph=True``: the
    kernels' gradients are not differentiable, and a graph over them would silently lack terms."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"the {what} has no second derivative (create_graph=True is not supported)")
