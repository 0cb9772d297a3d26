"""Hooks-based per-sample-gradient engine (mirror of opacus/grad_sample/grad_sample_module.py).

Forward hooks keep the detached inputs of every layer that owns trainable parameters;
full-backward hooks hand those inputs and the layer's output gradient to the layer's
registered sampler, which launches the HIP kernels, and file the result under
``p.grad_sample``.

Two passes of the reference over per-sample data are gone here:
  * the multiplication of the backprops by the batch size for a mean-reduced loss
    (grad_sample_module.py:402-406) is passed to the kernels as a scalar when the
    sampler accepts one (``fused_scale``);
  * the zero-filled ``[max_batch_len, ...]`` buffer and the copy into it
    (grad_sample_module.py:61-66) are skipped when the sampler's tensor already has that
    batch length and is the sampler's own fresh output (``owns_output``).
"""

from __future__ import annotations

import logging
import warnings
from functools import partial
from typing import Callable, Iterable, List, Optional, Tuple

import torch
import torch.nn as nn

from ..utils.module_utils import (
    has_trainable_params,
    requires_grad,
    trainable_modules,
    trainable_parameter_list,
    trainable_parameters,
)
from .. import kernels
from ..layers.param_rows import rows_dim
from ._common import tag_sumsq
from .lazy import LazyLinearGradSample, lazy_linear_grad_sample
from .functorch import ft_compute_per_sample_gradient, prepare_layer
from .gsm_base import AbstractGradSampleHooks, AbstractGradSampleModule

logger = logging.getLogger(__name__)
logger.disabled = True


def fused_scale(fn: Callable) -> Callable:
    """Marks a sampler that takes ``scale=`` and applies it to the backprops inside its kernels."""
    fn.accepts_scale = True
    return fn


def owns_output(fn: Callable) -> Callable:
    """Marks a sampler whose returned tensors are fresh allocations nobody else refers to."""
    fn.owns_output = True
    return fn


def _runs_on_kernels(fn: Callable) -> bool:
    """This package's own samplers, which work from activations and backprops alone; not the
    functorch fallback (it runs the layer, whose parameters keep their dtype) or a sampler a
    user registered (plain torch takes float16 as it is)."""
    mod = getattr(getattr(fn, "func", fn), "__module__", None) or ""
    return mod.startswith(__package__ + ".") and not mod.endswith(".functorch")


def call_sampler(fn: Callable, module: nn.Module, activations, backprops: torch.Tensor, scale: float):
    """Calls a grad or norm sampler, folding ``scale`` into it if it can take it.

    float16 backprops (the reference's low-precision tests cover them beside bfloat16,
    tests/mixed_precision_test.py:240-242) have no kernels of their own: they and the activations
    are widened to float32, which is exact, the sampler runs on the float32 kernels, and
    per-sample gradients come back as float16 with their float32 sums of squares still attached
    (per-sample norms stay float32, as for bfloat16)."""
    if backprops.dtype is torch.float16 and backprops.is_cuda and _runs_on_kernels(fn):
        wide = [kernels.widen(a) for a in activations]
        out = call_sampler(fn, module, wide, backprops.float(), scale)
        return {
            p: tag_sumsq(v.half(), getattr(v, "_dpk_sumsq", None)) if v.dtype is torch.float32 and v.dim() > 1 else v
            for p, v in out.items()
        }
    if getattr(fn, "accepts_scale", False):
        return fn(module, activations, backprops, scale=scale)
    if scale != 1.0:
        backprops = backprops * scale
    return fn(module, activations, backprops)


def create_or_accumulate_grad_sample(
    *, param: torch.Tensor, grad_sample: torch.Tensor, max_batch_len: int, adopt: bool = False
) -> None:
    """Starts or continues ``param._current_grad_sample`` for the backward pass in flight.

    A later result for the same parameter in the same pass (tied weights, recurrent steps)
    is added into the first ``len(grad_sample)`` rows (grad_sample_module.py:58-59). The
    first result is copied into a zero-filled ``[max_batch_len, ...]`` buffer (:61-66),
    unless ``adopt`` says the tensor may be kept as it is.
    """
    if not param.requires_grad:
        return
    if isinstance(grad_sample, LazyLinearGradSample):
        # kept as factors only as the pass's one full-batch result for this parameter
        if not hasattr(param, "_current_grad_sample") and grad_sample.shape[0] == max_batch_len:
            param._current_grad_sample = grad_sample
            return
        grad_sample = grad_sample.materialize()
        adopt = True  # the tensor was formed for this parameter alone
    if hasattr(param, "_current_grad_sample"):
        if isinstance(param._current_grad_sample, LazyLinearGradSample):
            param._current_grad_sample = param._current_grad_sample.materialize()
        param._current_grad_sample[: grad_sample.shape[0]] += grad_sample
    elif adopt and grad_sample.shape[0] == max_batch_len:
        param._current_grad_sample = grad_sample
    else:
        buf = torch.zeros(
            torch.Size([max_batch_len]) + grad_sample.shape[1:], device=grad_sample.device, dtype=grad_sample.dtype
        )
        buf[: grad_sample.shape[0]] = grad_sample
        param._current_grad_sample = buf


def promote_current_grad_sample(p: nn.Parameter) -> None:
    """Moves the finished pass's tensor to ``p.grad_sample``; a second pass makes it a list (:69-79)."""
    if not p.requires_grad:
        return
    if p.grad_sample is None:
        p.grad_sample = p._current_grad_sample
    elif isinstance(p.grad_sample, list):
        p.grad_sample.append(p._current_grad_sample)
    else:
        p.grad_sample = [p.grad_sample, p._current_grad_sample]
    del p._current_grad_sample


def _get_batch_size(*, module: nn.Module, batch_dim: int) -> int:
    """Largest batch length among the pending activations of ``module`` (:552-573)."""
    return max((acts[-1].shape[batch_dim] for acts in module.activations), default=0)


def _batch_first_view(t: torch.Tensor, batch_dim: int) -> torch.Tensor:
    return t.permute([batch_dim] + [d for d in range(t.dim()) if d != batch_dim])


class _GradTap(torch.autograd.Function):
    """Identity whose output takes part in autograd although its input does not: gives the
    output of a layer at the start of the graph, run with its parameters switched off, a
    gradient for the hook to read. Nothing flows further back."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, _anchor: torch.Tensor) -> torch.Tensor:
        # the same tensor, not a view of it, so that an in-place op may follow (ReLU(inplace=True))
        ctx.mark_dirty(x)
        return x

    @staticmethod
    def backward(ctx, _grad):
        return None, None


# The layer types that run with their parameters switched off during forward: the library's
# own samplers cover all their parameters, and they return one tensor, so that the output of
# such a layer at the start of the graph can be re-attached through _GradTap. (Subclasses
# included: RNNLinear.) Layers with a user-registered sampler keep autograd's gradients.
_ONE_TENSOR_OUT = (
    nn.Linear,
    nn.modules.conv._ConvNd,
    nn.Embedding,
    nn.EmbeddingBag,
    nn.GroupNorm,
    nn.LayerNorm,
    nn.RMSNorm,
    nn.modules.instancenorm._InstanceNorm,
)


class GradSampleHooks(AbstractGradSampleHooks):
    """Attaches per-sample-gradient hooks to a module without wrapping it.

    ``autograd_weight_grads=True`` (the default) is the reference's behaviour: ``backward()``
    leaves the non-private summed gradient in ``p.grad`` until ``DPOptimizer.step``
    overwrites it. With ``autograd_weight_grads=False`` (an option the reference does not
    have), while the hooks are enabled a torch.nn layer served by one of the library's
    samplers runs its forward with ``requires_grad`` off on its own parameters, so the
    backward pass forms the gradients with respect to activations only. The aggregate weight
    gradients autograd would otherwise compute (a second GEMM or weight-gradient convolution
    per layer) are never read on this path: ``DPOptimizer.step`` writes ``p.grad`` from the
    clipped per-sample gradients (optimizers/optimizer.py:477-504). Until then ``p.grad`` of
    such a layer stays as it was (``None`` after ``zero_grad``), which a caller that reads
    ``p.grad`` between ``backward()`` and ``step()`` must know; the switch also changes
    ``requires_grad`` inside forward, so it is not for models whose forward runs concurrently
    from several threads.

    ``lazy_linear_grad_sample=True`` (off by default; the reference has no such option) leaves
    ``weight.grad_sample`` of every ``nn.Linear`` served by the library's own sampler as a
    :class:`~opacus_amd.grad_sample.lazy.LazyLinearGradSample`: the layer's activations and
    backprops instead of the ``[n, out, in]`` tensor they define (grad_sample/linear.py:41-48).
    ``DPOptimizer`` takes the per-sample norms and the clipped sum from the factors; whoever else
    reads the attribute gets the tensor, formed at that moment. ``isinstance(p.grad_sample,
    torch.Tensor)`` is false for such a parameter until then."""

    GRAD_SAMPLERS = {}
    # ghost clipping needs autograd's weight gradients in its second pass
    CAN_SKIP_AUTOGRAD_WEIGHT_GRADS = True
    # what ``autograd_weight_grads=None`` means
    DEFAULT_AUTOGRAD_WEIGHT_GRADS = True

    def __init__(
        self,
        m: nn.Module,
        *,
        batch_first=True,
        loss_reduction="mean",
        strict: bool = True,
        force_functorch=False,
        autograd_weight_grads: Optional[bool] = None,
        lazy_linear_grad_sample: bool = False,
    ):
        super().__init__(m, batch_first=batch_first, loss_reduction=loss_reduction)
        self.lazy_linear_grad_sample = bool(lazy_linear_grad_sample)
        errors = self.validate(module=m, strict=strict)
        if errors and not strict:
            logger.info(f"Validation found the following errors: {errors}. Using non-strict mode, continuing")
        self.hooks_enabled = False
        self.grad_accumulation_allowed = True
        self.force_functorch = force_functorch
        if autograd_weight_grads is None:
            autograd_weight_grads = self.DEFAULT_AUTOGRAD_WEIGHT_GRADS
        self.autograd_weight_grads = bool(autograd_weight_grads) or not self.CAN_SKIP_AUTOGRAD_WEIGHT_GRADS
        self._tap_anchor = torch.zeros((), requires_grad=True)
        self.add_hooks(loss_reduction=loss_reduction, batch_first=batch_first, force_functorch=force_functorch)

    # ---- hook installation -----------------------------------------------------------
    def _get_module_type(self, module: nn.Module):
        return type(module)

    def iterate_submodules(self, module: nn.Module) -> Iterable[nn.Module]:
        """Modules that get hooks: every one with trainable parameters of its own. Below a
        module that has them but no registered sampler nothing is visited: the generic
        fallback differentiates that whole subtree (grad_sample_module.py:152-165)."""
        # a module that only lists its children's parameters under other names (DPLSTM and
        # its kind, grad_sample_module.py:202-204) gets no hook of its own
        own = has_trainable_params(module) and not getattr(module, "grad_sample_through_children", False)
        if own:
            yield module
            if self._get_module_type(module) not in self.GRAD_SAMPLERS:
                return
        for child in module.children():
            yield from self.iterate_submodules(child)

    def add_hooks(self, *, loss_reduction: str = "mean", batch_first: bool = True, force_functorch: bool = False) -> None:
        if hasattr(self._module, "autograd_grad_sample_hooks"):
            raise ValueError("Trying to add hooks twice to the same model")
        for module in self.iterate_submodules(self._module):
            if force_functorch or self._get_module_type(module) not in self.GRAD_SAMPLERS:
                for m in module.modules():
                    if getattr(m, "per_sample_rows", False):
                        raise NotImplementedError(
                            f"{type(m).__name__} has no functorch path: its per-sample gradients come from its own "
                            "backward kernel (grad_sample_mode='hooks' or 'ghost', outside layers without a sampler)"
                        )
        self._module.autograd_grad_sample_hooks = []
        self.autograd_grad_sample_hooks = self._module.autograd_grad_sample_hooks
        for module in self.iterate_submodules(self._module):
            if getattr(module, "per_sample_rows", False):
                follows = getattr(module, "follows_layout", False)
                module.__dict__["_dpk_rows_hooked"] = 0 if batch_first or not follows else 1
            if force_functorch or self._get_module_type(module) not in self.GRAD_SAMPLERS:
                prepare_layer(module, batch_first=batch_first)
            elif not self.autograd_weight_grads:
                # order matters: parameters are switched back on before the capturing hook looks
                self.autograd_grad_sample_hooks.append(
                    module.register_forward_pre_hook(self._params_off_for_forward, with_kwargs=True)
                )
                self.autograd_grad_sample_hooks.append(
                    module.register_forward_hook(self._params_back_on, always_call=True)
                )
            self.autograd_grad_sample_hooks.append(
                module.register_forward_hook(
                    partial(self._forward_hook, loss_reduction=loss_reduction, batch_first=batch_first)
                )
            )
        self.enable_hooks()

    def _params_off_for_forward(self, module: nn.Module, args, kwargs) -> None:
        if not self.hooks_enabled or not module.training or not torch.is_grad_enabled():
            return
        if not isinstance(module, _ONE_TENSOR_OUT):
            return
        params = [p for p in module._parameters.values() if p is not None and p.requires_grad]
        if not params:
            return
        at_start = not any(isinstance(t, torch.Tensor) and t.requires_grad for t in args) and not any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in kwargs.values()
        )
        for p in params:
            p.requires_grad_(False)
        # plain attributes go through the instance dict: nn.Module.__setattr__ is a visible
        # cost per layer and step for a small model
        module.__dict__["_dpk_params_off"] = (params, at_start)

    def _params_back_on(self, module: nn.Module, _args, _output) -> None:
        state = module.__dict__.pop("_dpk_params_off", None)
        if state is not None:
            for p in state[0]:
                p.requires_grad_(True)
            module.__dict__["_dpk_at_start"] = state[1]

    def _forward_hook(self, module: nn.Module, forward_input, forward_output, *, loss_reduction: str, batch_first: bool):
        """Captures the activations and arranges for ``capture_backprops_hook`` to run when the
        gradient of this call's output is known. The reference installs a full backward hook
        on the module for that (grad_sample_module.py:215-224); a hook on the output tensor
        delivers the same ``grad_output`` without wrapping the module's inputs and outputs in
        an extra autograd node per call, which is what a small launch-bound model pays for
        in every step, and it tolerates an in-place op on the output."""
        d = module.__dict__
        rows = d.pop("_dpk_param_rows", None)
        pending = len(d.get("activations", ()))
        self.capture_activations_hook(module, forward_input, forward_output)
        if len(d.get("activations", ())) == pending:
            return  # nothing captured: eval mode, no grad, hooks disabled, frozen module
        out = forward_output if isinstance(forward_output, torch.Tensor) else forward_output[0]
        if rows is not None:
            # the layer's own backward kernel leaves the per-sample gradients: they arrive as the
            # gradient of its parameters' rows (layers/param_rows.py), which the sampler gets as backprops
            out = rows
        tapped = d.pop("_dpk_at_start", False) and isinstance(forward_output, torch.Tensor)
        if tapped and not out.requires_grad:
            out = _GradTap.apply(out, self._tap_anchor)
        if not out.requires_grad:
            return

        def on_grad_output(grad: torch.Tensor) -> None:
            self.capture_backprops_hook(module, None, (grad,), loss_reduction=loss_reduction, batch_first=batch_first)

        out.register_hook(on_grad_output)
        if tapped:
            return out  # replaces the module's output

    def remove_hooks(self) -> None:
        self.disable_hooks()
        for p in self._module.parameters():
            if hasattr(p, "ddp_hooks"):
                while p.ddp_hooks:
                    p.ddp_hooks.pop().remove()
                delattr(p, "ddp_hooks")
        if hasattr(self, "autograd_grad_sample_hooks"):
            while self.autograd_grad_sample_hooks:
                self.autograd_grad_sample_hooks.pop().remove()
            delattr(self, "autograd_grad_sample_hooks")
            if hasattr(self._module, "autograd_grad_sample_hooks"):
                delattr(self._module, "autograd_grad_sample_hooks")
        for module in self._module.modules():
            module.__dict__.pop("_dpk_rows_hooked", None)
            module.__dict__.pop("_dpk_param_rows", None)
        for _, module in trainable_modules(self._module):
            if hasattr(module, "ft_compute_sample_grad"):
                delattr(module, "ft_compute_sample_grad")

    def disable_hooks(self) -> None:
        """Hooks stay installed (autograd keeps those of a built graph anyway) but do nothing."""
        self.hooks_enabled = False

    def enable_hooks(self) -> None:
        self.hooks_enabled = True

    # ---- the hooks ----------------------------------------------------------------------
    def capture_activations_hook(self, module: nn.Module, forward_input: List[torch.Tensor], _forward_output):
        if not self.hooks_enabled or not module.training or not torch.is_grad_enabled():
            return
        if not requires_grad(module):
            return
        params = trainable_parameter_list(module)
        acts = module.__dict__.get("activations")
        if acts is None:
            acts = module.__dict__["activations"] = []
        # non-tensor inputs (an omitted optional argument passed as None) are not activations
        acts.append([t.detach() for t in forward_input if isinstance(t, torch.Tensor)])
        for p in params:
            p._forward_counter += 1

    def _sampler_for(self, module: nn.Module) -> Callable:
        if not self.force_functorch and self._get_module_type(module) in self.GRAD_SAMPLERS:
            return self.GRAD_SAMPLERS[self._get_module_type(module)]
        return ft_compute_per_sample_gradient

    def capture_backprops_hook(
        self, module: nn.Module, _forward_input, forward_output, loss_reduction: str, batch_first: bool
    ):
        """Per-sample gradients of ``module`` from its stored input and its output gradient.

        Results of one backward pass accumulate in ``p._current_grad_sample``; when the
        parameter's forward counter is back at zero the pass is over for it and the tensor
        moves to ``p.grad_sample`` (grad_sample_module.py:291-365).
        """
        if not self.hooks_enabled:
            return
        backprops = forward_output[0].detach()
        activations, backprops, scale = self._take_activations(
            module=module, backprops=backprops, loss_reduction=loss_reduction, batch_first=batch_first
        )
        sampler = self._sampler_for(module)
        if getattr(module, "stack_uses", False):
            stacked = self._stack_uses(module, activations, backprops)
            if stacked is None:
                return  # earlier uses of this pass are still to come
            activations, backprops = stacked
            for p in trainable_parameter_list(module):
                p._forward_counter += 1  # taken off again below, as for a module used once
        if self._keeps_factors(module, sampler, backprops):
            grad_samples = lazy_linear_grad_sample(module, activations, backprops, scale)
        else:
            grad_samples = call_sampler(sampler, module, activations, backprops, scale)
        adopt = getattr(sampler, "owns_output", False)
        for param, gs in grad_samples.items():
            create_or_accumulate_grad_sample(
                param=param, grad_sample=gs, max_batch_len=module.max_batch_len, adopt=adopt
            )
        for p in trainable_parameter_list(module):
            p._forward_counter -= 1
            if p._forward_counter == 0:
                promote_current_grad_sample(p)
            if not self.grad_accumulation_allowed:
                if isinstance(p.grad_sample, list) and len(p.grad_sample) > 1:
                    raise ValueError(
                        "Poisson sampling is not compatible with grad accumulation. "
                        "You need to call optimizer.step() after every forward/backward pass "
                        "or consider using BatchMemoryManager"
                    )
        if len(module.activations) == 0:
            module.__dict__.pop("max_batch_len", None)

    def _keeps_factors(self, module: nn.Module, sampler: Callable, backprops: torch.Tensor) -> bool:
        """Whether this use of ``module`` is filed as activations and backprops
        (``lazy_linear_grad_sample``): an ``nn.Linear`` itself, served by the library's sampler
        (a sampler the user registered for it must run), in a dtype the kernels contract."""
        return (
            getattr(self, "lazy_linear_grad_sample", False)
            and type(module) is nn.Linear
            and not self.force_functorch
            and _runs_on_kernels(sampler)
            and backprops.is_cuda
            and kernels.native_dtype(backprops.dtype)
            and backprops.shape[0] > 0
        )

    def _stack_uses(self, module: nn.Module, activations: List[torch.Tensor], backprops: torch.Tensor):
        """For a module applied many times per forward pass (``stack_uses``, the RNNLinear
        of the recurrent layers): keeps this use's activations and backprops and takes the use
        off the parameters' forward counters. Once the counters are back at zero, returns
        every use of the pass stacked along a new dimension 1, so that the sampler sums over
        the uses inside one contraction instead of the hooks adding one full per-sample
        gradient per use in memory (what grad_sample_module.py:43-66 does for such layers).
        Uses that saw fewer samples than ``max_batch_len`` are padded with zero rows."""
        pending = module.__dict__.setdefault("_pending_uses", [])
        pending.append((activations, backprops))
        done = True
        for _, p in trainable_parameters(module):
            p._forward_counter -= 1
            done = done and p._forward_counter == 0
        if not done:
            return None
        module.__dict__.pop("_pending_uses")
        if len(pending) == 1:
            return pending[0]
        n = module.max_batch_len

        def rows(t: torch.Tensor) -> torch.Tensor:
            if t.shape[0] == n:
                return t
            return torch.cat([t, t.new_zeros((n - t.shape[0],) + tuple(t.shape[1:]))], dim=0)

        acts = [torch.stack([rows(u[0][i]) for u in pending], dim=1) for i in range(len(pending[0][0]))]
        return acts, torch.stack([rows(u[1]) for u in pending], dim=1)

    def _take_activations(
        self, *, module: nn.Module, backprops: torch.Tensor, loss_reduction: str, batch_first: bool
    ) -> Tuple[List[torch.Tensor], torch.Tensor, float]:
        """Pops the matching activations and returns them batch-first with the backprops
        (not yet scaled) and the factor that turns them into sum-loss backprops."""
        if not hasattr(module, "activations"):
            raise ValueError(f"No activations detected for {type(module)}, run forward after add_hooks(model)")
        # the recurrent layers feed their RNNLinear batch first whatever the model's layout
        # (grad_sample_module.py:391)
        rows = getattr(module, "per_sample_rows", False)
        batch_dim = 0 if batch_first or getattr(module, "stack_uses", False) else 1
        if rows:
            batch_dim = rows_dim(module)
        if "max_batch_len" not in module.__dict__:
            module.__dict__["max_batch_len"] = _get_batch_size(module=module, batch_dim=batch_dim)
        activations = module.activations.pop()
        if loss_reduction == "mean":
            scale = float(module.max_batch_len)
        elif loss_reduction == "sum":
            scale = 1.0
        else:
            raise ValueError(f"loss_reduction = {loss_reduction}. Only 'sum' and 'mean' losses are supported")
        if batch_dim != 0 and not rows:  # (the parameters' rows are samples first)
            activations = [_batch_first_view(t, batch_dim) for t in activations]
            backprops = _batch_first_view(backprops, batch_dim)
        return activations, backprops, scale

    def rearrange_grad_samples(
        self, *, module: nn.Module, backprops: torch.Tensor, loss_reduction: str, batch_first: bool
    ) -> Tuple[List[torch.Tensor], torch.Tensor]:
        """Activations and backprops as a plain sampler expects them: batch first, backprops
        multiplied by the batch size for a mean loss (grad_sample_module.py:367-422)."""
        activations, backprops, scale = self._take_activations(
            module=module, backprops=backprops, loss_reduction=loss_reduction, batch_first=batch_first
        )
        if scale != 1.0:
            backprops = backprops * scale
        return activations, backprops

    # ---- validation ----------------------------------------------------------------------
    @classmethod
    def is_supported(cls, module: nn.Module) -> bool:
        warnings.warn(
            "GradSampleModule.is_supported is deprecated, as all layers can now be used with functorch.",
            DeprecationWarning,
        )
        return True

    @classmethod
    def validate(cls, module: nn.Module, *, strict: bool = False) -> List[NotImplementedError]:
        """Trainable modules that own buffers (BatchNorm and the like) cannot have per-sample
        gradients: the buffers mix samples (grad_sample_module.py:446-485)."""
        errors = [
            NotImplementedError(
                f"Model contains a trainable layer with buffers that Opacus doesn't currently support({name}:{m}). "
            )
            for name, m in trainable_modules(module)
            if len(list(m.buffers())) > 0
        ]
        if strict and errors:
            raise NotImplementedError(errors)
        return errors

    def forbid_grad_accumulation(self):
        self.grad_accumulation_allowed = False

    def allow_grad_accumulation(self):
        self.grad_accumulation_allowed = True


class GradSampleModule(GradSampleHooks, AbstractGradSampleModule):
    """``nn.Module`` wrapper whose parameters carry ``.grad_sample`` after ``backward``."""

    def __init__(
        self,
        m: nn.Module,
        *,
        batch_first=True,
        loss_reduction="mean",
        strict: bool = True,
        force_functorch=False,
        autograd_weight_grads: Optional[bool] = None,
        lazy_linear_grad_sample: bool = False,
    ):
        nn.Module.__init__(self)
        GradSampleHooks.__init__(
            self,
            m,
            batch_first=batch_first,
            loss_reduction=loss_reduction,
            strict=strict,
            force_functorch=force_functorch,
            autograd_weight_grads=autograd_weight_grads,
            lazy_linear_grad_sample=lazy_linear_grad_sample,
        )
        self.grad_accumulation_hook = None

    def forward(self, *args, **kwargs):
        return self._module(*args, **kwargs)
