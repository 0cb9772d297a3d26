"""A recurrent layer whose recurrence is linear in the state, so that long sequences are scanned.

``DPGatedRNN`` stands beside ``DPRNN``, ``DPGRU`` and ``DPLSTM`` (reference: opacus/layers/dp_rnn.py).
Their gates read the previous state and force one launch after the other along time; here the
gates depend on the input alone,

    [x | r | i] = W_ih input + b_ih,   a = exp(-softplus(decay) * sigmoid(r)),
    h_t = a_t * h_{t-1} + sqrt(1 - a_t^2) * sigmoid(i_t) * x_t,

so one kernel scans a whole sequence, forward and backward, and one tiny kernel advances the
state by a token (:meth:`DPGatedRNN.step`). ``num_heads`` adds a norm and SiLU over the heads of
each output. Every trainable part has per-sample gradients: ``W_ih`` through the samplers of
``RNNLinear``, ``decay`` and the norm's weight and bias from the backward kernels themselves.
"""

from __future__ import annotations

import math
from typing import List, Optional, Tuple, Union

import torch
import torch.nn as nn
from torch import Tensor
from torch.nn.utils.rnn import PackedSequence

from .. import kernels
from .dp_rnn import RNNLinear, apply_permutation
from .norm_act import HeadNormAct
from .param_rows import first_derivative_only, forget_rows, parameter_rows


class _GatedScanFn(torch.autograd.Function):
    """``rows`` ``[n, D]`` stands for ``decay`` per sample and only receives its gradient."""

    @staticmethod
    def forward(ctx, gates, rows, state, decay, lengths, reverse):
        out, last, kept = kernels.gated_scan(
            gates, decay, state, lengths, reverse, keep_states=any(ctx.needs_input_grad)
        )
        ctx.save_for_backward(gates, decay, kept, lengths)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    def backward(ctx, grad_out, grad_last):
        first_derivative_only("gated scan")
        gates, decay, kept, lengths = ctx.saved_tensors
        if grad_out is None:
            grad_out = torch.zeros(gates.shape[0], gates.shape[1], decay.shape[0], dtype=gates.dtype, device=gates.device)
        d_gates, d_rows, d_state = kernels.gated_scan_backward(gates, decay, kept, grad_out, grad_last, lengths, ctx.reverse)
        need = ctx.needs_input_grad
        return (d_gates if need[0] else None), (d_rows if need[1] else None), (d_state if need[2] else None), None, None, None


class GatedScan(nn.Module):
    """The recurrence alone, with its ``decay`` per channel: ``[n, T, 3 D]`` gates (values, decay
    gates, input gates side by side; batch first) to the states ``[n, T, D]`` and the last state
    (float32 ``[n, D]``). At the start a half-open gate decays a channel by 0.9 to 0.999 a position."""

    per_sample_rows = True

    def __init__(self, hidden_size: int, reverse: bool = False, device=None, dtype=None) -> None:
        super().__init__()
        self.hidden_size, self.reverse = hidden_size, bool(reverse)
        self.decay = nn.Parameter(torch.empty(hidden_size, device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        with torch.no_grad():
            a = torch.empty(self.hidden_size).uniform_(0.9, 0.999)
            # softplus(decay) / 2 = -log a
            self.decay.copy_(torch.log(torch.expm1(-2.0 * torch.log(a))))

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, reverse={self.reverse}"

    def forward(
        self, gates: Tensor, state: Optional[Tensor] = None, lengths: Optional[Tensor] = None
    ) -> Tuple[Tensor, Tensor]:
        wide = kernels.widen(gates)  # float16 runs on the float32 kernels
        rows = None
        if torch.is_grad_enabled() and self.decay.requires_grad:
            rows = parameter_rows(self, (self.decay,), gates.shape[0])
        state = None if state is None else state.float()
        try:
            out, last = _GatedScanFn.apply(wide, rows, state, kernels.widen(self.decay.detach()), lengths, self.reverse)
        except BaseException:
            forget_rows(self)
            raise
        return (out if out.dtype == gates.dtype else out.to(gates.dtype)), last

    @torch.no_grad()
    def step(self, gates: Tensor, state: Tensor) -> Tensor:
        """One position, ``gates`` ``[n, 3 D]``; ``state`` (float32 ``[n, D]``) is advanced in place."""
        if self.reverse:
            raise ValueError("a reverse scan cannot be continued token by token")
        out = kernels.gated_scan_step(kernels.widen(gates), kernels.widen(self.decay.detach()), state)
        return out if out.dtype == gates.dtype else out.to(gates.dtype)


class DPGatedRNNCell(nn.Module):
    """One layer in one direction: projection, scan, and with ``num_heads`` norm and SiLU."""

    def __init__(self, input_size: int, hidden_size: int, bias: bool, reverse: bool, num_heads: Optional[int]) -> None:
        super().__init__()
        self.ih = RNNLinear(input_size, 3 * hidden_size, bias)
        stdv = 1.0 / math.sqrt(hidden_size)
        for p in self.ih.parameters():
            nn.init.uniform_(p, -stdv, stdv)
        self.scan = GatedScan(hidden_size, reverse)
        self.norm = None if num_heads is None else HeadNormAct(num_heads, hidden_size, activation="silu")
        if self.norm is not None:
            self.norm.follows_layout = False  # fed batch first whatever the model's layout

    def forward(self, x: Tensor, state: Optional[Tensor], lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
        out, last = self.scan(self.ih(x), state, lengths)
        return (out if self.norm is None else self.norm(out)), last

    def step(self, x: Tensor, state: Tensor) -> Tensor:
        out = self.scan.step(self.ih(x), state)
        return out if self.norm is None else self.norm(out)


class DPGatedRNN(nn.Module):
    """Inputs, outputs and the common arguments as ``DPGRU``: a ``[T, B, D]`` tensor (``[B, T, D]``
    with ``batch_first``) or a ``PackedSequence``, initial states ``[layers * directions, B, H]``;
    returns the outputs and the last states, which are float32 whatever the dtype of the inputs.

    ``lengths`` (int64 ``[B]`` on the inputs' device) marks a padded tensor's positions from
    ``lengths[b]`` on as padding, without the reordering of a ``PackedSequence``: the recurrence
    passes over them (its outputs there are zero, and ``silu(bias)`` behind the norm). A ``PackedSequence``
    is spread out and gathered again with masks, for which the host waits and which cannot be captured into a
    graph; ``lengths`` have neither drawback.
    ``num_heads`` normalises every head of each output and applies SiLU."""

    def __init__(
        self,
        input_size: int,
        hidden_size: int,
        num_layers: int = 1,
        bias: bool = True,
        batch_first: bool = False,
        dropout: float = 0.0,
        bidirectional: bool = False,
        num_heads: Optional[int] = None,
    ) -> None:
        super().__init__()
        if num_layers < 1:
            raise ValueError("num_layers must be at least 1")
        if not 0 <= dropout <= 1:
            raise ValueError("dropout should be a number in range [0, 1]")
        if num_heads is not None and (num_heads < 1 or hidden_size % num_heads != 0):
            raise ValueError("hidden_size must be divisible by num_heads")
        self.input_size, self.hidden_size, self.num_layers = input_size, hidden_size, num_layers
        self.batch_first, self.bidirectional, self.num_heads = batch_first, bidirectional, num_heads
        self.num_directions = 2 if bidirectional else 1
        self.dropout_layer = nn.Dropout(dropout) if dropout > 0 else None
        self.cells = nn.ModuleList(
            DPGatedRNNCell(
                input_size if layer == 0 else hidden_size * self.num_directions, hidden_size, bias, direction == 1, num_heads
            )
            for layer in range(num_layers)
            for direction in range(self.num_directions)
        )

    def forward(
        self,
        input: Union[Tensor, PackedSequence],
        state_init: Optional[Tensor] = None,
        lengths: Optional[Tensor] = None,
    ) -> Tuple[Union[Tensor, PackedSequence], Tensor]:
        packed = isinstance(input, PackedSequence)
        if packed:
            if lengths is not None:
                raise ValueError("a PackedSequence has its own lengths")
            data, batch_sizes, sorted_indices, unsorted_indices = input
            # live[b, t]: sample b (packed order) has a step t
            live = (torch.arange(int(batch_sizes[0])).unsqueeze(1) < batch_sizes.unsqueeze(0)).to(data.device)
            x = data.new_zeros(len(batch_sizes), live.shape[0], data.shape[-1])
            x[live.t()] = data  # row-major over (t, b) is the packed order
            x, lengths = x.transpose(0, 1), live.sum(dim=1)
            if unsorted_indices is not None:  # the caller's sample order, as in the layers around this one
                x, lengths = x.index_select(0, unsorted_indices), lengths.index_select(0, unsorted_indices)
        else:
            if input.dim() != 3:
                raise ValueError(f"expected a batch of sequences, got {tuple(input.shape)}")
            x = input if self.batch_first else input.transpose(0, 1)
        n_states = self.num_layers * self.num_directions
        if state_init is not None and tuple(state_init.shape) != (n_states, x.shape[0], self.hidden_size):
            raise ValueError(f"state_init must be {(n_states, x.shape[0], self.hidden_size)}, got {tuple(state_init.shape)}")
        last: List[Tensor] = []
        for layer in range(self.num_layers):
            if layer and self.dropout_layer is not None:
                x = self.dropout_layer(x)
            outs = []
            for direction in range(self.num_directions):
                k = layer * self.num_directions + direction
                out, h = self.cells[k](x, None if state_init is None else state_init[k], lengths)
                outs.append(out)
                last.append(h)
            x = outs[0] if len(outs) == 1 else torch.cat(outs, dim=2)
        hs = torch.stack(last, dim=0)
        if packed:
            x = apply_permutation(x, 0, sorted_indices).transpose(0, 1)
            return PackedSequence(x[live.t()], batch_sizes, sorted_indices, unsorted_indices), hs
        return (x if self.batch_first else x.transpose(0, 1)), hs

    def initial_state(self, batch_size: int, device=None) -> Tensor:
        """Zeros to start :meth:`step` from."""
        device = self.cells[0].scan.decay.device if device is None else device
        return torch.zeros(self.num_layers, batch_size, self.hidden_size, dtype=torch.float32, device=device)

    @torch.no_grad()
    def step(self, input: Tensor, state: Tensor) -> Tensor:
        """The next token of every sequence: ``input`` ``[B, input_size]``; ``state`` (dense float32
        ``[layers, B, H]``, from :meth:`initial_state` or a forward pass) is advanced in place. Returns
        the last layer's output ``[B, H]``. Dropout does not act here, and autograd records nothing."""
        if self.bidirectional:
            raise ValueError("a bidirectional layer cannot be continued token by token")
        if input.dim() != 2:
            raise ValueError(f"expected one token per sequence, [B, input_size], got {tuple(input.shape)}")
        if tuple(state.shape) != (self.num_layers, input.shape[0], self.hidden_size):
            raise ValueError(
                f"state must be {(self.num_layers, input.shape[0], self.hidden_size)}, got {tuple(state.shape)}"
            )
        x = input
        for k, cell in enumerate(self.cells):
            x = cell.step(x, state[k])
        return x
