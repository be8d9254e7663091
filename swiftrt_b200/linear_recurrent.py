"""A recurrent layer whose gates depend on its input alone: one product over all time steps and an elementwise,
gated linear recurrence (srtGatedRecurrence) in the place of a product per step.

The column blocks of the fused weight are named as those of the reference's LSTM cell (Part,
Sources/SwiftRTLayers/Recurrent.swift:173); the state is what its State.cell is (Recurrent.swift:222-241), kept in
Float32 so that a gate close to one still moves it."""
from __future__ import annotations

import torch

from .dense import bias_activation_backward
from .matmul import binding, matmul, rows_of
from .tensor import ActivationType

STATE_CHUNK = 64            # steps between two kept states (SRT_GATED_RECURRENCE_CHUNK)


def gated_recurrence(update: torch.Tensor, forget: torch.Tensor, input: torch.Tensor | None = None,
                     output: torch.Tensor | None = None, initial: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, keep: bool = False, last: torch.Tensor | None = None):
    """(hidden, last state) -- and the kept states with `keep`, for gated_recurrence_backward -- of

        c_t = s(forget_t) c_{t-1} + i_t update_t,   i_t = s(input_t), or 1 - s(forget_t) without `input`
        hidden_t = c_t s(output_t), or c_t without `output`                        (s: the logistic function)

    over [batch, steps, channels] tensors, or [batch, channels] for one step.  `initial` and the last state are
    Float32 [batch, channels]; `last` names the tensor that receives the latter and may be `initial` itself (a
    state advanced in place).  `lengths` (int32, one per batch item): steps behind them leave the state alone and
    have a hidden value of zero.  Asynchronous on torch's current stream of update's device."""
    return binding.recurrence(update, forget, input, output, initial, lengths, keep, last)


def gated_recurrence_backward(out_grad: torch.Tensor, update: torch.Tensor, forget: torch.Tensor, input: torch.Tensor | None,
                              output: torch.Tensor | None, states: torch.Tensor, lengths: torch.Tensor | None = None,
                              last_grad: torch.Tensor | None = None, out: tuple | None = None):
    """Gradients of (update, forget, input, output, initial) of gated_recurrence for the gradient of its hidden
    values and, with `last_grad`, of its last state; None for a gate that is None.  `states` are the ones that the
    forward pass kept.  `out` names the four tensors (None for an absent gate) that receive the first four."""
    return binding.recurrence_backward(out_grad, update, forget, input, output, states, lengths, last_grad, *(out or (None,) * 4))


class LinearRecurrentCell:
    """A recurrent layer over [batch, steps, inputSize] sequences: one product with fusedWeight
    [inputSize x (3 or 4) hiddenSize] (+ fusedBias) gives the column blocks (input,) update, forget and output of
    every step, and gated_recurrence does the rest.  With three blocks the input gate is 1 - forget gate."""

    def __init__(self, fused_weight: torch.Tensor, fused_bias: torch.Tensor | None, hidden_size: int):
        if fused_weight.dim() != 2 or fused_weight.shape[1] not in (3 * hidden_size, 4 * hidden_size):
            raise ValueError("fusedWeight must be [inputSize x 3 hiddenSize] or [inputSize x 4 hiddenSize]")
        if fused_bias is not None and tuple(fused_bias.shape) != (fused_weight.shape[1],):
            raise ValueError("fusedBias has one element per column of fusedWeight")
        self.fused_weight = fused_weight
        self.fused_bias = fused_bias
        self.hidden_size = int(hidden_size)
        self.has_input_gate = fused_weight.shape[1] == 4 * hidden_size

    def zero_state(self, input: torch.Tensor) -> torch.Tensor:
        """zeroState(for:) (Recurrent.swift:245-248): Float32 [batch, hiddenSize]."""
        return torch.zeros((input.shape[0], self.hidden_size), dtype=torch.float32, device=input.device)

    def _gates(self, input: torch.Tensor):
        """(fused, (update, forget, input gate or None, output)) of [batch, (steps,) inputSize]."""
        fused = matmul(rows_of(input), self.fused_weight, bias=self.fused_bias)
        return fused, self._blocks(fused.view(*input.shape[:-1], fused.shape[-1]))

    def _blocks(self, fused: torch.Tensor):
        h = self.hidden_size
        blocks = [fused[..., i * h:(i + 1) * h] for i in range(fused.shape[-1] // h)]
        return (blocks[1], blocks[2], blocks[0], blocks[3]) if self.has_input_gate else (blocks[0], blocks[1], None, blocks[2])

    def __call__(self, input: torch.Tensor, state: torch.Tensor | None = None, lengths: torch.Tensor | None = None):
        """(hidden [batch, steps, hiddenSize], last state) of a [batch, steps, inputSize] sequence."""
        _, (update, forget, gate, output) = self._gates(input)
        return gated_recurrence(update, forget, gate, output, state, lengths)

    def step(self, input: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """One step of generation: hidden [batch, hiddenSize] for an input [batch, inputSize]; `state` advances in place."""
        _, (update, forget, gate, output) = self._gates(input)
        return gated_recurrence(update, forget, gate, output, state, last=state)[0]

    def forward_keep(self, input: torch.Tensor, state: torch.Tensor | None = None, lengths: torch.Tensor | None = None):
        """(hidden, last state, saved) for training; `saved` goes to backward()."""
        fused, (update, forget, gate, output) = self._gates(input)
        hidden, last, states = gated_recurrence(update, forget, gate, output, state, lengths, keep=True)
        return hidden, last, (fused, states, lengths)

    def backward(self, input: torch.Tensor, saved: tuple, out_grad: torch.Tensor, last_grad: torch.Tensor | None = None):
        """(input gradient, weight gradient, bias gradient or None, initial state gradient)."""
        fused, states, lengths = saved
        update, forget, gate, output = self._blocks(fused.view(*input.shape[:-1], fused.shape[-1]))
        fused_grad = torch.empty_like(fused)
        grads = self._blocks(fused_grad.view(*input.shape[:-1], fused.shape[-1]))
        initial_grad = gated_recurrence_backward(out_grad, update, forget, gate, output, states, lengths, last_grad, out=grads)[-1]
        dx = matmul(fused_grad, self.fused_weight, False, True).view(input.shape)
        dw = matmul(rows_of(input), fused_grad, True, False)
        db = None
        if self.fused_bias is not None:
            db = bias_activation_backward(fused_grad, None, ActivationType.identity, want_dz=False)[1]
        return dx, dw, db, initial_grad
