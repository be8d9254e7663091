"""Dense layer: y = activation(x . W + b), the semantics that the reference's Dense declares
(Sources/SwiftRTLayers/Dense.swift:21-71: fields activation / weight / bias, weight
[inputSize x outputSize], bias [outputSize], init assertion bias.shape[0] == weight.shape[1])
but does not compute (callAsFunction returns its input, Dense.swift:36-39).  One fused kernel
launch per call."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import lib
from .int4 import Int4Weight, gated_matmul_int4, matmul_int4
from .matmul import MatmulError, _descriptor, binding, matmul, rows_of
from .tensor import ActivationType, order_of


def bias_activation_backward(out_grad: torch.Tensor, output: torch.Tensor | None, activation: ActivationType,
                             want_dz: bool = True, want_dbias: bool = True):
    """(dz, dbias) of the fused epilogue: dz = out_grad * activation'(output), dbias = column sums of dz.
    For gelu and geluTanh `output` is the PRE-activation tensor (see Dense.forward_keep).

    The derivatives that the reference leaves unimplemented for matmul(bias:)
    (differentiable/MathDerivatives.swift:520-554), written in terms of the forward output like the
    reference's cuDNN activation backward (cuda/layers/CudaActivation.swift:101-127).  One pass over
    out_grad and output on torch's current stream."""
    if not out_grad.is_cuda:
        raise ValueError("device tensors expected")
    activation = ActivationType(activation)
    dz = torch.empty_like(out_grad, memory_format=torch.contiguous_format) if want_dz else None
    dbias = torch.empty((out_grad.shape[-1],), dtype=out_grad.dtype, device=out_grad.device) if want_dbias else None
    d_dy = _descriptor(out_grad)
    d_y = _descriptor(output) if output is not None else None
    d_dz = _descriptor(dz) if dz is not None else None
    d_db = _descriptor(dbias) if dbias is not None else None
    with torch.cuda.device(out_grad.device):
        rc = lib.srtBiasActivationBackward(
            out_grad.data_ptr(), d_dy.ref(), output.data_ptr() if output is not None else None,
            d_y.ref() if d_y is not None else None, int(activation),
            dz.data_ptr() if dz is not None else None, d_dz.ref() if d_dz is not None else None,
            dbias.data_ptr() if dbias is not None else None, d_db.ref() if d_db is not None else None,
            torch.cuda.current_stream(out_grad.device).cuda_stream)
    if rc != _lib.cudaSuccess:
        raise MatmulError(rc, _lib.last_error())
    return dz, dbias


def activation_forward(pre_activation: torch.Tensor, activation: ActivationType, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = activation(z), elementwise (srtActivationForward): the layer output of a Dense that kept
    its pre-activation values for the backward pass."""
    if not pre_activation.is_cuda:
        raise ValueError("device tensors expected")
    y = out if out is not None else torch.empty_like(pre_activation, memory_format=torch.contiguous_format)
    dz, dy = _descriptor(pre_activation), _descriptor(y)
    with torch.cuda.device(pre_activation.device):
        rc = lib.srtActivationForward(pre_activation.data_ptr(), dz.ref(), int(ActivationType(activation)), y.data_ptr(), dy.ref(),
                                      torch.cuda.current_stream(pre_activation.device).cuda_stream)
    if rc != _lib.cudaSuccess:
        raise MatmulError(rc, _lib.last_error())
    return y


_NEEDS_PRE_ACTIVATION = (ActivationType.gelu, ActivationType.geluTanh)


class Dense:
    """`weight` may be an Int4Weight (forward only, `bias` may then be None)."""

    def __init__(self, weight: torch.Tensor | Int4Weight, bias: torch.Tensor | None, activation: ActivationType):
        self.int4 = isinstance(weight, Int4Weight)
        # Dense.swift:48-49
        if not self.int4:
            assert order_of(weight) == order_of(bias) or bias.dim() == 1
        if bias is not None:
            assert bias.shape[0] == weight.shape[-1], "bias.shape[0] must equal weight.shape[1]"
        self.weight = weight
        self.bias = bias
        self.activation = ActivationType(activation)
        self.plan = None            # Dense.plan (Dense.swift:29): the plan is chosen per call

    def __call__(self, input: torch.Tensor) -> torch.Tensor:
        if self.int4:
            return matmul_int4(input, self.weight, self.bias, self.activation)
        return matmul(input, self.weight, bias=self.bias, activation=self.activation)

    def forward_keep(self, input: torch.Tensor):
        """(output, saved) for training: `saved` is what backward() needs in place of the output.  For
        activations whose derivative is a function of the output (identity, relu, sigmoid, tanh) this is
        the fused call and saved is the output itself; GELU's derivative needs the pre-activation
        values, so the product runs with the identity epilogue, its result is kept, and the activation
        is a second elementwise pass."""
        if self.int4:
            raise ValueError("a 4-bit weight has no backward pass")
        if self.activation in _NEEDS_PRE_ACTIVATION:
            z = matmul(input, self.weight, bias=self.bias, activation=ActivationType.identity)
            return activation_forward(z, self.activation), z
        y = self(input)
        return y, y

    def backward(self, input: torch.Tensor, output: torch.Tensor, out_grad: torch.Tensor):
        """(input gradient, weight gradient, bias gradient) for y = activation(x . W + b); `output` is
        the second value of forward_keep (the layer output, or the pre-activation values for GELU).

        dz and db come from one fused pass; dx = dz . W^T and dW = x^T . dz are the two transposed
        products that matmulGradients composes (MathDerivatives.swift:460-482, case (false, false))."""
        if self.int4:
            raise ValueError("a 4-bit weight has no backward pass")
        dz, db = bias_activation_backward(out_grad, output, self.activation)
        dx = matmul(dz, self.weight, False, True)
        dw = matmul(input, dz, True, False)
        return dx, dw, db


class GatedDense:
    """y = activation(x . weightGate + biasGate) * (x . weightUp + biasUp): two Dense layers over one input and the
    product of their results, as one launch (srtMatmulGated).  Weights [inputSize x outputSize], both tensors or both
    Int4Weight (forward only), biases [outputSize] or None.  Inputs may have any leading dimensions."""

    def __init__(self, weight_gate, weight_up, bias_gate: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
                 activation: ActivationType = ActivationType.silu):
        if tuple(weight_gate.shape) != tuple(weight_up.shape) or len(weight_gate.shape) != 2:
            raise ValueError("weightGate and weightUp must be matrices of one shape")
        self.int4 = isinstance(weight_gate, Int4Weight)
        if self.int4 != isinstance(weight_up, Int4Weight):
            raise ValueError("weightGate and weightUp are both 4-bit weights or neither is")
        for bias in (bias_gate, bias_up):
            if bias is not None and tuple(bias.shape) != (weight_gate.shape[1],):
                raise ValueError("a bias has one element per column of its weight")
        self.weight_gate, self.weight_up = weight_gate, weight_up
        self.bias_gate, self.bias_up = bias_gate, bias_up
        self.activation = ActivationType(activation)

    def _forward(self, x: torch.Tensor, keep: bool):
        return binding.gated(x, self.weight_gate, self.weight_up, self.bias_gate, self.bias_up, int(self.activation), keep)

    def __call__(self, input: torch.Tensor) -> torch.Tensor:
        if self.int4:
            return gated_matmul_int4(input, self.weight_gate, self.weight_up, self.bias_gate, self.bias_up, self.activation)
        y = self._forward(rows_of(input), False)
        return y if input.dim() == 2 else y.view(*input.shape[:-1], y.shape[-1])

    def forward_keep(self, input: torch.Tensor):
        """(output, saved) for training; `saved` is the pair of pre-activations that backward() needs."""
        if self.int4:
            raise ValueError("4-bit weights have no backward pass")
        y, gate, up = self._forward(rows_of(input), True)
        return y.view(*input.shape[:-1], y.shape[-1]), (gate, up)

    def backward(self, input: torch.Tensor, saved: tuple, out_grad: torch.Tensor):
        """Gradients of (input, weightGate, weightUp, biasGate, biasUp); None for a bias that is None.  `saved` is the
        second value of forward_keep.  Both weights' gradients are parts of one allocation."""
        if self.int4:
            raise ValueError("4-bit weights have no backward pass")
        gate, up = saved
        dx, dwg, dwu, dbg, dbu = binding.gated_backward(rows_of(input), rows_of(out_grad), self.weight_gate, self.weight_up, gate, up, self.bias_gate,
                                                        self.bias_up, int(self.activation))
        return dx.view(input.shape), dwg, dwu, dbg, dbu
