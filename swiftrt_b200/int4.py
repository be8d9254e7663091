"""Weights in 4 bits with one scale (and possibly one zero point) per column and group of rows, and products of a few
rows with them (srtMatmulInt4): W[k, n] = (q[k, n] - z[k // group, n]) * scale[k // group, n]."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import lib
from .matmul import binding, descriptor_args, enqueue, on_one_device, rows_of
from .tensor import ActivationType, data_type


def _on_rows_of(t: torch.Tensor, nbytes: int) -> torch.Tensor:
    """`t` itself where its rows lie behind each other and start on multiples of `nbytes`, else a copy whose rows do."""
    width = nbytes // t.element_size()
    if t.numel() == 0 or (t.data_ptr() % nbytes == 0 and (t.shape[0] == 1 or (t.stride(0) >= t.shape[1] and t.stride(0) % width == 0))):
        return t
    out = torch.empty((t.shape[0], -(-t.shape[1] // width) * width), dtype=t.dtype, device=t.device)[:, :t.shape[1]]
    return out.copy_(t)


class Int4Weight:
    """A [rows, cols] weight: `packed` int32 [ceil(rows / 8), cols] (row 8 j + i of column n in bits 4 i .. 4 i + 3 of word
    (j, n)), `scales` [ceil(rows / group), cols] in Float16 or BFloat16, `zeros` uint8 of the same shape or None (8).
    Stands where a layer takes a weight (Dense, GatedDense) for its forward pass.

    The products read 16 bytes of a row at a time: tensors whose rows do not start on 16 bytes (8 for scales, 4 for
    zeros), as those of 1001 contiguous columns, are copied once into ones whose rows do; so are repeated rows (one
    scale expanded over all groups)."""

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int, rows: int):
        self.rows, self.cols, self.group = int(rows), int(packed.shape[-1]), int(group)
        groups = -(-self.rows // self.group) if self.group > 0 else 0
        for name, t, dtypes, count in (("packed", packed, (torch.int32,), -(-self.rows // 8)),
                                       ("scales", scales, (torch.float16, torch.bfloat16), groups), ("zeros", zeros, (torch.uint8,), groups)):
            if t is None:
                continue
            if t.dtype not in dtypes or tuple(t.shape) != (count, self.cols) or (self.cols > 1 and t.stride(1) != 1):
                raise ValueError(f"{name} must be [{count}, {self.cols}] of {' or '.join(map(str, dtypes))} with contiguous columns")
        on_one_device(packed, scales, zeros)
        packed, scales = _on_rows_of(packed, 16), _on_rows_of(scales, 8)
        zeros = _on_rows_of(zeros, 4) if zeros is not None else None
        self._tensors = packed, scales, zeros
        self.shape, self.dtype, self.device = (self.rows, self.cols), scales.dtype, packed.device
        stride = lambda t: max(t.stride(0), self.cols)  # noqa: E731  (a single row may have any stride)
        self._struct = _lib.Int4Matrix(data_type(scales), self.group, self.rows, self.cols, packed.data_ptr(), stride(packed), scales.data_ptr(),
                                       stride(scales), zeros.data_ptr() if zeros is not None else None, stride(zeros) if zeros is not None else 0)
        self.address = ctypes.addressof(self._struct)

    # (the library holds their addresses: their elements may change, the tensors may not)
    packed = property(lambda self: self._tensors[0])
    scales = property(lambda self: self._tensors[1])
    zeros = property(lambda self: self._tensors[2])

    def dequantize(self) -> torch.Tensor:
        """The weight as a [rows, cols] tensor of its type, each element rounded once (srtDequantizeInt4)."""
        out = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        enqueue(lib.srtDequantizeInt4, self.device, self.address, *descriptor_args(out))
        return out


def quantize_int4(weight: torch.Tensor, group: int = 128, zero_points: bool = False) -> Int4Weight:
    """A Float16 or BFloat16 [rows, cols] weight to 4 bits (srtQuantizeInt4): symmetric about zero, or with a zero point
    per column and group."""
    on_one_device(weight)
    rows, cols = weight.shape
    groups = -(-rows // group)
    q = Int4Weight(torch.empty((-(-rows // 8), cols), dtype=torch.int32, device=weight.device),
                   torch.empty((groups, cols), dtype=weight.dtype, device=weight.device),
                   torch.empty((groups, cols), dtype=torch.uint8, device=weight.device) if zero_points else None, group, rows)
    enqueue(lib.srtQuantizeInt4, weight.device, *descriptor_args(weight), q.address)
    return q


def matmul_int4(x: torch.Tensor, weight: Int4Weight, bias: torch.Tensor | None = None,
                activation: ActivationType = ActivationType.identity) -> torch.Tensor:
    """activation(x . weight + bias) for an [..., rows] tensor x; asynchronous on torch's current stream."""
    out = binding.int4(rows_of(x), weight.address, 0, weight.packed, weight.cols, bias, None, int(activation))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], out.shape[-1])


def gated_matmul_int4(x: torch.Tensor, weight_gate: Int4Weight, weight_up: Int4Weight, bias_gate: torch.Tensor | None = None,
                      bias_up: torch.Tensor | None = None, activation: ActivationType = ActivationType.silu) -> torch.Tensor:
    """activation(x . weight_gate + bias_gate) * (x . weight_up + bias_up) (srtMatmulGatedInt4)."""
    if weight_up.device != weight_gate.device:
        raise ValueError(f"tensors on different devices: {weight_gate.device} and {weight_up.device}")
    out = binding.int4(rows_of(x), weight_gate.address, weight_up.address, weight_gate.packed, weight_gate.cols, bias_gate, bias_up, int(activation))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], out.shape[-1])
