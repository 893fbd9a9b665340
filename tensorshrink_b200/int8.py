"""Matrices of 8-bit integers with a scale per row, quantised on the GPU and
multiplied by the integer tensor cores.

Weights have a scale per output channel, activations one per token, found as
they come (no calibration): value = code * scale, code in [-127, 127]. The sums
of products are exact 32-bit integers, so that results do not depend on how a
product is split. The 8-bit format of `codec` is another: affine groups of
weights, dequantised on the way to 16-bit tensor cores, activations kept
(reference codec.py:102-151).

The functions are thin layers over `torch.ops.tensorshrink.int8_*`, with the
conventions of `fp4`: the current stream of the tensors' device, no
synchronisation, CUDA tensors only, no gradients (a backward pass that reaches a
result raises, and inputs with tangents are refused; a quantised tensor has no history).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .fp4 import _op


def padded_cols(cols: int) -> int:
    """Columns as stored: padded to a multiple of 16."""
    return -(-cols // 16) * 16


class Int8Tensor:
    """A [rows, cols] matrix of 8-bit integers with a scale per row.

    codes: int8 [rows, columns], at least `cols` padded to a multiple of 16
    columns; rows contiguous and on 16 bytes; columns behind `cols` (default:
    all are meant) do not count. scales: fp32 [rows]; a NaN makes its row's values
    NaN. cols: at most 131072."""

    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: Optional[int] = None):
        cols = codes.shape[-1] if cols is None else cols
        _op("int8_check")(codes, scales, cols)
        self.codes, self.scales, self.cols = codes, scales, cols

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def int8_quantize(x: torch.Tensor) -> Int8Tensor:
    """Quantise x [rows, cols] (fp16, bf16 or fp32; rows may be strided): each
    row's scale is max|x| / 127 (at least 2^-100), its codes x / scale rounded to
    nearest even. A row that holds an infinity or a NaN gets a NaN scale: its
    values come back as NaN."""
    t = Int8Tensor.__new__(Int8Tensor)
    t.codes, t.scales = _op("int8_quantize")(x)
    t.cols = x.shape[1]
    return t


def int8_dequantize(t: Int8Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of `t` as a [rows, cols] tensor."""
    return _op("int8_dequantize")(t.codes, t.scales, t.cols, dtype)


def int8_matmul(a: Int8Tensor, b: Int8Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] . b [N, K]^T (+ bias [N]): exact integer sums, scaled in fp32
    and rounded once to `out_dtype`."""
    if a.cols != b.cols:
        raise ValueError(f"int8_matmul of {a.shape} and {b.shape}")
    return _op("int8_matmul")(a.codes, a.scales, b.codes, b.scales, b.cols, bias, out_dtype)


def int8_linear(x: torch.Tensor, w: Int8Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] . w^T (+ bias): each token's activations are quantised as
    `int8_quantize` does and multiplied by the integer tensor cores. The result
    has x's type unless `out_dtype` says otherwise."""
    return _op("int8_linear")(x, w.codes, w.scales, w.cols, bias, out_dtype)


class Int8Linear(nn.Module):
    """A linear layer with an Int8Tensor weight. Buffers: `codes`, `scales`,
    `bias`. Casting the module (`.to(dtype)`, `.half()`) casts the bias; the
    scales stay fp32."""

    def __init__(self, weight: Int8Tensor, bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.in_features, self.out_features = weight.cols, weight.rows
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, layer: nn.Linear) -> "Int8Linear":
        """Quantise an nn.Linear whose weight is on the GPU."""
        return cls(int8_quantize(layer.weight.detach()), layer.bias.detach() if layer.bias is not None else None)

    def _apply(self, fn, recurse=True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)              # moved, but not rounded
        return self

    def weight(self) -> Int8Tensor:
        return Int8Tensor(self.codes, self.scales, self.in_features)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _op("int8_linear")(x, self.codes, self.scales, self.in_features, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"
