"""Microscaled 4-bit floating point: tensors whose E2M1 elements share a scale
per block, quantised on the GPU and multiplied by the block-scaled tensor
cores.

Next to the GOAP formats of `codec` (2/4/8-bit affine or codebook weights,
dequantised on the way to the tensor cores), these are formats that the
tensor cores of sm_100a multiply as they are, for weights and activations
alike:

* "nvfp4": blocks of 16 columns with an E4M3 scale, and one fp32 scale of the
  whole tensor;
* "mxfp4": blocks of 32 columns with a power of two as scale.

The reference has neither (its 4-bit codes are integers, codec.py:102-151).
The functions are thin layers over `torch.ops.tensorshrink.fp4_*`, which check
their arguments and launch on the current stream of the tensors' device;
nothing synchronises, so calls can be captured in a graph. They take CUDA
tensors only and compute no gradients: a backward pass that reaches one of their
results raises. (Codes are integers, so that none reaches `fp4_quantize`.)
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import _C

FORMATS = {"nvfp4": _C.TS_NVFP4, "mxfp4": _C.TS_MXFP4}
BLOCK = {"nvfp4": 16, "mxfp4": 32}

_ops = {}


def _op(name: str, overload: str = "default"):
    """The operator `torch.ops.tensorshrink.<name>.<overload>`, looked up once."""
    f = _ops.get((name, overload))
    if f is None:
        f = _ops[name, overload] = getattr(getattr(_C.serving_ops(), name), overload)
    return f


def _format(name: str) -> int:
    try:
        return FORMATS[name]
    except KeyError:
        raise NotImplementedError(f"format {name!r} is not one of {sorted(FORMATS)}") from None


def padded_cols(cols: int) -> int:
    """Columns as stored: padded with zeros to a multiple of 64."""
    return -(-cols // 64) * 64


def scales_nbytes(rows: int, cols: int, format: str) -> int:
    """Bytes of the scales: tiles of 128 rows x 4 blocks, 512 bytes each."""
    return -(-rows // 128) * -(-(padded_cols(cols) // BLOCK[format]) // 4) * 512


class Fp4Tensor:
    """A [rows, cols] matrix in a microscaled 4-bit format.

    codes: uint8 [rows, padded_cols / 2], the even column in the low nibble.
    scales: uint8, flat, `scales_nbytes` long: E4M3 or E8M0 bytes in tiles of
    128 rows x 4 blocks, the byte of (row r, block j) at
    (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4 of its tile; bytes of rows behind
    the last one are never read. global_scale: fp32 [1] of an nvfp4 tensor
    (None counts as 1)."""

    __slots__ = ("codes", "scales", "global_scale", "rows", "cols", "format", "_code")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, global_scale: Optional[torch.Tensor], rows: int,
                 cols: int, format: str):
        code = _format(format)
        _op("fp4_check")(codes, scales, global_scale, rows, cols, code)
        self.codes, self.scales, self.global_scale = codes, scales, global_scale
        self.rows, self.cols, self.format, self._code = rows, cols, format, code

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + (4 if self.global_scale is not None else 0)


def fp4_quantize(x: torch.Tensor, format: str = "nvfp4", global_scale: Optional[torch.Tensor] = None) -> Fp4Tensor:
    """Quantise x [rows, cols] (fp16, bf16 or fp32; rows may be strided).

    nvfp4: with `global_scale` (fp32, one value, e.g. from a calibration) that
    scale is used, otherwise the tensor's own, max|x| / 2688 over its finite
    elements, is found first. Rounding is to nearest even throughout. A block
    that holds an infinity or a NaN gets a NaN scale: its values come back as
    NaN."""
    t = Fp4Tensor.__new__(Fp4Tensor)
    t.format, t._code = format, _format(format)
    t.codes, t.scales, found = _op("fp4_quantize")(x, t._code, global_scale)
    t.global_scale = global_scale if found is None else found
    t.rows, t.cols = x.shape
    return t


def fp4_dequantize(t: Fp4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of `t` as a [rows, cols] tensor."""
    return _op("fp4_dequantize")(t.codes, t.scales, t.global_scale, t.rows, t.cols, t._code, dtype)


def fp4_matmul(a: Fp4Tensor, b: Fp4Tensor, bias: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] . b [N, K]^T (+ bias [N]) of two tensors of one format, summed
    in fp32 and rounded once to `out_dtype`."""
    if a._code != b._code or a.cols != b.cols:
        raise ValueError(f"fp4_matmul of {a.format} {a.shape} and {b.format} {b.shape}")
    return _op("fp4_matmul")(a.codes, a.scales, a.global_scale, a.rows, b.codes, b.scales, b.global_scale, b.rows, b.cols,
                             b._code, bias, out_dtype)


def fp4_linear(x: torch.Tensor, w: Fp4Tensor, bias: Optional[torch.Tensor] = None,
               input_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] . w^T (+ bias): the activations are quantised to w's format
    (nvfp4: with `input_scale`, fp32, None for 1) and multiplied by the
    tensor cores. The result has x's type unless `out_dtype` says otherwise."""
    return _op("fp4_linear")(x, w.codes, w.scales, w.global_scale, w.rows, w.cols, w._code, bias, input_scale, out_dtype)


class Fp4Linear(nn.Module):
    """A linear layer with an Fp4Tensor weight. Buffers: `codes`, `scales`,
    `global_scale` (nvfp4) and `input_scale` (nvfp4: the activations' tensor
    scale, 1 until `calibrate`), `bias`. Casting the module (`.to(dtype)`,
    `.half()`) casts the bias; the tensor scales stay fp32."""

    def __init__(self, weight: Fp4Tensor, bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.in_features, self.out_features, self.format = weight.cols, weight.rows, weight.format
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("global_scale", weight.global_scale)
        one = torch.ones(1, dtype=torch.float32, device=weight.device) if weight.format == "nvfp4" else None
        self.register_buffer("input_scale", one)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, layer: nn.Linear, format: str = "nvfp4") -> "Fp4Linear":
        """Quantise an nn.Linear whose weight is on the GPU."""
        b = layer.bias.detach() if layer.bias is not None else None
        return cls(fp4_quantize(layer.weight.detach(), format), b)

    def _apply(self, fn, recurse=True):
        scales = {name: getattr(self, name) for name in ("global_scale", "input_scale")}
        super()._apply(fn, recurse)
        for name, scale in scales.items():
            cast = getattr(self, name)
            if cast is not None and cast.dtype != torch.float32:
                setattr(self, name, scale.to(cast.device))      # moved, but not rounded
        return self

    def weight(self) -> Fp4Tensor:
        return Fp4Tensor(self.codes, self.scales, self.global_scale, self.out_features, self.in_features, self.format)

    @torch.no_grad()
    def calibrate(self, x: torch.Tensor) -> None:
        """Set `input_scale` from sample activations: max|x| / 2688 over the
        finite ones, as `fp4_quantize` finds a tensor's scale."""
        if self.input_scale is not None:
            x = x.detach().float()
            top = torch.where(x.isfinite(), x, torch.zeros_like(x)).abs().amax()
            self.input_scale.copy_((top / 2688.0).clamp(min=2.0 ** -100).reshape(1))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _op("fp4_linear")(x, self.codes, self.scales, self.global_scale, self.out_features, self.in_features,
                                 FORMATS[self.format], self.bias, self.input_scale)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, format={self.format}"
