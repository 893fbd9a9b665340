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
Every launch goes to `torch.cuda.current_stream()` of the input's device.
"""

from __future__ import annotations

import ctypes as C
from contextlib import nullcontext
from typing import Optional

import torch
from torch import nn

from . import _C
from .kernels import _DTYPES, _ptr, _require_cuda, _serving_workspace, _stream_handle, dtype_code

FORMATS = {"nvfp4": _C.TS_NVFP4, "mxfp4": _C.TS_MXFP4}
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def _on(device: torch.device):
    """The device made current, for launches on another than the current one."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _format(name: str) -> int:
    try:
        return FORMATS[name]
    except KeyError:
        raise NotImplementedError(f"format {name!r} is not one of {sorted(FORMATS)}") from None


def padded_cols(cols: int) -> int:
    """Columns as stored: padded with zeros to a multiple of 64."""
    return -(-cols // 64) * 64


def scales_nbytes(rows: int, cols: int, format: str) -> int:
    """Bytes of the scales: tiles of 128 rows x 4 blocks of 512 bytes."""
    return -(-rows // 128) * -(-(padded_cols(cols) // BLOCK[format]) // 4) * 512


class Fp4Tensor:
    """A [rows, cols] matrix in a microscaled 4-bit format.

    codes: uint8 [rows, padded_cols / 2], the even column in the low nibble.
    scales: uint8, flat, `scales_nbytes` long: E4M3 or E8M0 bytes in tiles of
    128 rows x 4 blocks, the byte of (row r, block j) at
    (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4 of its tile; bytes of rows behind
    the last one are never read. global_scale: fp32 [1] of an nvfp4 tensor
    (None counts as 1)."""

    __slots__ = ("codes", "scales", "global_scale", "rows", "cols", "format", "_c")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, global_scale: Optional[torch.Tensor], rows: int,
                 cols: int, format: str):
        code = _format(format)
        rows, cols = int(rows), int(cols)
        if rows < 0 or cols <= 0:
            raise ValueError(f"bad shape [{rows}, {cols}]")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("codes and scales must be uint8")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        if codes.numel() != rows * (padded_cols(cols) // 2):
            raise ValueError(f"codes hold {codes.numel()} bytes, [{rows}, {padded_cols(cols) // 2}] wanted")
        if scales.numel() < scales_nbytes(rows, cols, format):
            raise ValueError(f"scales hold {scales.numel()} bytes, {scales_nbytes(rows, cols, format)} wanted")
        if global_scale is not None:
            if code != _C.TS_NVFP4:
                raise ValueError("only nvfp4 has a global_scale")
            if global_scale.dtype != torch.float32 or global_scale.numel() != 1:
                raise ValueError("global_scale must be one fp32 value")
        _require_cuda(codes, scales, global_scale, what="Fp4Tensor")
        self.codes, self.scales, self.global_scale = codes, scales, global_scale
        self.rows, self.cols, self.format = rows, cols, format
        self._c = _C.TsFp4Tensor(codes.data_ptr(), scales.data_ptr(), _ptr(global_scale), rows, cols, code, 0)

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + (4 if self.global_scale is not None else 0)


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"{what}: dtype {x.dtype} is not supported")
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    return x


def _scale_arg(g: Optional[torch.Tensor], what: str) -> Optional[torch.Tensor]:
    if g is not None and (g.dtype != torch.float32 or g.numel() != 1):
        raise ValueError(f"{what} must be one fp32 value")
    return g


def fp4_quantize(x: torch.Tensor, format: str = "nvfp4", global_scale: Optional[torch.Tensor] = None) -> Fp4Tensor:
    """Quantise x [rows, cols] (fp16, bf16 or fp32; rows may be strided).

    nvfp4: with `global_scale` (fp32, one value, e.g. from a calibration) that
    scale is used, otherwise the tensor's own, max|x| / 2688 over its finite
    elements, is found first. Rounding is to nearest even throughout. A block
    that holds an infinity or a NaN gets a NaN scale: its values come back as
    NaN."""
    code = _format(format)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"fp4_quantize takes a [rows, cols] tensor, got {tuple(x.shape)}")
    dev = _require_cuda(x, global_scale, what="fp4_quantize")
    if global_scale is not None and code != _C.TS_NVFP4:
        raise ValueError("only nvfp4 has a global_scale")
    x = _rows(x, "fp4_quantize")
    rows, cols = x.shape
    find = code == _C.TS_NVFP4 and global_scale is None
    g = torch.empty(1, dtype=torch.float32, device=dev) if find else _scale_arg(global_scale, "global_scale")
    if find and rows == 0:
        g.fill_(1.0)
    kb = padded_cols(cols) // 2
    buf = torch.empty(rows * kb + scales_nbytes(rows, cols, format), dtype=torch.uint8, device=dev)
    t = Fp4Tensor(buf[:rows * kb].view(rows, kb), buf[rows * kb:], g, rows, cols, format)
    lib = _C.load()
    with _on(dev):
        ws = _serving_workspace(dev, _SCRATCH_AT + lib.ts_fp4_quantize_workspace_size()) if find else None
        rc = lib.ts_fp4_quantize(x.data_ptr(), dtype_code(x.dtype), x.stride(0), t._c, 1 if find else 0,
                                 ws.data_ptr() + _SCRATCH_AT if find else None,
                                 ws.numel() - _SCRATCH_AT if find else 0, _stream_handle(dev))
    _C.check(rc, "ts_fp4_quantize")
    return t


_SCRATCH_AT = 256 * 1024     # behind the serving workspace's counters


def fp4_dequantize(t: Fp4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of `t` as a [rows, cols] tensor."""
    code = dtype_code(dtype)
    out = torch.empty((t.rows, t.cols), dtype=dtype, device=t.device)
    with _on(t.device):
        rc = _C.load().ts_fp4_dequantize(t._c, out.data_ptr(), code, t.cols, _stream_handle(t.device))
    _C.check(rc, "ts_fp4_dequantize")
    return out


def _check_out(bias, n: int, out_dtype: torch.dtype):
    if bias is not None and (bias.numel() != n or bias.dtype not in _DTYPES or not bias.is_contiguous()):
        raise ValueError(f"bias must be {n} contiguous fp16, bf16 or fp32 values")
    return dtype_code(out_dtype)


def fp4_matmul(a: Fp4Tensor, b: Fp4Tensor, bias: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] . b [N, K]^T (+ bias [N]) of two tensors of one format, summed
    in fp32 and rounded once to `out_dtype`."""
    dev = _require_cuda(a.codes, b.codes, bias, what="fp4_matmul")
    if a.format != b.format or a.cols != b.cols:
        raise ValueError(f"fp4_matmul of {a.format} {a.shape} and {b.format} {b.shape}")
    code = _check_out(bias, b.rows, out_dtype)
    out = torch.empty((a.rows, b.rows), dtype=out_dtype, device=dev)
    lib = _C.load()
    with _on(dev):
        ws = _serving_workspace(dev, lib.ts_fp4_matmul_workspace_size(a.rows, b.rows, b.cols, b._c.format))
        rc = lib.ts_fp4_matmul(a._c, b._c, _ptr(bias), dtype_code(bias.dtype) if bias is not None else 0,
                               out.data_ptr(), code, b.rows, ws.data_ptr(), ws.numel(), _stream_handle(dev))
    _C.check(rc, "ts_fp4_matmul")
    return out


def fp4_linear(x: torch.Tensor, w: Fp4Tensor, bias: Optional[torch.Tensor] = None,
               input_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] . w^T (+ bias): the activations are quantised to w's format
    (nvfp4: with `input_scale`, fp32, None for 1) and multiplied by the
    tensor cores. The result has x's type unless `out_dtype` says otherwise."""
    dev = _require_cuda(x, w.codes, bias, input_scale, what="fp4_linear")
    if x.shape[-1] != w.cols:
        raise ValueError(f"fp4_linear: x has {x.shape[-1]} features, the weight {w.cols}")
    if input_scale is not None:
        if w._c.format != _C.TS_NVFP4:
            raise ValueError("only nvfp4 has an input_scale")
        _scale_arg(input_scale, "input_scale")
    x2d = _rows(x if x.dim() == 2 else x.reshape(-1, w.cols), "fp4_linear")
    out_dtype = out_dtype or x.dtype
    code = _check_out(bias, w.rows, out_dtype)
    m = x2d.shape[0]
    out = torch.empty((*x.shape[:-1], w.rows), dtype=out_dtype, device=dev)
    lib = _C.load()
    with _on(dev):
        ws = _serving_workspace(dev, lib.ts_fp4_linear_workspace_size(m, w.rows, w.cols, w._c.format))
        rc = lib.ts_fp4_linear(x2d.data_ptr(), dtype_code(x2d.dtype), m, x2d.stride(0), _ptr(input_scale), w._c,
                               _ptr(bias), dtype_code(bias.dtype) if bias is not None else 0, out.data_ptr(), code,
                               w.rows, ws.data_ptr(), ws.numel(), _stream_handle(dev))
    _C.check(rc, "ts_fp4_linear")
    return out


class Fp4Linear(nn.Module):
    """A linear layer with an Fp4Tensor weight. Buffers: `codes`, `scales`,
    `global_scale` (nvfp4) and `input_scale` (nvfp4: the activations' tensor
    scale, 1 until `calibrate`), `bias`."""

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

    def weight(self) -> Fp4Tensor:
        return Fp4Tensor(self.codes, self.scales, self.global_scale, self.out_features, self.in_features, self.format)

    @torch.no_grad()
    def calibrate(self, x: torch.Tensor) -> None:
        """Set `input_scale` from sample activations: max|x| / 2688."""
        if self.input_scale is not None:
            top = x.detach().float().abs().amax()
            self.input_scale.copy_((top / 2688.0).clamp(min=2.0 ** -100).reshape(1))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp4_linear(x, self.weight(), self.bias, self.input_scale)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, format={self.format}"
