"""Microscaled 4-bit floating point (MXFP4): quantised rows and their product.

A row of K values is cut into blocks of 32; a block holds 32 e2m1 codes (magnitudes 0, .5,
1, 1.5, 2, 3, 4, 6, two codes per byte, the even value in the low nibble) and one power of
two as its scale (a byte e: 2^(e-127); 255: the block is NaN).  The scale's exponent is
floor(log2(max|x|)) - 2 in [-127, 127]; codes round to nearest, ties to the even code, and
saturate at 6.  A block with an infinity or a NaN becomes a NaN block.

The matrix cores multiply such rows as they are stored, so a weight matrix [N, K] is
quantised once along K and needs no other layout:

    weight = mx_quantize(dense)                 # [N, K], kept
    y = mx_product(x, weight, bias=bias)        # x [..., K] floats or an MXTensor -> [..., N]

This is the dense counterpart of the sparse weights' NVFP4 storage (``precision.py``), for
serving: products give no gradients.  Kernels: csrc/mx.hip and mx_product.hip behind
include/neurosim_hip_mx.h; calls run on the current stream and never synchronise.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import lru_cache

import torch

from .native import _raise_on, load_library
from .signal_ops import TYPES, _needs_grad, on_device

MX_BLOCK = 32                        # NS_MX_BLOCK
_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class _Matrix(ctypes.Structure):
    _fields_ = [("rows", _i64), ("columns", _i64), ("codes", _ptr), ("scales", _ptr)]


class _ProductArgs(ctypes.Structure):
    _fields_ = [("a", _Matrix), ("b", _Matrix), ("bias", _ptr), ("out", _ptr), ("stride", _i64),
                ("type", _i32), ("splits", _i32), ("partials", _ptr)]


@lru_cache(maxsize=1)
def _library() -> ctypes.CDLL:
    lib = load_library()
    for name in ("ns_mx_quantize", "ns_mx_dequantize"):
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.POINTER(_Matrix), _ptr, _i64, _i32, _ptr]
    lib.ns_mx_product.restype = ctypes.c_int
    lib.ns_mx_product.argtypes = [ctypes.POINTER(_ProductArgs), _ptr]
    lib.ns_mx_product_splits.restype = _i32
    lib.ns_mx_product_splits.argtypes = [_i64, _i64, _i64]
    return lib


@dataclass(frozen=True)
class MXTensor:
    """Quantised rows: ``codes`` uint8 [..., blocks * 16] and ``scales`` uint8 [..., blocks] of
    rows of ``columns`` values, blocks = ceil(columns / 32)."""

    codes: torch.Tensor
    scales: torch.Tensor
    columns: int

    def __post_init__(self) -> None:
        blocks = -(-self.columns // MX_BLOCK)
        for value, what, width in ((self.codes, "codes", blocks * (MX_BLOCK // 2)),
                                   (self.scales, "scales", blocks)):
            if (not isinstance(value, torch.Tensor) or value.dtype != torch.uint8
                    or value.dim() < 1 or value.shape[-1] != width):
                raise ValueError(f"{what} must be uint8 [..., {width}] for {self.columns} columns")
            if not value.is_contiguous():
                raise ValueError(f"{what} must be contiguous")
        if self.codes.shape[:-1] != self.scales.shape[:-1] or self.codes.device != self.scales.device:
            raise ValueError("codes and scales need the same rows on the same device")
        if self.codes.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.columns))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return mx_dequantize(self, dtype)


def _rows(value: MXTensor) -> int:
    return value.scales.shape[:-1].numel()


def _matrix(value: MXTensor) -> _Matrix:
    return _Matrix(_rows(value), value.columns,
                   value.codes.data_ptr() if value.codes.numel() else None,
                   value.scales.data_ptr() if value.scales.numel() else None)


def _stream(device: torch.device):
    return torch.cuda.current_stream(device).cuda_stream


def mx_quantize(x: torch.Tensor) -> MXTensor:
    """``x`` [..., K] (float32, bfloat16 or float16, on a GPU) quantised along its last dimension."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.dtype not in TYPES:
        raise ValueError("quantisation takes [..., K] tensors of float32, bfloat16 or float16")
    if x.device.type != "cuda":
        raise ValueError("quantisation needs its input on a GPU")
    if _needs_grad(x):
        raise ValueError("quantisation gives no gradients; detach its input")
    rows, columns = x.shape[:-1].numel(), x.shape[-1]
    blocks = -(-columns // MX_BLOCK)
    flat = x.detach().reshape(rows, columns) if x.dim() != 2 else x.detach()
    if columns > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    storage = torch.empty(rows * blocks * 17, dtype=torch.uint8, device=x.device)
    out = MXTensor(storage[:rows * blocks * 16].view(*x.shape[:-1], blocks * 16),
                   storage[rows * blocks * 16:].view(*x.shape[:-1], blocks), columns)
    lib, matrix = _library(), _matrix(out)
    with on_device(x.device):
        _raise_on(lib.ns_mx_quantize(ctypes.byref(matrix), flat.data_ptr() or None, flat.stride(0),
                                     TYPES[x.dtype], _stream(x.device)), lib)
    return out


def mx_dequantize(value: MXTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of quantised rows, rounded to ``dtype`` (exact in float32 and bfloat16)."""
    if not isinstance(value, MXTensor) or value.device.type != "cuda":
        raise ValueError("reading back needs an MXTensor on a GPU")
    if dtype not in TYPES:
        raise ValueError("values are read back as float32, bfloat16 or float16")
    out = torch.empty(value.shape, dtype=dtype, device=value.device)
    lib, matrix = _library(), _matrix(value)
    with on_device(value.device):
        _raise_on(lib.ns_mx_dequantize(ctypes.byref(matrix), out.data_ptr() or None, value.columns,
                                       TYPES[dtype], _stream(value.device)), lib)
    return out


def mx_product(x: torch.Tensor | MXTensor, weight: MXTensor, *, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` of quantised rows: x [..., K], weight [N, K], result [..., N].

    A float ``x`` is quantised on the way.  Sums are float32; the result is rounded once to
    ``dtype`` (x's own for a float x, else float32)."""
    if not isinstance(weight, MXTensor) or weight.codes.dim() != 2:
        raise ValueError("weight must be an MXTensor of [N, K]")
    if isinstance(x, torch.Tensor):
        dtype = dtype or x.dtype
        if x.dim() >= 1 and x.shape[-1] != weight.columns:
            raise ValueError(f"x has {x.shape[-1]} columns, the weight {weight.columns}")
        x = mx_quantize(x)
    elif not isinstance(x, MXTensor):
        raise ValueError("x must be a float tensor or an MXTensor")
    dtype = dtype or torch.float32
    if dtype not in TYPES:
        raise ValueError("a product is float32, bfloat16 or float16")
    if x.columns != weight.columns:
        raise ValueError(f"x has {x.columns} columns, the weight {weight.columns}")
    if x.device != weight.device or weight.device.type != "cuda":
        raise ValueError("x and the weight must be on the same GPU")
    rows, outputs = _rows(x), weight.codes.shape[0]
    if bias is not None:
        if (not isinstance(bias, torch.Tensor) or bias.shape != (outputs,)
                or bias.dtype != torch.float32 or bias.device != weight.device):
            raise ValueError("bias must be float32 [N] on the weight's device")
        if _needs_grad(bias):
            raise ValueError("a 4-bit product gives no gradients")
        bias = bias.detach().contiguous()
    out = torch.empty((*x.shape[:-1], outputs), dtype=dtype, device=weight.device)
    lib = _library()
    splits = lib.ns_mx_product_splits(rows, outputs, weight.columns)
    partials = (torch.empty(splits * rows * outputs, dtype=torch.float32, device=weight.device)
                if splits > 1 else None)
    args = _ProductArgs(_matrix(x), _matrix(weight), bias.data_ptr() if bias is not None else None,
                        out.data_ptr() or None, outputs, TYPES[dtype], splits,
                        partials.data_ptr() if partials is not None else None)
    with on_device(weight.device):
        _raise_on(lib.ns_mx_product(ctypes.byref(args), _stream(weight.device)), lib)
    return out
