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
import struct
from functools import lru_cache

import torch

from .native import load_library
from .signal_ops import TYPES, _needs_grad, call

MX_BLOCK = 32                        # NS_MX_BLOCK
_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p

# The C argument structs, packed: ns_mx_matrix (rows, columns, codes, scales), and
# ns_mx_product_args (a; b; bias, out; stride; types; x; its stride; workspace).
_MATRIX = struct.Struct("=2q2Q")
_PRODUCT = struct.Struct("=2q2Q 2q2Q 2Q q 2i Q q Q")


@lru_cache(maxsize=1)
def _library() -> ctypes.CDLL:
    lib = load_library()
    for name in ("ns_mx_quantize", "ns_mx_dequantize"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = ctypes.c_int, [_ptr, _ptr, _i64, _i32, _ptr]
    lib.ns_mx_product.restype, lib.ns_mx_product.argtypes = ctypes.c_int, [_ptr, _ptr]
    lib.ns_mx_product_bytes.restype = _i64
    lib.ns_mx_product_bytes.argtypes = [_i64, _i64, _i64, _i32]
    return lib


class MXTensor:
    """Quantised rows: ``codes`` uint8 [..., blocks * 16] and ``scales`` uint8 [..., blocks] of
    rows of ``columns`` values, blocks = ceil(columns / 32)."""

    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: int) -> None:
        blocks = (columns + MX_BLOCK - 1) // MX_BLOCK
        for value, what, width in ((codes, "codes", blocks * (MX_BLOCK // 2)),
                                   (scales, "scales", blocks)):
            if (not isinstance(value, torch.Tensor) or value.dtype != torch.uint8
                    or value.dim() < 1 or value.shape[-1] != width):
                raise ValueError(f"{what} must be uint8 [..., {width}] for {columns} columns")
            if not value.is_contiguous():
                raise ValueError(f"{what} must be contiguous")
        if codes.shape[:-1] != scales.shape[:-1] or codes.device != scales.device:
            raise ValueError("codes and scales need the same rows on the same device")
        if codes.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        self.codes, self.scales, self.columns = codes, scales, columns

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.columns))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __repr__(self) -> str:
        return f"MXTensor(shape={list(self.shape)}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return mx_dequantize(self, dtype)


def _rows(lead) -> int:
    rows = 1
    for size in lead:
        rows *= size
    return rows


def _float_rows(x: torch.Tensor, rows: int, columns: int) -> torch.Tensor:
    """x as [rows, columns] with dense rows (a copy where they are not)."""
    if x.dim() != 2:
        x = x.reshape(rows, columns)
    return x if columns <= 1 or x.stride(1) == 1 else x.contiguous()


def _check_floats(x) -> None:
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.dtype not in TYPES:
        raise ValueError("quantisation takes [..., K] tensors of float32, bfloat16 or float16")
    if not x.is_cuda:
        raise ValueError("quantisation needs its input on a GPU")
    if _needs_grad(x):
        raise ValueError("quantisation gives no gradients; detach its input")


def mx_quantize(x: torch.Tensor) -> MXTensor:
    """``x`` [..., K] (float32, bfloat16 or float16, on a GPU) quantised along its last dimension."""
    _check_floats(x)
    *lead, columns = x.shape
    rows, blocks, device = _rows(lead), (columns + MX_BLOCK - 1) // MX_BLOCK, x.device
    flat = _float_rows(x, rows, columns)
    codes = x.new_empty((*lead, blocks * 16), dtype=torch.uint8)
    scales = x.new_empty((*lead, blocks), dtype=torch.uint8)
    matrix = _MATRIX.pack(rows, columns, codes.data_ptr(), scales.data_ptr())
    call(_library().ns_mx_quantize, device, matrix, flat.data_ptr(), flat.stride(0), TYPES[x.dtype])
    result = MXTensor.__new__(MXTensor)              # as made here, without checks
    result.codes, result.scales, result.columns = codes, scales, columns
    return result


def mx_dequantize(value: MXTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of quantised rows, rounded to ``dtype`` (exact in float32 and bfloat16)."""
    if not isinstance(value, MXTensor) or not value.codes.is_cuda:
        raise ValueError("reading back needs an MXTensor on a GPU")
    if dtype not in TYPES:
        raise ValueError("values are read back as float32, bfloat16 or float16")
    codes, scales, columns = value.codes, value.scales, value.columns
    lead, device = codes.shape[:-1], codes.device
    out = codes.new_empty((*lead, columns), dtype=dtype)
    matrix = _MATRIX.pack(_rows(lead), columns, codes.data_ptr(), scales.data_ptr())
    call(_library().ns_mx_dequantize, device, matrix, out.data_ptr(), columns, TYPES[dtype])
    return out


def mx_product(x: torch.Tensor | MXTensor, weight: MXTensor, *, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` of quantised rows: x [..., K], weight [N, K], result [..., N]
    (K up to 2^23).

    A float ``x`` is quantised on the way.  Sums are float32; the result is rounded once to
    ``dtype`` (x's own for a float x, else float32)."""
    if not isinstance(weight, MXTensor) or weight.codes.dim() != 2:
        raise ValueError("weight must be an MXTensor of [N, K]")
    columns, outputs, device = weight.columns, weight.codes.shape[0], weight.codes.device
    floats = isinstance(x, torch.Tensor)
    if floats:
        _check_floats(x)
        *lead, width = x.shape
        dtype = dtype or x.dtype
    elif isinstance(x, MXTensor):
        lead, width = x.codes.shape[:-1], x.columns
        dtype = dtype or torch.float32
    else:
        raise ValueError("x must be a float tensor or an MXTensor")
    if width != columns:
        raise ValueError(f"x has {width} columns, the weight {columns}")
    if dtype not in TYPES:
        raise ValueError("a product is float32, bfloat16 or float16")
    if x.device != device or not weight.codes.is_cuda:
        raise ValueError("x and the weight must be on the same GPU")
    if bias is not None:
        if (not isinstance(bias, torch.Tensor) or bias.shape != (outputs,)
                or bias.dtype != torch.float32 or bias.device != device):
            raise ValueError("bias must be float32 [N] on the weight's device")
        if _needs_grad(bias):
            raise ValueError("a 4-bit product gives no gradients")
        bias = bias.contiguous()
    rows, lib = _rows(lead), _library()
    out = weight.codes.new_empty((*lead, outputs), dtype=dtype)
    size = lib.ns_mx_product_bytes(rows, outputs, columns, floats)
    work = out.new_empty(size, dtype=torch.uint8) if size else None
    if floats and size:
        flat = _float_rows(x, rows, columns)
        a, rest = (0, 0), (TYPES[x.dtype], flat.data_ptr(), flat.stride(0))
    else:
        a = (0, 0) if floats else (x.codes.data_ptr(), x.scales.data_ptr())
        rest = (0, 0, 0)
    args = _PRODUCT.pack(rows, columns, *a, outputs, columns, weight.codes.data_ptr(),
                         weight.scales.data_ptr(), 0 if bias is None else bias.data_ptr(),
                         out.data_ptr(), outputs, TYPES[dtype], *rest,
                         0 if work is None else work.data_ptr())
    call(lib.ns_mx_product, device, args)
    return out
