"""4-bit integer weights with a scale per group of columns, and their product with float rows.

A row of K values is cut into groups of 32, 64 or a multiple of 128 columns; a value is
``(code - zero) * scale`` with a 4-bit code, one scale of a float type and, unless the codes
are symmetric around 8, one zero point per group.  Only the weight has few bits: the rows it
multiplies stay float32, bfloat16 or float16, so a read-out of rates or the drive of one tick
loses nothing but the weight's rounding (``microscaled`` quantises both).

    weight = q4_quantize(dense, group=128)      # [N, K], kept
    y = q4_product(x, weight, bias=bias)        # x [..., K] -> [..., N]

Quantising takes ``scale = hi/15 - lo/15`` of a group's range with 0 in it, ``zero =
round(-lo/scale)`` and ``code = round(x/scale) + zero`` (symmetric: ``max|x|/7`` and 8), ties to
even.  A group with an infinity or a NaN reads back as NaN.  For serving: products give no
gradients.  Kernels: csrc/q4.hip and q4_product.hip behind include/neurosim_hip_q4.h; calls
run on the current stream and never synchronise.
"""

from __future__ import annotations

import ctypes
import struct
from functools import lru_cache

import torch

from .microscaled import _check_floats, _float_rows, _rows
from .native import load_library
from .signal_ops import TYPES, _address, _needs_grad, call

_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
_MAX_COLUMNS = 1 << 23                     # NS_Q4_MAX_COLUMNS

# ns_q4_matrix: N, K, group; codes, scales, zeros; scale_type.  ns_q4_product_args: the weight;
# M; x and its stride; bias, out and its stride; type; workspace.
_MATRIX = struct.Struct("=3q3Qi4x")
_PRODUCT = struct.Struct("=3q3Qi4x q Qq 2Q q i4x Q")


@lru_cache(maxsize=1)
def _library() -> ctypes.CDLL:
    lib = load_library()
    for name in ("ns_q4_quantize", "ns_q4_dequantize"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = ctypes.c_int, [_ptr, _ptr, _i64, _i32, _ptr]
    lib.ns_q4_product.restype, lib.ns_q4_product.argtypes = ctypes.c_int, [_ptr, _ptr]
    lib.ns_q4_product_floats.restype = _i64
    lib.ns_q4_product_floats.argtypes = [_i64, _i64, _i64, _i32]
    return lib


def _check_group(group, columns: int) -> None:
    if (not isinstance(group, int) or group > _MAX_COLUMNS
            or (group not in (32, 64) and (group <= 0 or group % 128))):
        raise ValueError(f"a group has 32, 64 or a multiple of 128 columns, up to {_MAX_COLUMNS}")
    if columns > _MAX_COLUMNS:
        raise ValueError(f"a 4-bit row has at most {_MAX_COLUMNS} columns")


class Q4Tensor:
    """Rows of 4-bit integers: ``codes`` uint8 [..., ceil(columns/32) * 16], two a byte, the even
    value in the low nibble; ``scales`` [..., ceil(columns/group)] (float32, bfloat16 or float16);
    ``zeros`` uint8 like the scales, or None where every zero point is 8."""

    __slots__ = ("codes", "scales", "zeros", "columns", "group")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None,
                 columns: int, group: int) -> None:
        _check_group(group, columns)
        width, groups = -(-columns // 32) * 16, -(-columns // group)
        if (not isinstance(codes, torch.Tensor) or codes.dtype != torch.uint8 or codes.dim() < 1
                or codes.shape[-1] != width):
            raise ValueError(f"codes must be uint8 [..., {width}] for {columns} columns")
        if (not isinstance(scales, torch.Tensor) or scales.dtype not in TYPES or scales.dim() < 1
                or scales.shape[-1] != groups):
            raise ValueError(f"scales must be float32, bfloat16 or float16 [..., {groups}]")
        if zeros is not None and (not isinstance(zeros, torch.Tensor) or zeros.dtype != torch.uint8
                                  or zeros.shape != scales.shape or zeros.device != codes.device):
            raise ValueError("zeros must be uint8, like the scales")
        if codes.shape[:-1] != scales.shape[:-1] or codes.device != scales.device:
            raise ValueError("codes and scales need the same rows on the same device")
        for value, what in ((codes, "codes"), (scales, "scales"), (zeros, "zeros")):
            if value is not None and not value.is_contiguous():
                raise ValueError(f"{what} must be contiguous")
        if codes.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.columns, self.group = columns, group

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.columns))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __repr__(self) -> str:
        return f"Q4Tensor(shape={list(self.shape)}, group={self.group}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return q4_dequantize(self, dtype)


def _fields(weight: Q4Tensor, rows: int) -> tuple:
    return (rows, weight.columns, weight.group, weight.codes.data_ptr(), weight.scales.data_ptr(),
            _address(weight.zeros), TYPES[weight.scales.dtype])


def q4_quantize(x: torch.Tensor, group: int = 128, *, symmetric: bool = False,
                dtype: torch.dtype = torch.bfloat16) -> Q4Tensor:
    """``x`` [..., K] (float32, bfloat16 or float16, on a GPU) quantised along its last
    dimension, with scales of ``dtype``; ``symmetric`` ones have no zero points."""
    _check_floats(x)
    if dtype not in TYPES:
        raise ValueError("scales are float32, bfloat16 or float16")
    *lead, columns = x.shape
    _check_group(group, columns)
    rows, groups = _rows(lead), -(-columns // group)
    flat = _float_rows(x, rows, columns)
    result = Q4Tensor.__new__(Q4Tensor)              # as made here, without checks
    result.codes = x.new_empty((*lead, -(-columns // 32) * 16), dtype=torch.uint8)
    result.scales = x.new_empty((*lead, groups), dtype=dtype)
    result.zeros = None if symmetric else x.new_empty((*lead, groups), dtype=torch.uint8)
    result.columns, result.group = columns, group
    call(_library().ns_q4_quantize, x.device, _MATRIX.pack(*_fields(result, rows)), flat.data_ptr(),
         flat.stride(0), TYPES[x.dtype])
    return result


def q4_dequantize(value: Q4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of quantised rows, rounded to ``dtype``."""
    if not isinstance(value, Q4Tensor) or not value.codes.is_cuda:
        raise ValueError("reading back needs a Q4Tensor on a GPU")
    if dtype not in TYPES:
        raise ValueError("values are read back as float32, bfloat16 or float16")
    lead = value.codes.shape[:-1]
    out = value.codes.new_empty((*lead, value.columns), dtype=dtype)
    call(_library().ns_q4_dequantize, value.codes.device, _MATRIX.pack(*_fields(value, _rows(lead))),
         out.data_ptr(), value.columns, TYPES[dtype])
    return out


def q4_product(x: torch.Tensor, weight: Q4Tensor, *, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias``: x [..., K] (float32, bfloat16 or float16), weight [N, K] of 4-bit
    groups, result [..., N] of x's type.  Sums are float32 and the result is rounded once.  A
    group's sum (of 128 columns at most) is off by some 2^-24 of its scale times (16 + zero) times
    the sum of |x|, for float32 rows of |x - their mean|: a value much larger than its
    neighbours costs them bits even where its own weight is zero.  A row of x that holds an
    infinity or a NaN gives NaN, and one with values beyond 2^115, 128 of which times a code
    pass float32, may."""
    if not isinstance(weight, Q4Tensor) or weight.codes.dim() != 2:
        raise ValueError("weight must be a Q4Tensor of [N, K]")
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.dtype not in TYPES:
        raise ValueError("x must be a [..., K] tensor of float32, bfloat16 or float16")
    columns, outputs, device = weight.columns, weight.codes.shape[0], weight.codes.device
    *lead, width = x.shape
    if width != columns:
        raise ValueError(f"x has {width} columns, the weight {columns}")
    if x.device != device or not x.is_cuda:
        raise ValueError("x and the weight must be on the same GPU")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.shape != (outputs,)
                             or bias.dtype != torch.float32 or bias.device != device):
        raise ValueError("bias must be float32 [N] on the weight's device")
    if _needs_grad(x, bias):
        raise ValueError("a 4-bit product gives no gradients")
    if bias is not None:
        bias = bias.contiguous()
    rows, lib = _rows(lead), _library()
    flat = _float_rows(x, rows, columns)
    out = x.new_empty((*lead, outputs))
    size = lib.ns_q4_product_floats(rows, outputs, columns, TYPES[x.dtype])
    work = x.new_empty(size, dtype=torch.float32) if size else None
    args = _PRODUCT.pack(*_fields(weight, outputs), rows, flat.data_ptr(), flat.stride(0),
                         _address(bias), out.data_ptr(), outputs,
                         TYPES[x.dtype], _address(work))
    call(lib.ns_q4_product, device, args)
    return out
