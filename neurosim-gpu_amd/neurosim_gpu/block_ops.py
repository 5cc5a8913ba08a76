"""Operators of a gated block over the ticks of a signal: gated projection and dropout.

* ``gated_projection``: ``f(x gate^T) * (x up^T)`` with f silu or gelu, both products, the
  activation and the product in one kernel, with native gradients of x and both weights;
* ``dropout``: elements kept by a counter-based generator, whose mask is computed anew where
  it is used and never stored; optionally added to a residual in the same pass.

float32, bfloat16 and float16 are taken; sums are float32 and each output is rounded once.  The
projection's 16-bit gradients multiply dg and du (``gated_projection``) rounded to that type too.
Forward-mode derivatives are refused, and so is a backward under graph capture.  The kernels
are csrc/gated.hip, gated_grad.hip and dropout.hip behind include/neurosim_hip_block.h; calls run
on the current stream, allocate their outputs and workspaces from torch, and never synchronise.
"""

from __future__ import annotations

import ctypes
import struct
import sys
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from .microscaled import _float_rows, _rows
from .native import load_library
from .signal_ops import TYPES, _address, _needs_grad, call, refuse_capture

ACTIVATIONS = {"silu": 0, "gelu": 1}       # NS_GATE_*
_MAX_ROWS = 1 << 21                        # NS_GATED_MAX_ROWS

_i64, _ptr = ctypes.c_int64, ctypes.c_void_p
# ns_gated_args: M, K, F; type, activation; x, gate, up, y with their strides; pre; dy and its
# stride; dx, dweights, workspace.
_GATED = struct.Struct("=3q2i Qq Qq Qq Qq Q Qq 3Q")
# ns_dropout_args: count; type, threshold; x, residual, out; seed_data, seed, offset.
_DROPOUT = struct.Struct("=q2i 3Q 3Q")
_WORD = (1 << 64) - 1


@lru_cache(maxsize=1)
def _library() -> ctypes.CDLL:
    lib = load_library()
    for name in ("ns_gated_forward", "ns_gated_backward", "ns_dropout"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = ctypes.c_int, [_ptr, _ptr]
    for name in ("ns_gated_forward_bytes", "ns_gated_backward_bytes"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _i64, [_ptr]
    return lib


# ---- gated projection ----------------------------------------------------------------

def _gated_args(x, gate, up, activation, y=None, pre=None, dy=None, dx=None, dweights=None) -> bytes:
    """The packed arguments, without a workspace: its size goes by the others."""
    (rows, columns), width = x.shape, gate.shape[0]
    return _GATED.pack(rows, columns, width, TYPES[x.dtype], activation, x.data_ptr(), x.stride(0),
                       gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0), _address(y),
                       width, _address(pre), _address(dy), 0 if dy is None else dy.stride(0),
                       _address(dx), _address(dweights), 0)


def _call_with_workspace(fn, size: int, device, args: bytes) -> None:
    if size:
        work = torch.empty(size, dtype=torch.uint8, device=device)
        args = args[:-8] + work.data_ptr().to_bytes(8, sys.byteorder)     # its last field
    call(fn, device, args)


def _gated_forward(x, gate, up, activation, keep: bool):
    """(y, the two products or None) of rows with dense values."""
    lib, (rows, _), width = _library(), x.shape, gate.shape[0]
    y = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    pre = torch.empty((2, rows, width), dtype=torch.float32, device=x.device) if keep else None
    args = _gated_args(x, gate, up, activation, y, pre)
    _call_with_workspace(lib.ns_gated_forward, lib.ns_gated_forward_bytes(args), x.device, args)
    return y, pre


class _GatedProjection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, activation):
        y, pre = _gated_forward(x, gate, up, activation, True)
        ctx.save_for_backward(x, gate, up, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_capture("gated_projection")
        x, gate, up, pre = ctx.saved_tensors
        wants, lib, (rows, columns), width = ctx.needs_input_grad, _library(), x.shape, gate.shape[0]
        if not rows or not columns or not width:
            return (*(torch.zeros_like(v) if w else None for v, w in zip((x, gate, up), wants)), None)
        dy = _float_rows(dy, rows, width)
        dx = torch.empty((rows, columns), dtype=x.dtype, device=x.device) if wants[0] else None
        dweights = (torch.empty((2, width, columns), dtype=x.dtype, device=x.device)
                    if wants[1] or wants[2] else None)
        args = _gated_args(x, gate, up, ctx.activation, None, pre, dy, dx, dweights)
        _call_with_workspace(lib.ns_gated_backward, lib.ns_gated_backward_bytes(args), x.device, args)
        return (dx, dweights[0] if wants[1] else None, dweights[1] if wants[2] else None, None)


def gated_projection(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, *,
                     activation: str = "silu") -> torch.Tensor:
    """``f(x @ gate.T) * (x @ up.T)`` of ``x`` [..., K], ``gate`` and ``up`` [F, K] (K and F up
    to 2^20), all of one type; the result is [..., F].  ``activation`` f is "silu" or "gelu"
    (of the normal distribution function, not its tanh form).  Call it with a batch's ticks
    or with a single one; up to 16 rows are bound by the weights' bytes.  Large float32 calls,
    and all float32 gradients, are multiplied in three bfloat16 parts at float32's precision;
    an infinity in x or a weight then makes its row or column NaN.  A call with gradients takes
    up to 2^21 rows and keeps both products in float32 for its backward, whose
    ``dg = dy u f'(g)`` and ``du = dy f(g)`` (g and u: the two products) are rounded to x's type
    before they are multiplied: half a unit of a 16-bit type more than float32 between the
    products would leave.  In float16 they are rounded as multiples of a power of two per row and
    column, so only the gradients themselves have to be in its range."""
    if activation not in ACTIVATIONS:
        raise ValueError("activation must be 'silu' or 'gelu'")
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.dtype not in TYPES:
        raise ValueError("x must be a [..., K] tensor of float32, bfloat16 or float16")
    if not x.is_cuda:
        raise ValueError("x must be on a GPU")
    *lead, columns = x.shape
    for value, what in ((gate, "gate"), (up, "up")):
        if not isinstance(value, torch.Tensor) or value.dim() != 2 or value.shape[1] != columns:
            raise ValueError(f"{what} must be a [F, {columns}] tensor")
        if value.dtype != x.dtype:
            raise ValueError(f"{what} must be {str(x.dtype).removeprefix('torch.')} as x is")
        if value.device != x.device:
            raise ValueError(f"{what} must be on x's device")
    if gate.shape != up.shape:
        raise ValueError("gate and up need the same shape")
    rows, width = _rows(lead), gate.shape[0]
    flat = _float_rows(x, rows, columns)
    gate, up = _float_rows(gate, width, columns), _float_rows(up, width, columns)
    if _needs_grad(x, gate, up):
        if rows > _MAX_ROWS:
            raise ValueError(f"a projection with gradients takes up to {_MAX_ROWS} rows")
        y = _GatedProjection.apply(flat, gate, up, ACTIVATIONS[activation])
    else:
        y, _ = _gated_forward(flat, gate, up, ACTIVATIONS[activation], False)
    return y if x.dim() == 2 else y.view(*lead, width)


# ---- dropout -------------------------------------------------------------------------

def _drop(x, residual, threshold: int, seed, offset: int) -> torch.Tensor:
    """Dense tensors in, a dense one out."""
    out = torch.empty_like(x)
    drawn = isinstance(seed, torch.Tensor)
    args = _DROPOUT.pack(x.numel(), TYPES[x.dtype], threshold, x.data_ptr(), _address(residual),
                         out.data_ptr(), seed.data_ptr() if drawn else 0, 0 if drawn else seed, offset)
    call(_library().ns_dropout, x.device, args)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, offset):
        drawn = isinstance(seed, torch.Tensor)
        # The backward draws the same numbers: a seed changed in between is noticed.
        ctx.save_for_backward(seed if drawn else None)
        ctx.rest = threshold, None if drawn else seed, offset
        return _drop(x.contiguous(), None if residual is None else residual.contiguous(), threshold,
                     seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_capture("dropout")
        (drawn,), (threshold, seed, offset) = ctx.saved_tensors, ctx.rest
        dx = (_drop(dy.contiguous(), None, threshold, seed if drawn is None else drawn, offset)
              if ctx.needs_input_grad[0] else None)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, *, seed, offset: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + x`` with each element of ``x`` dropped with probability ``p`` (to the
    nearest 1/65536, which the kept ones' scale follows) and the kept ones divided by 1 - p.

    Which are kept depends on ``seed``, ``offset`` and the element's place in x's own order,
    not on strides: eight 16-bit numbers from each counter of Philox4x32 with 10 rounds (Salmon
    et al. 2011).  ``seed`` is an integer (64 bits count), or a one-element int64 tensor on x's
    device, read when the kernel runs, so that replays of a captured graph follow it; the
    backward draws the mask again and refuses a seed tensor changed since.  Calls with one
    seed take other offsets (integers of 64 bits)."""
    if not isinstance(x, torch.Tensor) or x.dtype not in TYPES:
        raise ValueError("x must be a tensor of float32, bfloat16 or float16")
    if not x.is_cuda:
        raise ValueError("x must be on a GPU")
    if not 0.0 <= p <= 1.0:
        raise ValueError("p is a probability")
    if residual is not None and (not isinstance(residual, torch.Tensor) or residual.shape != x.shape
                                 or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("residual must be like x")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError("a seed tensor is one int64 on x's device")
    elif isinstance(seed, int):
        seed &= _WORD
    else:
        raise ValueError("seed must be an integer or an int64 tensor")
    if not isinstance(offset, int):
        raise ValueError("offset must be an integer")
    threshold, offset = round(p * 65536), offset & _WORD
    if _needs_grad(x, residual):
        return _Dropout.apply(x, residual, threshold, seed, offset)
    return _drop(x.contiguous(), None if residual is None else residual.contiguous(), threshold,
                 seed, offset)
