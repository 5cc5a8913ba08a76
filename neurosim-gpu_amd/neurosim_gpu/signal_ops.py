"""The signal operators around the tick: causal convolution and selective scan.

A signal is a [T, B, N] tensor: ticks, columns, channels, in the order of a rollout's
staged drives (a [B, T, N] tensor goes in as its ``transpose(0, 1)``, read in place).
float32, bfloat16 and float16 signals are taken; sums, states and gate functions are
float32 and each output is rounded once.

* ``causal_conv``: a short filter per channel, ``y[t] = silu(bias + sum_k w[k] x[t-W+1+k])``;
* ``selective_scan``: per channel S leaky integrators whose time step, input weights and
  read-out follow the signal,
  ``h[t] = exp(dt A) h[t-1] + dt x B[t]``, ``y[t] = (C[t] . h[t] + D x) silu(z)`` with
  ``dt = softplus(delta + delta_bias)``.

Both take and return the state that carries a signal on (``history``, ``state``), give
native gradients of every tensor input (forward-mode derivatives are refused), and have a
one-tick form that updates the carried state in place.  ``lengths`` gives columns their own
number of ticks: past it outputs and gradients are zero, the carried state stays that of the
column's last tick, and what the inputs hold there is never used.  The kernels are
csrc/conv.hip, scan.hip, scan_grad.hip behind include/neurosim_hip_signal.h; calls run on
the current stream, allocate their outputs and workspaces from torch, and never synchronise.
"""

from __future__ import annotations

import ctypes
import struct
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .native import _RAW_STREAM, _raise_on, load_library

MAX_TAPS, MAX_STATES = 8, 64         # NS_CONV_MAX_TAPS, NS_SCAN_MAX_STATES
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # NS_TYPE_*

# The C argument structs, packed in one go: a call's host time is most of a small call.
# ns_conv_args: shape; x; weight, bias; history; lengths; y, out_history, dy, dout_history,
# dx, dhistory; partials, dweight.
_CONV = struct.Struct("=3q4i Q2q 2Q Q2q Q Q2q Q2q Q2q Q2q Q2q Q2q 2Q")
_CONV_FORWARD = struct.Struct("=3q4i Q2q 2Q Q2q Q Q2q Q2q 112x")
# ns_scan_args: shape; x, delta, z, y; B, C; A, D, delta_bias, state, out_state, lengths,
# checkpoints, ends; dy; dout_state; dx, ddelta, dz, dB, dC; dstate, dparameters (those of A, D
# and delta_bias in one piece), partials.
_SCAN = struct.Struct("=4q4i Q2q Q2q Q2q Q2q Q2q Q2q 8Q Q2q Q Q2q Q2q Q2q Q2q Q2q 3Q")
_SCAN_FORWARD = struct.Struct("=4q4i Q2q Q2q Q2q Q2q Q2q Q2q 8Q 176x")
_ABSENT = (0, 0, 0)

_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
_Sizes = _i64 * 4


@lru_cache(maxsize=1)
def _library() -> ctypes.CDLL:
    lib = load_library()
    for name in ("ns_conv_forward", "ns_conv_step", "ns_conv_backward", "ns_scan_forward",
                 "ns_scan_step", "ns_scan_backward"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = ctypes.c_int, [_ptr, _ptr]
    lib.ns_conv_backward_floats.restype = _i64
    lib.ns_conv_backward_floats.argtypes = [_i64, _i64, _i64, _i32, _i32]
    lib.ns_scan_plan.restype = ctypes.c_int
    lib.ns_scan_plan.argtypes = [_i64, _i64, _i64, _i64, _i32, _i32, _ptr]
    return lib


def call(fn, device: torch.device, *args) -> None:
    """A library function with ``device`` current, on torch's current stream (its last
    argument)."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        code = fn(*args, _RAW_STREAM(index))
    else:
        with torch.cuda.device(device):
            code = fn(*args, _RAW_STREAM(index))
    if code:
        _raise_on(code, load_library())


def _address(value: torch.Tensor | None) -> int:
    return 0 if value is None else value.data_ptr()


def _signal(value: torch.Tensor | None) -> tuple[int, int, int]:
    """(address, tick stride, column stride); an empty tensor's address is 0."""
    if value is None:
        return _ABSENT
    return value.data_ptr(), value.stride(0), value.stride(1)


def _unit_channels(value: torch.Tensor | None, inner: int = 1):
    """``value`` with its last ``inner`` dimensions dense (a copy where they are not)."""
    if value is None:
        return None
    if value.is_contiguous():
        return value
    width = 1
    for k in range(1, inner + 1):
        if value.shape[-k] != 1 and value.stride(-k) != width:
            return value.contiguous()
        width *= value.shape[-k]
    return value


def _room(value: torch.Tensor) -> torch.Tensor:
    """A dense tensor of ``value``'s shape and type (the short way costs a third)."""
    if value.is_contiguous():
        return torch.empty_like(value)
    return torch.empty(value.shape, dtype=value.dtype, device=value.device)


def _check_signal(x, what: str, dims: int) -> None:
    if not isinstance(x, torch.Tensor) or x.dim() != dims:
        raise ValueError(f"{what} must be a {'[T, B, N]' if dims == 3 else '[B, N]'} tensor")
    if not x.is_cuda:
        raise ValueError(f"{what} must be on a GPU")
    if x.dtype not in TYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16")
    if x.shape[-1] == 0:
        raise ValueError(f"{what} has no channels")


def _check_like(value, what: str, shape: tuple, device: torch.device, dtype) -> None:
    if not isinstance(value, torch.Tensor) or value.shape != shape:
        raise ValueError(f"{what} must be a tensor of shape {list(shape)}")
    if value.device != device:
        raise ValueError(f"{what} must be on the signal's device")
    if value.dtype != dtype:
        raise ValueError(f"{what} must be {str(dtype).removeprefix('torch.')}")


def _lengths(lengths, x: torch.Tensor):
    if lengths is None:
        return None
    if (not isinstance(lengths, torch.Tensor) or lengths.dim() != 1
            or lengths.numel() != x.shape[1] or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError("lengths must be one int32 or int64 per column")
    if lengths.device != x.device:
        raise ValueError("lengths must be on the signal's device")
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, x.shape[0])
    return lengths.to(torch.int32).contiguous()


def _master(value: torch.Tensor | None):
    """Parameters as float32 (a cast that autograd follows where they are not)."""
    return value if value is None or value.dtype == torch.float32 else value.float()


def _dense(value: torch.Tensor | None):
    return value if value is None or value.is_contiguous() else value.contiguous()


def _moved_on(carried: torch.Tensor) -> None:
    """Tells autograd that a kernel has written ``carried`` in place: a backward that saved its
    earlier values then refuses.  Inference tensors keep no version."""
    if not carried.is_inference():
        increment_version(carried)


def _needs_grad(*values) -> bool:
    """Whether a backward has to be recorded.  Forward-mode derivatives, which no operator
    here gives, are refused: their tensors do not say that they require one."""
    if forward_ad._current_level >= 0:               # only then can a tensor carry one
        for value in values:
            if value is not None and forward_ad.unpack_dual(value).tangent is not None:
                raise ValueError("the signal operators give no forward-mode derivatives")
    if torch.is_grad_enabled():
        for value in values:
            if value is not None and value.requires_grad:
                return True
    return False


# ---- convolution ---------------------------------------------------------------------

_ACTIVATIONS = {None: 0, "silu": 1}


def _check_conv(x, weight, bias, history, activation, dims: int) -> None:
    _check_signal(x, "x", dims)
    shape, device = x.shape, x.device
    channels = shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] != channels:
        raise ValueError("weight must be a [N, W] tensor")
    taps = weight.shape[1]
    if not 1 <= taps <= MAX_TAPS:
        raise ValueError(f"a convolution has 1 to {MAX_TAPS} taps")
    if weight.device != device:
        raise ValueError("weight must be on the signal's device")
    if weight.dtype not in TYPES:
        raise ValueError("weight must be float32, bfloat16 or float16")
    if bias is not None:
        dtype = getattr(bias, "dtype", None)
        _check_like(bias, "bias", (channels,), device, dtype if dtype in TYPES else torch.float32)
    if history is not None:
        _check_like(history, "history", (taps - 1, shape[-2], channels), device, x.dtype)
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be 'silu' or None")


def _conv_forward(x, weight, bias, history, lengths, silu, chunk=0):
    """(y, last inputs) of dense operands."""
    ticks, batch, n = x.shape
    taps, device = weight.shape[1], x.device
    y = _room(x)
    last = torch.empty((taps - 1, batch, n), dtype=x.dtype, device=device)
    args = _CONV_FORWARD.pack(ticks, batch, n, taps, TYPES[x.dtype], silu, chunk, *_signal(x),
                              weight.data_ptr(), _address(bias), *_signal(history),
                              _address(lengths), *_signal(y), *_signal(last))
    call(_library().ns_conv_forward, device, args)
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, history, lengths, silu):
        operands = (_unit_channels(x), _dense(weight), _dense(bias), _unit_channels(history))
        ctx.save_for_backward(*operands, lengths)
        ctx.set_materialize_grads(False)
        ctx.silu = silu
        return _conv_forward(*operands, lengths, silu)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, history, lengths = ctx.saved_tensors
        wants, device = ctx.needs_input_grad, x.device
        (ticks, batch, channels), taps = x.shape, weight.shape[1]
        dy = torch.zeros_like(x) if dy is None else _unit_channels(dy)
        dlast = _unit_channels(dlast)
        dx = _room(x) if wants[0] else None
        dhistory = _room(history) if history is not None and wants[3] else None
        lib, count = _library(), channels * (taps + 1)
        parts = lib.ns_conv_backward_floats(ticks, batch, channels, taps, TYPES[x.dtype])
        # The parameters' gradients and the workspace share one allocation.
        sums = torch.empty(count + parts, dtype=torch.float32, device=device)
        args = _CONV.pack(ticks, batch, channels, taps, TYPES[x.dtype], ctx.silu, 0, *_signal(x),
                          weight.data_ptr(), _address(bias), *_signal(history), _address(lengths),
                          *_ABSENT, *_ABSENT, *_signal(dy), *_signal(dlast), *_signal(dx),
                          *_signal(dhistory), sums.data_ptr() + 4 * count, sums.data_ptr())
        call(lib.ns_conv_backward, device, args)
        return (dx, sums[:channels * taps].view(channels, taps) if wants[1] else None,
                sums[channels * taps:count] if bias is not None and wants[2] else None, dhistory,
                None, None)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                history: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                activation: str | None = "silu") -> tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution of every channel of ``x`` [T, B, N] with its own taps
    ``weight`` [N, W] (W up to 8; the last tap meets the current tick).

    ``history`` [W-1, B, N] holds the inputs before the first tick (zeros if absent).
    Returns ``(y, history)``: the outputs and the last W-1 inputs of every column, which
    carry the signal on.  ``activation`` is "silu" or None."""
    _check_conv(x, weight, bias, history, activation, 3)
    lengths, silu = _lengths(lengths, x), _ACTIVATIONS[activation]
    if _needs_grad(x, weight, bias, history):
        return _CausalConv.apply(x, _master(weight), _master(bias), history, lengths, silu)
    return _conv_forward(_unit_channels(x), _dense(_master(weight)), _dense(_master(bias)),
                         _unit_channels(history), lengths, silu)


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                     history: torch.Tensor, activation: str | None = "silu") -> torch.Tensor:
    """One tick of ``causal_conv``: ``x`` [B, N] to y [B, N], ``history`` [W-1, B, N]
    moved on by it in place.  Keeps nothing for gradients; a backward that saved the history
    as it was refuses."""
    _check_conv(x, weight, bias, history, activation, 2)
    if _needs_grad(x, weight, bias, history):
        raise ValueError("a step gives no gradients; use causal_conv")
    batch, n = x.shape
    taps = weight.shape[1]
    if history is None or (taps > 1 and not _own_elements(history)):
        raise ValueError("history must be a [W-1, B, N] tensor with dense channels, updated in place")
    if weight.dtype != torch.float32 or not weight.is_contiguous():
        weight = _dense(_master(weight))
    if bias is not None and (bias.dtype != torch.float32 or bias.stride(0) != 1):
        bias = _dense(_master(bias))
    if n > 1 and x.stride(1) != 1:
        x = x.contiguous()
    y = _room(x)
    carried = _signal(history)
    args = _CONV_FORWARD.pack(1, batch, n, taps, TYPES[x.dtype], _ACTIVATIONS[activation], 0,
                              x.data_ptr(), 0, x.stride(0), weight.data_ptr(), _address(bias),
                              *carried, 0, y.data_ptr(), 0, n, *carried)
    call(_library().ns_conv_step, x.device, args)
    _moved_on(history)
    return y


def _own_elements(value: torch.Tensor) -> bool:
    """Channels dense and no two elements the same memory."""
    if value.is_contiguous() or value.numel() == 0:
        return True
    rows, columns, n = value.shape
    if n > 1 and value.stride(2) != 1:
        return False
    near, far = sorted((s, c) for s, c in ((value.stride(0), rows), (value.stride(1), columns))
                       if c > 1)[:2] if rows > 1 and columns > 1 else ((n, 1), (n, 1))
    if rows > 1 and columns > 1:
        return near[0] >= n and far[0] >= near[0] * (near[1] - 1) + n
    single = value.stride(0) if rows > 1 else value.stride(1) if columns > 1 else n
    return single >= n


# ---- scan ----------------------------------------------------------------------------

def _check_scan(x, delta, A, B, C, D, z, delta_bias, state, dims: int) -> tuple[int, int]:
    """(groups, states) of valid operands."""
    _check_signal(x, "x", dims)
    *lead, channels = x.shape
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or A.shape[0] != channels:
        raise ValueError("A must be a [N, S] tensor")
    states = A.shape[1]
    if not 1 <= states <= MAX_STATES:
        raise ValueError(f"a channel has 1 to {MAX_STATES} states")
    if not isinstance(B, torch.Tensor) or B.dim() not in (dims, dims + 1):
        raise ValueError("B must be [T, B, S] or [T, B, G, S] (without T for a step)")
    grouped = B.dim() == dims + 1
    groups = B.shape[-2] if grouped else 1
    if groups == 0 or channels % groups:
        raise ValueError("the groups of B and C must divide the channels")
    device, dtype, full = x.device, x.dtype, (*lead, channels)
    shared = (*lead, groups, states) if grouped else (*lead, states)
    if delta is None or C is None:
        raise ValueError(f"{'delta' if delta is None else 'C'} is required")
    _check_like(delta, "delta", full, device, dtype)
    _check_like(B, "B", shared, device, dtype)
    _check_like(C, "C", shared, device, dtype)
    _check_like(A, "A", (channels, states), device, torch.float32)
    if z is not None:
        _check_like(z, "z", full, device, dtype)
    if D is not None:
        _check_like(D, "D", (channels,), device, torch.float32)
    if delta_bias is not None:
        _check_like(delta_bias, "delta_bias", (channels,), device, torch.float32)
    if state is not None:
        _check_like(state, "state", (lead[-1], channels, states), device, torch.float32)
    return groups, states


def _plan(shape, groups: int, states: int, backward: bool):
    """(chunks of time, floats of the chunk, checkpoint and partial workspaces)."""
    lib, sizes = _library(), _Sizes()
    code = lib.ns_scan_plan(*shape, groups, states, backward, ctypes.addressof(sizes))
    if code:
        _raise_on(code, lib)
    return sizes


def _dense_scan(x, delta, A, B, C, D, z, delta_bias):
    inner = 2 if B.dim() == x.dim() + 1 else 1
    return (_unit_channels(x), _unit_channels(delta), _dense(A), _unit_channels(B, inner),
            _unit_channels(C, inner), _dense(D), _unit_channels(z), _dense(delta_bias))


def _scan_forward(operands, state, lengths, softplus, groups, keep: bool):
    """(y, final state, checkpoints or None) of dense operands."""
    x, delta, A, B, C, D, z, delta_bias = operands
    ticks, batch, n = x.shape
    states, device = A.shape[1], x.device
    y = _room(x)
    final = torch.empty((batch, n, states), dtype=torch.float32, device=device)
    chunks, ends_floats, kept_floats, _ = _plan(x.shape, groups, states, False)
    ends = torch.empty(ends_floats, dtype=torch.float32, device=device) if ends_floats else None
    kept = torch.empty(kept_floats, dtype=torch.float32, device=device) if keep else None
    args = _SCAN_FORWARD.pack(
        ticks, batch, n, groups, states, TYPES[x.dtype], softplus, chunks, *_signal(x),
        *_signal(delta), *_signal(z), *_signal(y), *_signal(B), *_signal(C), A.data_ptr(),
        _address(D), _address(delta_bias), _address(state), final.data_ptr(), _address(lengths),
        _address(kept), _address(ends))
    call(_library().ns_scan_forward, device, args)
    return y, final, kept


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, state, lengths, softplus, groups):
        operands = _dense_scan(x, delta, A, B, C, D, z, delta_bias)
        y, final, kept = _scan_forward(operands, _dense(state), lengths, softplus, groups, True)
        ctx.save_for_backward(*operands, lengths, kept)
        ctx.set_materialize_grads(False)
        ctx.softplus, ctx.groups = softplus, groups
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        *operands, lengths, kept = ctx.saved_tensors
        x, delta, A, B, C, D, z, delta_bias = operands
        wants, device = ctx.needs_input_grad, x.device
        ticks, batch, n = x.shape
        dfinal, states = _dense(dfinal), A.shape[1]
        if ticks == 0 or batch == 0:                  # no tick: the state passes through
            zeros = [torch.zeros_like(v) if v is not None and w else None
                     for v, w in zip(operands, wants)]
            return (*zeros, dfinal if wants[8] else None, None, None, None)
        dy = torch.zeros_like(x) if dy is None else _unit_channels(dy)
        chunks, ends_floats, _, part_floats = _plan(x.shape, ctx.groups, states, True)

        dx, ddelta, dB, dC = _room(x), _room(delta), _room(B), _room(C)
        dz = None if z is None else _room(z)
        dstate = (torch.empty((batch, n, states), dtype=torch.float32, device=device)
                  if wants[8] else None)
        # The parameters' gradients and the workspaces share one allocation.
        sums = torch.empty(n * (states + 2), dtype=torch.float32, device=device)
        work = torch.empty(part_floats + ends_floats, dtype=torch.float32, device=device)
        args = _SCAN.pack(
            ticks, batch, n, ctx.groups, states, TYPES[x.dtype], ctx.softplus, chunks,
            *_signal(x), *_signal(delta), *_signal(z), *_ABSENT, *_signal(B), *_signal(C),
            A.data_ptr(), _address(D), _address(delta_bias), 0, 0, _address(lengths),
            kept.data_ptr(), work.data_ptr() + 4 * part_floats if ends_floats else 0,
            *_signal(dy), _address(dfinal), *_signal(dx), *_signal(ddelta), *_signal(dz),
            *_signal(dB), *_signal(dC), _address(dstate), sums.data_ptr(), work.data_ptr())
        call(_library().ns_scan_backward, device, args)
        grads = (dx, ddelta, sums[:n * states].view(n, states), dB, dC,
                 sums[n * states:n * (states + 1)] if D is not None else None, dz,
                 sums[n * (states + 1):] if delta_bias is not None else None, dstate)
        return (*(g if w else None for g, w in zip(grads, wants)), None, None, None)


def selective_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                   C: torch.Tensor, D: torch.Tensor | None = None, *,
                   z: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None,
                   softplus: bool = True, state: torch.Tensor | None = None,
                   lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Selective state space scan of ``x`` [T, B, N] with S states per channel (up to 64).

    ``delta`` and the optional gate ``z`` are [T, B, N]; ``A`` [N, S] (negative rates decay),
    ``D`` [N] and ``delta_bias`` [N] are float32; ``B`` and ``C`` are [T, B, S], shared by all
    channels, or [T, B, G, S], each shared by N/G neighbouring channels.  ``state``
    [B, N, S] float32 is h before the first tick (zeros if absent).  With
    ``softplus=False`` the time step is ``delta + delta_bias`` itself.

    Returns ``(y, state)``: y [T, B, N] of x's type and h after each column's last tick."""
    groups, _ = _check_scan(x, delta, A, B, C, D, z, delta_bias, state, 3)
    lengths = _lengths(lengths, x)
    if _needs_grad(x, delta, A, B, C, D, z, delta_bias, state):
        return _SelectiveScan.apply(x, delta, A, B, C, D, z, delta_bias, state, lengths,
                                    bool(softplus), groups)
    y, final, _ = _scan_forward(_dense_scan(x, delta, A, B, C, D, z, delta_bias), _dense(state),
                                lengths, softplus, groups, False)
    return y, final


def selective_scan_step(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: torch.Tensor | None = None, *,
                        z: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None,
                        softplus: bool = True, state: torch.Tensor) -> torch.Tensor:
    """One tick of ``selective_scan``: ``x``, ``delta``, ``z`` [B, N], ``B`` and ``C`` [B, S]
    or [B, G, S], y [B, N]; ``state`` [B, N, S] (float32, contiguous) is updated in place.
    Keeps nothing for gradients; a backward that saved the state as it was refuses."""
    groups, states = _check_scan(x, delta, A, B, C, D, z, delta_bias, state, 2)
    if _needs_grad(x, delta, A, B, C, D, z, delta_bias, state):
        raise ValueError("a step gives no gradients; use selective_scan")
    if state is None or not state.is_contiguous():
        raise ValueError("state must be a contiguous [B, N, S] tensor, updated in place")
    x, delta, A, B, C, D, z, delta_bias = _dense_scan(x, delta, A, B, C, D, z, delta_bias)
    batch, n = x.shape
    y = _room(x)
    args = _SCAN_FORWARD.pack(
        1, batch, n, groups, states, TYPES[x.dtype], softplus, 1, x.data_ptr(), 0, x.stride(0),
        delta.data_ptr(), 0, delta.stride(0),
        *(_ABSENT if z is None else (z.data_ptr(), 0, z.stride(0))), y.data_ptr(), 0, n,
        B.data_ptr(), 0, B.stride(0), C.data_ptr(), 0, C.stride(0), A.data_ptr(), _address(D),
        _address(delta_bias), state.data_ptr(), state.data_ptr(), 0, 0, 0)
    call(_library().ns_scan_step, x.device, args)
    _moved_on(state)
    return y
