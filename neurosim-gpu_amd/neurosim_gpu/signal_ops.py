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
native gradients of every tensor input, and have a one-tick form that updates the carried
state in place.  ``lengths`` gives columns their own number of ticks: past it outputs and
gradients are zero, the carried state stays that of the column's last tick, and what the
inputs hold there is never used.  The kernels are csrc/conv.hip, scan.hip, scan_grad.hip
behind include/neurosim_hip_signal.h; calls run on the current stream, allocate their
outputs and workspaces from torch, and never synchronise.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from .native import _raise_on, load_library

MAX_TAPS, MAX_STATES = 8, 64         # NS_CONV_MAX_TAPS, NS_SCAN_MAX_STATES
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # NS_TYPE_*

_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class _Signal(ctypes.Structure):
    _fields_ = [("data", _ptr), ("stride_t", _i64), ("stride_b", _i64)]


class _ConvArgs(ctypes.Structure):
    _fields_ = [("ticks", _i64), ("batch", _i64), ("channels", _i64), ("taps", _i32),
                ("type", _i32), ("silu", _i32), ("chunk", _i32), ("x", _Signal),
                ("weight", _ptr), ("bias", _ptr), ("history", _Signal), ("lengths", _ptr),
                ("y", _Signal), ("out_history", _Signal), ("dy", _Signal),
                ("dout_history", _Signal), ("dx", _Signal), ("dhistory", _Signal),
                ("partials", _ptr), ("dweight", _ptr)]


class _ScanArgs(ctypes.Structure):
    _fields_ = [("ticks", _i64), ("batch", _i64), ("channels", _i64), ("groups", _i64),
                ("states", _i32), ("type", _i32), ("softplus", _i32), ("chunks", _i32),
                ("x", _Signal), ("delta", _Signal), ("z", _Signal), ("y", _Signal),
                ("write", _Signal), ("read", _Signal), ("rates", _ptr), ("skip", _ptr),
                ("delta_bias", _ptr), ("state", _ptr), ("out_state", _ptr), ("lengths", _ptr),
                ("checkpoints", _ptr), ("ends", _ptr), ("dy", _Signal), ("dout_state", _ptr),
                ("dx", _Signal), ("ddelta", _Signal), ("dz", _Signal), ("dwrite", _Signal),
                ("dread", _Signal), ("dstate", _ptr), ("drates", _ptr), ("dskip", _ptr),
                ("ddelta_bias", _ptr), ("partials", _ptr)]


@lru_cache(maxsize=1)
def _library() -> ctypes.CDLL:
    lib = load_library()
    for name, kind in (("ns_conv_forward", _ConvArgs), ("ns_conv_step", _ConvArgs),
                       ("ns_conv_backward", _ConvArgs), ("ns_scan_forward", _ScanArgs),
                       ("ns_scan_step", _ScanArgs), ("ns_scan_backward", _ScanArgs)):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = ctypes.c_int, [ctypes.POINTER(kind), _ptr]
    for name, kind in (("ns_conv_backward_floats", _ConvArgs),
                       ("ns_scan_checkpoint_floats", _ScanArgs),
                       ("ns_scan_chunk_floats", _ScanArgs),
                       ("ns_scan_backward_floats", _ScanArgs)):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _i64, [ctypes.POINTER(kind)]
    lib.ns_conv_chunk.restype = _i64
    lib.ns_conv_chunk.argtypes = [_i64, _i64, _i64, _i32, _i32]
    lib.ns_scan_chunks.restype = _i32
    lib.ns_scan_chunks.argtypes = [_i64, _i64, _i64, _i64, _i32, _i32]
    return lib


def on_device(device: torch.device):
    """A guard that makes ``device`` current where it is not."""
    if device.index is None or device.index == torch.cuda.current_device():
        return nullcontext()
    return torch.cuda.device(device)


def _call(name: str, args, device: torch.device) -> None:
    lib = _library()
    with on_device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        _raise_on(getattr(lib, name)(ctypes.byref(args), stream), lib)


def _floats(name: str, args, device: torch.device):
    """A workspace of the size ``name`` gives (None: none needed)."""
    lib = _library()
    count = getattr(lib, name)(ctypes.byref(args))
    if count < 0:
        _raise_on(1, lib)
    return torch.empty(count, dtype=torch.float32, device=device) if count else None


def _address(value: torch.Tensor | None):
    return None if value is None or value.numel() == 0 else value.data_ptr()


def _signal(value: torch.Tensor | None) -> _Signal:
    if value is None or value.numel() == 0:
        return _Signal(None, 0, 0)
    return _Signal(value.data_ptr(), value.stride(0), value.stride(1))


def _unit_channels(value: torch.Tensor | None, inner: int = 1):
    """``value`` with its last ``inner`` dimensions dense (a copy where they are not)."""
    if value is None:
        return None
    width = 1
    for k in range(1, inner + 1):
        if value.shape[-k] != 1 and value.stride(-k) != width:
            return value.contiguous()
        width *= value.shape[-k]
    return value


def _check_signal(x, what: str, dims: int) -> None:
    if not isinstance(x, torch.Tensor) or x.dim() != dims:
        raise ValueError(f"{what} must be a {'[T, B, N]' if dims == 3 else '[B, N]'} tensor")
    if x.device.type != "cuda":
        raise ValueError(f"{what} must be on a GPU")
    if x.dtype not in TYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16")
    if x.shape[-1] == 0:
        raise ValueError(f"{what} has no channels")


def _check_like(value, like: torch.Tensor, shape, what: str, dtype=None) -> None:
    if value is None:
        return
    if not isinstance(value, torch.Tensor) or tuple(value.shape) != tuple(shape):
        raise ValueError(f"{what} must be a tensor of shape {list(shape)}")
    if value.device != like.device:
        raise ValueError(f"{what} must be on the signal's device")
    dtype = dtype or like.dtype
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
    return None if value is None else value.detach().contiguous()


def _needs_grad(*values) -> bool:
    return torch.is_grad_enabled() and any(v is not None and v.requires_grad for v in values)


# ---- convolution ---------------------------------------------------------------------

_ACTIVATIONS = {None: 0, "silu": 1}


def _check_conv(x, weight, bias, history, activation, dims: int) -> None:
    _check_signal(x, "x", dims)
    channels = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] != channels:
        raise ValueError("weight must be a [N, W] tensor")
    if not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"a convolution has 1 to {MAX_TAPS} taps")
    for value, what, shape in ((weight, "weight", weight.shape), (bias, "bias", (channels,))):
        _check_like(value, x, shape, what, dtype=getattr(value, "dtype", None))
        if value is not None and value.dtype not in TYPES:
            raise ValueError(f"{what} must be float32, bfloat16 or float16")
    _check_like(history, x, (weight.shape[1] - 1, x.shape[-2], channels), "history")
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be 'silu' or None")


def _conv_args(x, weight, bias, history, lengths, silu) -> _ConvArgs:
    args = _ConvArgs(*x.shape, weight.shape[1], TYPES[x.dtype], silu)
    args.x, args.history = _signal(x), _signal(history)
    args.weight, args.bias = _address(weight), _address(bias)
    args.lengths = _address(lengths)
    return args


def _conv_forward(x, weight, bias, history, lengths, silu):
    """(y, last inputs) of detached dense operands."""
    args = _conv_args(x, weight, bias, history, lengths, silu)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    last = torch.empty((weight.shape[1] - 1, *x.shape[1:]), dtype=x.dtype, device=x.device)
    args.y, args.out_history = _signal(y), _signal(last)
    _call("ns_conv_forward", args, x.device)
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, history, lengths, silu):
        operands = (_unit_channels(x), _dense(weight), _dense(bias), _unit_channels(history))
        ctx.save_for_backward(*operands, lengths)
        ctx.silu = silu
        return _conv_forward(*operands, lengths, silu)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, history, lengths = ctx.saved_tensors
        wants = ctx.needs_input_grad
        channels, taps = weight.shape
        args = _conv_args(x, weight, bias, history, lengths, ctx.silu)
        dy, dlast = _unit_channels(dy), _unit_channels(dlast)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if wants[0] else None
        dhistory = (torch.empty(history.shape, dtype=x.dtype, device=x.device)
                    if history is not None and wants[3] else None)
        sums = torch.empty(channels * (taps + 1), dtype=torch.float32, device=x.device)
        partials = _floats("ns_conv_backward_floats", args, x.device)
        args.dy, args.dout_history = _signal(dy), _signal(dlast)
        args.dx, args.dhistory = _signal(dx), _signal(dhistory)
        args.partials, args.dweight = _address(partials), sums.data_ptr()
        _call("ns_conv_backward", args, x.device)
        return (dx, sums[:channels * taps].view(channels, taps) if wants[1] else None,
                sums[channels * taps:] if bias is not None and wants[2] else None, dhistory,
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
    moved on by it in place.  Keeps nothing for gradients."""
    _check_conv(x, weight, bias, history, activation, 2)
    if _needs_grad(x, weight, bias, history):
        raise ValueError("a step gives no gradients; use causal_conv")
    if history is None or (weight.shape[1] > 1 and not _own_elements(history)):
        raise ValueError("history must be a [W-1, B, N] tensor with dense channels, updated in place")
    weight, bias, x = _dense(_master(weight)), _dense(_master(bias)), _unit_channels(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    args = _conv_args(x.unsqueeze(0), weight, bias, history, None, _ACTIVATIONS[activation])
    args.out_history, args.y = args.history, _signal(y.unsqueeze(0))
    _call("ns_conv_step", args, x.device)
    return y


def _own_elements(value: torch.Tensor) -> bool:
    """Channels dense and no two elements the same memory."""
    rows, columns, n = value.shape
    if value.numel() == 0:
        return True
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
    lead, channels = tuple(x.shape[:-1]), x.shape[-1]
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or A.shape[0] != channels:
        raise ValueError("A must be a [N, S] tensor")
    states = A.shape[1]
    if not 1 <= states <= MAX_STATES:
        raise ValueError(f"a channel has 1 to {MAX_STATES} states")
    if not isinstance(B, torch.Tensor) or B.dim() not in (dims, dims + 1):
        raise ValueError("B must be [T, B, S] or [T, B, G, S] (without T for a step)")
    groups = B.shape[-2] if B.dim() == dims + 1 else 1
    if groups == 0 or channels % groups:
        raise ValueError("the groups of B and C must divide the channels")
    shared = (*lead, groups, states) if B.dim() == dims + 1 else (*lead, states)
    for value, what, shape, dtype in (
            (delta, "delta", x.shape, x.dtype), (z, "z", x.shape, x.dtype),
            (B, "B", shared, x.dtype), (C, "C", shared, x.dtype),
            (A, "A", A.shape, torch.float32), (D, "D", (channels,), torch.float32),
            (delta_bias, "delta_bias", (channels,), torch.float32),
            (state, "state", (x.shape[-2], channels, states), torch.float32)):
        if value is None and what in ("delta", "C"):
            raise ValueError(f"{what} is required")
        _check_like(value, x, shape, what, dtype=dtype)
    return groups, states


def _scan_args(x, delta, A, B, C, D, z, delta_bias, lengths, softplus, groups) -> _ScanArgs:
    args = _ScanArgs(*x.shape, groups, A.shape[1], TYPES[x.dtype], int(softplus), 1)
    args.x, args.delta, args.z = _signal(x), _signal(delta), _signal(z)
    args.write, args.read = _signal(B), _signal(C)
    args.rates, args.skip, args.delta_bias = _address(A), _address(D), _address(delta_bias)
    args.lengths = _address(lengths)
    return args


def _chunks(args: _ScanArgs, backward: bool) -> int:
    return _library().ns_scan_chunks(args.ticks, args.batch, args.channels, args.groups,
                                     args.states, int(backward))


def _dense_scan(x, delta, A, B, C, D, z, delta_bias):
    inner = 2 if B.dim() == x.dim() + 1 else 1
    return (_unit_channels(x), _unit_channels(delta), _dense(A), _unit_channels(B, inner),
            _unit_channels(C, inner), _dense(D), _unit_channels(z), _dense(delta_bias))


def _scan_forward(operands, state, lengths, softplus, groups, keep: bool):
    """(y, final state, checkpoints or None) of dense operands."""
    x, A = operands[0], operands[2]
    args = _scan_args(*operands, lengths, softplus, groups)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    final = torch.empty((x.shape[1], *A.shape), dtype=torch.float32, device=x.device)
    args.y, args.state, args.out_state = _signal(y), _address(state), _address(final)
    args.chunks = _chunks(args, False)
    ends = _floats("ns_scan_chunk_floats", args, x.device)
    checkpoints = _floats("ns_scan_checkpoint_floats", args, x.device) if keep else None
    args.ends, args.checkpoints = _address(ends), _address(checkpoints)
    _call("ns_scan_forward", args, x.device)
    return y, final, checkpoints


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, state, lengths, softplus, groups):
        operands = _dense_scan(x, delta, A, B, C, D, z, delta_bias)
        start = _dense(state)
        y, final, checkpoints = _scan_forward(operands, start, lengths, softplus, groups, True)
        ctx.save_for_backward(*operands, lengths, checkpoints)
        ctx.softplus, ctx.groups = softplus, groups
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        *operands, lengths, checkpoints = ctx.saved_tensors
        x, delta, A, B, C, D, z, delta_bias = operands
        wants = ctx.needs_input_grad
        dfinal = dfinal.contiguous()
        if x.shape[0] == 0 or x.shape[1] == 0:        # no tick: the state passes through
            zeros = [torch.zeros_like(v) if v is not None and w else None
                     for v, w in zip(operands, wants)]
            return (*zeros, dfinal if wants[8] else None, None, None, None)
        args = _scan_args(*operands, lengths, ctx.softplus, ctx.groups)
        dy = _unit_channels(dy)

        def like(value):
            return None if value is None else torch.empty(value.shape, dtype=value.dtype,
                                                          device=x.device)

        dx, ddelta, dz, dB, dC, dA = (like(v) for v in (x, delta, z, B, C, A))
        dskip, dbias = (torch.empty(x.shape[2], dtype=torch.float32, device=x.device)
                        for _ in range(2))
        dstate = torch.empty_like(dfinal) if wants[8] else None
        args.dy, args.dout_state = _signal(dy), _address(dfinal)
        args.dx, args.ddelta, args.dz = _signal(dx), _signal(ddelta), _signal(dz)
        args.dwrite, args.dread, args.dstate = _signal(dB), _signal(dC), _address(dstate)
        args.drates, args.dskip, args.ddelta_bias = (dA.data_ptr(), dskip.data_ptr(),
                                                     dbias.data_ptr())
        args.chunks = _chunks(args, True)
        ends = _floats("ns_scan_chunk_floats", args, x.device)
        partials = _floats("ns_scan_backward_floats", args, x.device)
        args.ends, args.partials = _address(ends), _address(partials)
        args.checkpoints = checkpoints.data_ptr()
        _call("ns_scan_backward", args, x.device)
        grads = (dx, ddelta, dA, dB, dC, dskip if D is not None else None, dz,
                 dbias if delta_bias is not None else None, dstate)
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
    Keeps nothing for gradients."""
    groups, _ = _check_scan(x, delta, A, B, C, D, z, delta_bias, state, 2)
    if _needs_grad(x, delta, A, B, C, D, z, delta_bias, state):
        raise ValueError("a step gives no gradients; use selective_scan")
    if state is None or not state.is_contiguous():
        raise ValueError("state must be a contiguous [B, N, S] tensor, updated in place")
    operands = _dense_scan(x, delta, A, B, C, D, z, delta_bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ticked = [v if i in (2, 5, 7) or v is None else v.unsqueeze(0) for i, v in enumerate(operands)]
    args = _scan_args(*ticked, None, softplus, groups)
    args.state = args.out_state = _address(state)
    args.y = _signal(y.unsqueeze(0))
    _call("ns_scan_step", args, x.device)
    return y
