"""Causal convolution and selective scan against float64 formulas (MI355X).

Tolerances.  A result is a sum of terms, each a product along a path through the ticks.
With u = 2^-24, a float32 operation adds a relative error of at most u to what it
computes, hardware exp2, log and reciprocal at most 2u (1 ulp), so a term that passes p
operations is off by at most about p u times its size, and a result by (p + its summands)
u times the sum of its terms' sizes, which the oracle gives (``magnitude=True``).  Per
tick a state passes the decay (its exponent dt A carries the errors of dt, at most 12u,
and of two products, times |dt A|, then exp2: in these tests |dt A| <= 4, so at most
62u), a multiply-add and the input's two products: at most 70.  Outputs are then rounded
once to their type.
"""

from __future__ import annotations

import math

import pytest
import torch

import signal_oracle as so
from neurosim_gpu import causal_conv, causal_conv_step, selective_scan, selective_scan_step
from neurosim_gpu import signal_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, want, size, operations: int, what: str):
    assert got.shape == want.shape, what
    error = (got.detach().double().cpu() - want).abs()
    bound = operations * U * size
    bound = bound + HALF_ULP[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    assert torch.isfinite(got).all(), what
    worst = float((error / bound).max()) if error.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of its bound"


class Draw:
    def __init__(self, gpu, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.gpu = gpu

    def __call__(self, *shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g) * scale).to(dtype).to(self.gpu)


def leaves(operands: dict) -> dict:
    return {k: None if v is None else v.detach().clone().requires_grad_()
            for k, v in operands.items()}


def gradients(outs, inputs: dict, ups) -> dict:
    named = {k: v for k, v in inputs.items() if v is not None}
    got = torch.autograd.grad(outs, list(named.values()), ups, allow_unused=True)
    return {k: v for k, v in zip(named, got) if v is not None}


# ---- convolution ---------------------------------------------------------------------

CONV_SHAPES = [  # T, B, N, W
    (1, 1, 1, 1), (1, 2, 3, 4), (2, 1, 7, 4), (3, 1, 8, 8), (37, 3, 5, 8), (40, 2, 64, 4),
    (70, 1, 129, 3), (150, 2, 33, 2), (64, 5, 16, 5), (130, 1, 24, 6), (9, 2, 40, 7),
]


def conv_operands(draw, T, B, N, W, dtype, bias=True, history=True):
    return {"x": draw(T, B, N, dtype=dtype), "weight": draw(N, W),
            "bias": draw(N) if bias else None,
            "history": draw(W - 1, B, N, dtype=dtype) if history else None}


def check_conv(operands, lengths, activation, dy=None, dlast=None):
    x, W = operands["x"], operands["weight"].shape[1]
    T, B, N = x.shape
    inputs = leaves(operands) if dy is not None else operands
    y, last = causal_conv(**inputs, lengths=lengths, activation=activation)
    kw = dict(lengths=lengths, activation=activation, dy=dy, dlast=dlast)
    want, grads = so.conv(**operands, **kw)
    size, grad_size = so.conv(**operands, **kw, magnitude=True)
    # p: W products and adds; silu: exponent, exp2, add, reciprocal, product (at most 12).
    close(y, want["y"], size["y"], W + 14, "y")
    assert torch.equal(last.detach().double().cpu(), want["history"])
    if dy is None:
        return
    got = gradients((y, last), inputs, (dy, dlast))
    # q: pre (W) and the slope's operations (at most 20); then W more, or a sum over ticks.
    for name, value in got.items():
        summands = T * B if name in ("weight", "bias") else W + 1
        close(value, grads[name], grad_size[name], W + 24 + summands, f"d{name}")
    assert set(got) == {k for k, v in operands.items() if v is not None}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", CONV_SHAPES)
def test_conv(gpu, shape, dtype):
    draw = Draw(gpu, sum(shape))
    operands = conv_operands(draw, *shape, dtype, bias=shape[0] % 2 == 1, history=shape[1] != 2)
    dy = draw(*shape[:3], dtype=dtype)
    dlast = draw(shape[3] - 1, *shape[1:3], dtype=dtype)
    check_conv(operands, None, "silu" if shape[2] != 64 else None, dy, dlast)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_conv_lengths(gpu, kind):
    """Columns of 0, 1, fewer than W, some, all and claimed more ticks; what stands past a
    column's end, in the inputs and in the gradient of y, is infinite or not a number."""
    draw, T, W = Draw(gpu, 5), 50, 5
    ends = [0, 1, 3, 20, T, T + 9, -4]
    operands = conv_operands(draw, T, len(ends), 11, W, torch.float32)
    dy, dlast = draw(T, len(ends), 11), draw(W - 1, len(ends), 11)
    for b, end in enumerate(so.ends_of(torch.tensor(ends), T, len(ends))):
        operands["x"][end:, b] = float("nan")
        dy[end:, b] = float("inf")
    lengths = torch.tensor(ends, dtype=kind, device=gpu)
    check_conv(operands, lengths, "silu", dy, dlast)


@pytest.mark.parametrize("shape", [(0, 3, 5, 4), (4, 0, 5, 4)])
def test_conv_without_ticks_or_columns(gpu, shape):
    draw = Draw(gpu, 1)
    operands = conv_operands(draw, *shape, torch.float32)
    check_conv(operands, None, "silu", draw(*shape[:3]), draw(shape[3] - 1, *shape[1:3]))


@pytest.mark.parametrize("dtype", TYPES)
def test_conv_views(gpu, dtype):
    """Batch-first signals, channel slices off every alignment, broadcast columns, and an
    output gradient that is one number, read as they are."""
    draw = Draw(gpu, 6)
    T, B, N, W = 21, 3, 18, 4
    first = draw(B, T, N + 5, dtype=dtype)
    for x in (first.transpose(0, 1)[..., 1:1 + N], first.transpose(0, 1)[..., 3:3 + N],
              draw(T, 1, N, dtype=dtype).expand(T, B, N), draw(N, T, B, dtype=dtype).permute(1, 2, 0)):
        weight, bias = draw(W, N).t(), draw(2 * N)[::2]
        leaf = x.detach().requires_grad_()
        y, last = causal_conv(leaf, weight, bias)
        want, grads = so.conv(x, weight, bias, dy=torch.ones(T, B, N))
        size, grad_size = so.conv(x, weight, bias, dy=torch.ones(T, B, N), magnitude=True)
        close(y, want["y"], size["y"], W + 14, "y")
        (dx,) = torch.autograd.grad(y.sum(), leaf)
        close(dx, grads["x"], grad_size["x"], 2 * W + 25, "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("W", [1, 2, 4, 8])
def test_conv_steps_are_the_signal(gpu, dtype, W):
    """Ticks one by one, and a signal in two parts, give the whole signal's bits."""
    draw, T = Draw(gpu, 7 + W), 12
    operands = conv_operands(draw, T, 3, 37, W, dtype)
    whole, last = causal_conv(**operands)
    first, carried = causal_conv(operands["x"][:5], operands["weight"], operands["bias"],
                                 history=operands["history"])
    second, carried = causal_conv(operands["x"][5:], operands["weight"], operands["bias"],
                                  history=carried)
    assert torch.equal(torch.cat((first, second)), whole) and torch.equal(carried, last)
    history = operands["history"].clone()
    for t in range(T):
        y = causal_conv_step(operands["x"][t], operands["weight"], operands["bias"], history=history)
        assert torch.equal(y, whole[t]), t
    assert torch.equal(history, last)


def test_conv_chunks_do_not_change_results(gpu):
    """Ticks per thread are a matter of speed: outputs are the same bits for any."""
    draw = Draw(gpu, 8)
    operands = conv_operands(draw, 90, 2, 20, 4, torch.float32)
    want, last = causal_conv(**operands)
    for chunk in (1, 4, 7, 90, 1000):
        y, history = signal_ops._conv_forward(operands["x"], operands["weight"], operands["bias"],
                                              operands["history"], None, 1, chunk)
        assert torch.equal(y, want) and torch.equal(history, last), chunk


# ---- scan ----------------------------------------------------------------------------

SCAN_SHAPES = [  # T, B, N, S, G
    (1, 1, 1, 1, 1), (1, 3, 5, 4, 1), (2, 1, 64, 16, 1), (16, 1, 64, 16, 1), (17, 2, 65, 16, 1),
    (33, 2, 66, 7, 3), (20, 1, 130, 8, 2), (40, 1, 12, 13, 12), (19, 2, 10, 24, 1), (9, 1, 70, 64, 1),
    (70, 1, 6, 3, 2), (35, 1, 64, 2, 1), (13, 2, 9, 33, 3),
]


def scan_operands(draw, T, B, N, S, G, dtype, optional=True, flat=False):
    shared = (T, B, S) if flat else (T, B, G, S)
    return {"x": draw(T, B, N, dtype=dtype), "delta": draw(T, B, N, scale=0.4, dtype=dtype),
            "A": -draw(N, S).abs().clamp(max=2) - 0.05, "B": draw(*shared, dtype=dtype),
            "C": draw(*shared, dtype=dtype), "D": draw(N) if optional else None,
            "z": draw(T, B, N, dtype=dtype) if optional else None,
            "delta_bias": draw(N, scale=0.5) - 1 if optional else None,
            "state": draw(B, N, S) if optional else None}


def check_scan(operands, lengths=None, softplus=True, dy=None, dfinal=None):
    T, B, N = operands["x"].shape
    S, G = operands["A"].shape[1], 1 if operands["B"].dim() == 3 else operands["B"].shape[2]
    inputs = leaves(operands) if dy is not None else operands
    y, final = selective_scan(**inputs, softplus=softplus, lengths=lengths)
    kw = dict(soft=softplus, lengths=lengths, dy=dy, dfinal=dfinal)
    want, grads = so.scan(**operands, **kw)
    size, grad_size = so.scan(**operands, **kw, magnitude=True)
    path = 70 * T + 20                    # the state's; then the read-out's sum and the gate
    close(y, want["y"], size["y"], path + S + 30, "y")
    close(final, want["state"], size["state"], path, "state")
    if dy is None:
        return
    got = gradients((y, final), inputs, (dy, dfinal))
    assert set(got) == {k for k, v in operands.items() if v is not None}
    for name, value in got.items():
        # Down the ticks and back, the gate and the slopes, then the sums the name says.
        summands = {"A": T * B, "D": T * B, "delta_bias": T * B, "B": N // G, "C": N // G}
        close(value, grads[name], grad_size[name], 2 * path + S + 60 + summands.get(name, 0),
              f"d{name}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SCAN_SHAPES)
def test_scan(gpu, shape, dtype):
    draw = Draw(gpu, sum(shape))
    T, B, N, S, G = shape
    operands = scan_operands(draw, *shape, dtype, optional=T != 20, flat=G == 1 and T % 2 == 1)
    softplus = T != 35
    if not softplus:      # time steps as given; negative ones would grow past float32's range
        operands["delta"], operands["delta_bias"] = operands["delta"].abs(), draw(N).abs() * 0.1
    check_scan(operands, None, softplus, draw(T, B, N, dtype=dtype), draw(B, N, S))


@pytest.mark.parametrize("S", [3, 16, 40])
def test_scan_lengths(gpu, S):
    """As the convolution's: columns of their own length, not-a-number past their end."""
    draw, T = Draw(gpu, 50 + S), 37
    ends = [0, 1, 15, 16, 17, T, T + 5, -1]
    operands = scan_operands(draw, T, len(ends), 6, S, 2, torch.float32)
    dy, dfinal = draw(T, len(ends), 6), draw(len(ends), 6, S)
    for b, end in enumerate(so.ends_of(torch.tensor(ends), T, len(ends))):
        for name in ("x", "delta", "z", "B", "C"):
            operands[name][end:, b] = float("nan") if name != "x" else float("inf")
        dy[end:, b] = float("nan")
    clean = {k: v.clone() for k, v in operands.items()}
    lengths = torch.tensor(ends, dtype=torch.int32, device=gpu)
    for b, end in enumerate(so.ends_of(lengths, T, len(ends))):
        for name in ("x", "delta", "z", "B", "C"):
            clean[name][end:, b] = 0
    inputs = leaves(operands)
    y, final = selective_scan(**inputs, lengths=lengths)
    got = gradients((y, final), inputs, (dy, dfinal))
    kw = dict(lengths=lengths, dy=torch.nan_to_num(dy), dfinal=dfinal)
    want, grads = so.scan(**clean, **kw)
    size, grad_size = so.scan(**clean, **kw, magnitude=True)
    path = 70 * T + 20
    close(y, want["y"], size["y"], path + S + 30, "y")
    close(final, want["state"], size["state"], path, "state")
    for name, value in got.items():
        close(value, grads[name], grad_size[name], 2 * path + S + 60 + T * len(ends), f"d{name}")


@pytest.mark.parametrize("S", [4, 16, 32])
@pytest.mark.parametrize("ragged", [False, True])
def test_scan_in_chunks_of_time(gpu, S, ragged):
    """A long signal of few channels: time is cut into chunks scanned side by side."""
    draw, T, B, N = Draw(gpu, 60 + S), 260, 2, 5
    assert signal_ops._plan((T, B, N), 1, S, False)[0] > 1
    assert signal_ops._plan((T, B, N), 1, S, True)[0] > 1
    operands = scan_operands(draw, T, B, N, S, 1, torch.float32)
    lengths = torch.tensor([T, 100], device=gpu) if ragged else None
    check_scan(operands, lengths, True, draw(T, B, N), draw(B, N, S))


def test_scan_strong_decay_and_large_steps(gpu):
    """Decays that underflow to zero, growth (positive rates), and steps far into softplus."""
    draw, T, N, S = Draw(gpu, 9), 20, 10, 4
    operands = scan_operands(draw, T, 1, N, S, 1, torch.float32)
    operands["A"] = operands["A"] * 200
    operands["delta"] = operands["delta"] * 100          # raw steps to about +-100
    y, final = selective_scan(**operands)
    want, _ = so.scan(**operands)
    size, _ = so.scan(**operands, magnitude=True)
    # A decay exp(dt A) that matters has |dt A| < 20; beyond, terms are below 2e-9 of their
    # size and enter with an absolute error as small.
    for got, name in ((y, "y"), (final, "state")):
        error = (got.double().cpu() - want[name]).abs()
        assert (error <= size[name] * U * (20 * 16 + 40) * 3 + 1e-30).all(), name
    operands["A"] = draw(N, S).abs() * 0.1               # growth
    operands["delta"] = operands["delta"] / 100
    check_scan(operands)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,G", [(1, 1), (5, 3), (16, 1), (64, 2)])
def test_scan_steps_are_the_signal(gpu, dtype, S, G):
    """Ticks one by one, and a signal in two parts carried by its state, against the whole."""
    draw, T, B, N = Draw(gpu, 11 + S), 20, 3, 66
    operands = scan_operands(draw, T, B, N, S, G, dtype)
    whole, last = selective_scan(**operands)
    want, _ = so.scan(**operands)
    size, _ = so.scan(**operands, magnitude=True)
    signals = ("x", "delta", "z", "B", "C")

    def part(ticks, state):
        return selective_scan(**{k: v[ticks] if k in signals else v for k, v in operands.items()
                                 if k != "state"}, state=state)

    first, carried = part(slice(0, 7), operands["state"])
    second, carried = part(slice(7, T), carried)
    path = 70 * T + 20
    close(torch.cat((first, second)), want["y"], size["y"], path + S + 30, "two parts")
    close(carried, want["state"], size["state"], path, "state of two parts")
    state = operands["state"].clone()
    steps = []
    for t in range(T):
        steps.append(selective_scan_step(**{k: v[t] if k in signals else v
                                            for k, v in operands.items() if k != "state"},
                                         state=state))
    close(torch.stack(steps), want["y"], size["y"], path + S + 30, "steps")
    close(state, want["state"], size["state"], path, "state of steps")


@pytest.mark.parametrize("shape", [(0, 3, 5, 4, 1), (4, 0, 5, 4, 1)])
def test_scan_without_ticks_or_columns(gpu, shape):
    draw = Draw(gpu, 2)
    operands = scan_operands(draw, *shape, torch.float32)
    check_scan(operands, None, True, draw(*shape[:3]), draw(shape[1], shape[2], shape[3]))


def test_scan_views(gpu):
    """Batch-first signals, channel slices off alignment, strided B and C, broadcast inputs
    and their summed gradients."""
    draw, T, B, N, S = Draw(gpu, 13), 19, 2, 35, 8
    base = draw(B, T, 3 * N + 1).transpose(0, 1)
    x, delta, z = base[..., 1:1 + N], base[..., 1 + N:1 + 2 * N] * 0.3, base[..., 1 + 2 * N:]
    both = draw(T, B, 2 * S)
    operands = {"x": x, "delta": delta, "A": -draw(S, N).abs().t() - 0.1, "B": both[..., :S],
                "C": both[..., S:], "D": draw(2 * N)[::2], "z": z, "delta_bias": None, "state": None}
    check_scan(operands)
    # One time step and one set of input weights for every column: gradients add up over them.
    delta, write = draw(T, 1, N, scale=0.3), draw(1, 1, S)
    d_leaf, b_leaf = delta.clone().requires_grad_(), write.clone().requires_grad_()
    y, _ = selective_scan(x, d_leaf.expand(T, B, N), operands["A"], b_leaf.expand(T, B, S),
                          operands["C"])
    got = torch.autograd.grad(y.sum(), (d_leaf, b_leaf))
    kw = dict(dy=torch.ones(T, B, N))
    parts = (x, delta.expand(T, B, N), operands["A"], write.expand(T, B, S), operands["C"])
    grads, size = so.scan(*parts, **kw)[1], so.scan(*parts, **kw, magnitude=True)[1]
    p = 2 * (70 * T + 20) + S + 60 + T * B + N
    close(got[0], grads["delta"].sum(1, keepdim=True), size["delta"].sum(1, keepdim=True), p, "ddelta")
    close(got[1], grads["B"].sum((0, 1), keepdim=True), size["B"].sum((0, 1), keepdim=True), p, "dB")


def test_gradients_against_differences(gpu):
    """Directional derivatives of a loss, from the kernels' gradients and from central
    differences of the float64 oracle (whose error, about 1e-9 here, is far below)."""
    draw = Draw(gpu, 14)
    T, B, N, S, W = 18, 2, 7, 5, 3

    def compare(operands, kernel, plain, extra):
        inputs = leaves(operands)
        outs = kernel(**inputs)
        ups = [draw(*o.shape) for o in outs]
        got = gradients(outs, inputs, ups)
        for name, grad in got.items():
            way = torch.randn(operands[name].shape, generator=draw.g, dtype=torch.float64)

            def loss(eps):
                moved = dict(operands, **{name: so.wide(operands[name]) + eps * way})
                out = plain(**moved)
                return sum((so.wide(u) * o).sum() for u, o in zip(ups, out.values()))

            slope = float((loss(1e-5) - loss(-1e-5)) / 2e-5)
            mine = float((so.wide(grad) * way).sum())
            scale = float((so.wide(grad) * way).abs().sum())
            assert abs(mine - slope) <= extra * U * scale + 1e-7 * scale, name

    compare(conv_operands(draw, T, B, N, W, torch.float32), causal_conv,
            lambda **kw: so.conv(**kw)[0], 4000)
    compare(scan_operands(draw, T, B, N, S, 1, torch.float32), selective_scan,
            lambda **kw: so.scan(**kw)[0], 4000)


def test_results_repeat_bit_for_bit(gpu):
    draw = Draw(gpu, 15)
    operands = scan_operands(draw, 70, 2, 200, 16, 2, torch.bfloat16)
    conv = conv_operands(draw, 300, 2, 50, 4, torch.bfloat16)

    def once():
        inputs = leaves(operands)
        y, final = selective_scan(**inputs)
        got = list(gradients((y, final), inputs, (torch.ones_like(y), torch.ones_like(final))).values())
        inputs = leaves(conv)
        q, last = causal_conv(**inputs)
        return [y, final, q, last, *got, *gradients((q,), inputs, (torch.ones_like(q),)).values()]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_only_what_needs_it_gets_a_gradient(gpu):
    draw = Draw(gpu, 16)
    operands = scan_operands(draw, 9, 2, 6, 4, 1, torch.float32)
    operands["A"].requires_grad_()
    y, _ = selective_scan(**operands)
    y.sum().backward()
    assert operands["A"].grad is not None and operands["x"].grad is None
    with torch.no_grad():
        assert not selective_scan(**operands)[0].requires_grad
    half = draw(6, 3).to(torch.bfloat16).requires_grad_()      # parameters in the signal's type
    y, _ = causal_conv(draw(9, 2, 6, dtype=torch.bfloat16), half)
    y.float().sum().backward()
    assert half.grad.dtype == torch.bfloat16


def test_offsets_past_32_bits(gpu):
    """Ticks 2^31 elements apart: offsets are formed in 64 bits."""
    far = 2 ** 31 + 64
    draw, N, S = Draw(gpu, 17), 16, 4
    base = torch.zeros(2 * far + N, dtype=torch.bfloat16, device=gpu)
    x = base.as_strided((3, 1, N), (far, N, 1))
    x.copy_(draw(3, 1, N, dtype=torch.bfloat16))
    near = x.contiguous()
    w = draw(N, 3)
    assert torch.equal(causal_conv(x, w)[0], causal_conv(near, w)[0])
    more = scan_operands(draw, 3, 1, N, S, 1, torch.bfloat16)
    del more["x"]
    assert torch.equal(selective_scan(x, **more)[0], selective_scan(near, **more)[0])


def test_other_streams_and_graphs(gpu):
    """Calls run on the current stream, and steps can be captured and replayed."""
    draw = Draw(gpu, 18)
    operands = scan_operands(draw, 40, 2, 70, 16, 1, torch.float32)
    want = selective_scan(**operands)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = selective_scan(**operands)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    conv = conv_operands(draw, 6, 2, 70, 4, torch.float32)
    x, state, history = draw(2, 70), operands["state"].clone(), conv["history"].clone()
    signals = ("delta", "z", "B", "C")
    fixed = {k: v[0] if k in signals else v for k, v in operands.items() if k not in ("x", "state")}

    def tick():
        filtered = causal_conv_step(x, conv["weight"], conv["bias"], history=history)
        return selective_scan_step(filtered, **fixed, state=state)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tick()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tick()
    state.copy_(operands["state"])
    history.copy_(conv["history"])
    mine, mine_history = operands["state"].clone(), conv["history"].clone()
    for t in range(4):
        x.copy_(conv["x"][t])
        graph.replay()
        torch.cuda.synchronize()
        filtered = causal_conv_step(conv["x"][t], conv["weight"], conv["bias"], history=mine_history)
        want = selective_scan_step(filtered, **fixed, state=mine)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, mine) and torch.equal(history, mine_history)


def test_refusals(gpu):
    draw = Draw(gpu, 19)
    x, w, hist = draw(4, 2, 6), draw(6, 3), draw(2, 2, 6)

    def refuses(text, fn, *args, **kw):
        with pytest.raises(ValueError, match=text):
            fn(*args, **kw)

    refuses("T, B, N", causal_conv, x[0], w)
    refuses("on a GPU", causal_conv, x.cpu(), w)
    refuses("float32, bfloat16 or float16", causal_conv, x.double(), w)
    refuses("N, W", causal_conv, x, draw(5, 3))
    refuses("1 to 8 taps", causal_conv, x, draw(6, 9))
    refuses("bias", causal_conv, x, w, draw(5))
    refuses("history", causal_conv, x, w, history=draw(3, 2, 6))
    refuses("history", causal_conv, x, w, history=hist.half())
    refuses("activation", causal_conv, x, w, activation="relu")
    refuses("lengths", causal_conv, x, w, lengths=torch.tensor([1.0, 2.0], device=gpu))
    refuses("lengths", causal_conv, x, w, lengths=torch.tensor([1, 2]))
    refuses("lengths", causal_conv, x, w, lengths=torch.tensor([1, 2, 3], device=gpu))
    refuses("no gradients", causal_conv_step, x[0].requires_grad_(), w, history=hist)
    refuses("in place", causal_conv_step, x[0].detach(), w, history=None)
    refuses("in place", causal_conv_step, x[0].detach(), w, history=draw(2, 1, 6).expand(2, 2, 6))
    refuses("in place", causal_conv_step, x[0].detach(), w, history=draw(2, 6, 2).transpose(1, 2))

    good = scan_operands(draw, 4, 2, 6, 5, 2, torch.float32)

    def scan_refuses(text, **changed):
        refuses(text, selective_scan, **{**good, **changed})

    scan_refuses("delta", delta=draw(4, 2, 5))
    scan_refuses("delta is required", delta=None)
    scan_refuses("delta must be float32", delta=good["delta"].half())
    scan_refuses("A must be", A=draw(5, 5))
    scan_refuses("1 to 64 states", A=draw(6, 65))
    scan_refuses("A must be float32", A=good["A"].half())
    scan_refuses("groups", B=draw(4, 2, 4, 5))
    scan_refuses("C must be", C=draw(4, 2, 2, 4))
    scan_refuses("B must be", B=draw(4, 2))
    scan_refuses("state", state=draw(2, 6, 4))
    scan_refuses("D must be", D=draw(7))
    step = {k: v[0] if k in ("x", "delta", "z", "B", "C") else v for k, v in good.items()}
    refuses("in place", selective_scan_step, **{**step, "state": None})
    refuses("in place", selective_scan_step, **{**step, "state": draw(2, 5, 6).transpose(1, 2)})
    refuses("no gradients", selective_scan_step, **{**step, "A": good["A"].clone().requires_grad_()})


def test_steps_move_the_version_of_what_they_update(gpu):
    """A step writes its history or state in place; a backward that kept the earlier values
    refuses, as after torch's own in-place operations."""
    draw = Draw(gpu, 20)
    conv = conv_operands(draw, 6, 2, 10, 4, torch.float32)
    wide_history = draw(3, 2, 14)
    for history in (conv["history"], wide_history[..., 2:12]):
        weight = conv["weight"].clone().requires_grad_()
        y, _ = causal_conv(conv["x"], weight, history=history)
        with torch.no_grad():
            before = history._version
            causal_conv_step(conv["x"][0], weight, history=history)
            assert history._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    assert wide_history._version == history._version

    scan = scan_operands(draw, 6, 2, 10, 5, 2, torch.float32)
    state, factor = scan.pop("state"), draw(2, 10, 5).requires_grad_()
    product = (state * factor).sum()
    selective_scan_step(**{k: v[0] if k in ("x", "delta", "z", "B", "C") else v
                           for k, v in scan.items()}, state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_steps_of_inference_tensors(gpu):
    """They keep no version, and are updated like any other."""
    draw = Draw(gpu, 21)
    conv = conv_operands(draw, 1, 2, 10, 4, torch.float32)
    scan = scan_operands(draw, 1, 2, 10, 5, 1, torch.float32)
    want_y, want_history = causal_conv(**conv)
    now = {k: v[0] if k in ("x", "delta", "z", "B", "C") else v for k, v in scan.items()
           if k != "state"}
    mine = scan["state"].clone()
    want_s = selective_scan_step(**now, state=mine)
    with torch.inference_mode():
        history, state = conv["history"].clone(), scan["state"].clone()
        y = causal_conv_step(conv["x"][0], conv["weight"], conv["bias"], history=history)
        s = selective_scan_step(**now, state=state)
        assert torch.equal(y, want_y[0]) and torch.equal(history, want_history)
        assert torch.equal(s, want_s) and torch.equal(state, mine)
        assert causal_conv_step(conv["x"][0], conv["weight"][:, :1].contiguous(),
                                history=history[:0]).shape == (2, 10)


GROWN_T, GROWN_N = 300, 5


def growing_operands(draw, S, step):
    """Rates of 2.5 to 4 and time steps of ``step`` [T, 1, N]; and the ticks of a chunk, over
    which a step of 1 a tick would multiply by more than float32 holds."""
    T, N = GROWN_T, GROWN_N
    chunks, tiles = signal_ops._plan((T, 1, N), 1, S, False)[0], -(-T // 16)
    ticks = -(-tiles // chunks) * 16
    assert chunks > 2 and 2.5 * ticks > 89
    operands = scan_operands(draw, T, 1, N, S, 1, torch.float32)
    rates = 2.5 + 1.5 * torch.rand(N, S, generator=draw.g)
    operands |= {"A": rates.to(draw.gpu), "delta": torch.log(torch.expm1(step)).to(draw.gpu),
                 "delta_bias": None, "state": None}
    return operands, ticks


@pytest.mark.parametrize("S", [4, 16])
def test_growth_over_chunks_that_hold_nothing(gpu, S):
    """A state of zero stays zero, however much a chunk would multiply it by, until the last
    ticks drive it; and so does an adjoint, until the first ticks."""
    draw, T, N, driven = Draw(gpu, 80 + S), GROWN_T, GROWN_N, 9
    operands, _ = growing_operands(draw, S, torch.full((T, 1, N), 1.0))
    x = operands["x"].clone()
    operands["x"][:T - driven] = 0
    check_scan(operands)

    operands["x"] = x.zero_()
    dy = draw(T, 1, N)
    dy[driven:] = 0
    inputs = leaves(operands)
    y, _ = selective_scan(**inputs)
    got = gradients((y,), inputs, (dy,))
    grads = so.scan(**operands, dy=dy)[1]
    size = so.scan(**operands, dy=dy, magnitude=True)[1]
    for name, value in got.items():
        close(value, grads[name], size[name], 2 * (70 * T + 20) + S + 60 + T + N, f"d{name}")
    assert float(got["x"][0].abs().max()) > 0


def test_growth_of_small_states_over_a_chunk(gpu):
    """A chunk that multiplies by more than float32 holds, on a state and a gradient of the
    final state that are small enough to bear it; the other chunks' steps are tiny."""
    draw, T, N, S = Draw(gpu, 90), GROWN_T, GROWN_N, 16
    step = torch.full((T, 1, N), 1e-13, dtype=torch.float64)
    operands, ticks = growing_operands(draw, S, step)
    step[ticks:2 * ticks] = 100 / (4.0 * ticks)             # A sum(dt) of 62 to 100
    operands["delta"] = torch.log(torch.expm1(step)).float().to(gpu)
    operands["x"].zero_()
    operands["state"] = (draw(1, N, S).abs() + 0.1) * 1e-30
    check_scan(operands, None, True, draw(T, 1, N) * 1e-30, draw(1, N, S) * 1e-30)


def test_forward_mode_derivatives_are_refused(gpu):
    """There are none: a tensor that carries one is refused, not taken without it."""
    from torch.autograd import forward_ad

    draw = Draw(gpu, 91)
    conv = conv_operands(draw, 4, 2, 6, 3, torch.float32)
    scan = scan_operands(draw, 4, 2, 6, 5, 2, torch.float32)
    tick = {k: v[0] if k in ("x", "delta", "z", "B", "C") else v for k, v in scan.items()}
    calls = [(causal_conv, conv), (selective_scan, scan), (selective_scan_step, tick),
             (causal_conv_step, {**conv, "x": conv["x"][0]})]
    with forward_ad.dual_level():
        for fn, operands in calls:
            for name, value in operands.items():
                dual = forward_ad.make_dual(value, torch.ones_like(value))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                        fn(**{**operands, name: dual})
            fn(**operands)                              # plain tensors stay welcome there


def test_forward_mode_derivatives_of_lower_precision_parameters_are_refused(gpu):
    from torch.autograd import forward_ad

    draw = Draw(gpu, 92)
    x, weight = draw(4, 2, 6, dtype=torch.bfloat16), draw(6, 3, dtype=torch.bfloat16)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        causal_conv(x, forward_ad.make_dual(weight, torch.ones_like(weight)))


@pytest.mark.parametrize("T", [1, 16, 20, 260])
def test_rates_of_minus_infinity(gpu, T):
    """They forget at once: the state is the last tick's input, in the signal's form (whose last
    tile may reach past the end, and whose time may be cut into chunks) as in the steps'."""
    draw, B, N, S = Draw(gpu, 93), 3, 6, 5
    operands = scan_operands(draw, T, B, N, S, 2, torch.float32)
    operands["A"][::2, 1:3] = -math.inf
    operands["A"][1, 0] = -3e38
    check_scan(operands)
    y, _ = selective_scan(**operands)
    lengths = torch.tensor([T, T // 2, 0], dtype=torch.int32, device=gpu)
    short, final = selective_scan(**operands, lengths=lengths)
    assert torch.equal(short[:, 0], y[:, 0]) and torch.equal(final[2], operands["state"][2])
    half = {k: v[:T // 2, 1:2] if k in ("x", "delta", "z", "B", "C") else v
            for k, v in operands.items()}
    half["state"] = operands["state"][1:2]
    alone = so.scan(**half)[0]["state"]
    size = so.scan(**half, magnitude=True)[0]["state"]
    close(final[1:2], alone, size, 70 * T + 20, "state of a column's own length")
    state = operands["state"].clone()
    for t in range(min(T, 3)):
        selective_scan_step(**{k: v[t] if k in ("x", "delta", "z", "B", "C") else v
                               for k, v in operands.items() if k != "state"}, state=state)
    assert torch.isfinite(state).all()

    # The gradients that the limit has: of x and B, and of the first state.
    if T > 100:
        return
    names = ("x", "B", "C", "state")
    inputs = {k: v.clone().requires_grad_() if k in names else v for k, v in operands.items()}
    dy, dfinal = draw(T, B, N), draw(B, N, S)
    y, final = selective_scan(**inputs)
    got = torch.autograd.grad((y, final), [inputs[k] for k in names], (dy, dfinal))
    grads = so.scan(**operands, dy=dy, dfinal=dfinal)[1]
    size = so.scan(**operands, dy=dy, dfinal=dfinal, magnitude=True)[1]
    for name, value in zip(names, got):
        close(value, grads[name], size[name], 2 * (70 * T + 20) + S + 60 + N, f"d{name}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,S,G,chunks", [(140, 16, 2, 19), (66, 24, 1, 25), (18, 40, 3, 75), (198, 7, 3, 19)])
def test_scan_in_many_chunks_of_time(gpu, N, S, G, chunks, dtype):
    """More chunks than the join asks for at a time, and no multiple of that; several groups and
    workgroups to a group, the last of them partly empty; columns that end inside a chunk, at
    a chunk's first tick, and before the first tick."""
    draw, T, B = Draw(gpu, 100 + S), 600, 4
    assert signal_ops._plan((T, B, N), G, S, True)[0] == chunks and chunks % 16
    operands = scan_operands(draw, T, B, N, S, G, dtype)
    ticks = -(-T // chunks)
    lengths = torch.tensor([T, 333, 0, 5 * ticks], device=gpu) if S != 40 else None
    check_scan(operands, lengths, True, draw(T, B, N, dtype=dtype), draw(B, N, S))
