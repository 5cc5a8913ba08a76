"""Gated linear recurrence against float64 formulas (MI355X).

Tolerances.  With u = 2^-24, a float32 operation adds a relative error of at most u to what
it computes, hardware exp2, reciprocal and square root at most 2u.  A sigmoid of |v| <= 5 is
off by at most 10u (the exponent's |v| u, then exp2, an add and a reciprocal), the fade rate s
by 11u, the decay exp(-fade), fade <= 2, by 28u, the room sqrt(1 - a^2) by 15u (its series by
18u; from the threshold on, 1 - a^2 by 2 a^2 / (1 - a^2) times the decay's few u: at most 26u;
the root halves that), what a tick takes in by 30u, and a term gains at most 30u with every
tick that it passes.  A result is then off by (30 ticks + what follows) u times the sum of its
terms' sizes, which the oracle gives.  Gradients pass the states' ticks and the adjoint's:
60 ticks, and at most 150 around them.  Outputs are then rounded once to their type.
"""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from test_gpu_signal import Draw, close, gradients, leaves
from neurosim_gpu import gated_recurrence, gated_recurrence_step

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("x", "forget", "write", "rates", "z", "state")
SHAPES = [  # T, B, N
    (1, 1, 1), (1, 3, 2), (7, 2, 1), (31, 2, 5), (32, 1, 66), (33, 1, 3), (63, 1, 129), (64, 2, 65), (65, 3, 33), (130, 2, 257),
    (128, 5, 64), (300, 1, 40), (513, 2, 130), (9, 16, 3), (512, 1, 9), (1030, 1, 17),
    (70, 256, 3), (130, 90, 257), (64, 256, 1), (5, 300, 2), (200, 256, 2),
]


def operands(draw, T, B, N, dtype, gate=True, state=True):
    bounded = lambda: draw(T, B, N).clamp(-5, 5).to(dtype)  # noqa: E731
    return {"x": draw(T, B, N, dtype=dtype), "forget": bounded(), "write": bounded(),
            "rates": draw(N).abs().clamp(1e-4, 2.0), "z": bounded() if gate else None,
            "state": draw(B, N) if state else None}


def check(values, lengths=None, dy=None, dfinal=None):
    T, B, N = values["x"].shape
    inputs = leaves(values) if dy is not None else values
    y, final = gated_recurrence(**inputs, lengths=lengths)
    kw = dict(lengths=lengths, dy=dy, dfinal=dfinal)
    want, grads = bo.recurrence(**values, **kw)
    size, grad_size = bo.recurrence(**values, **kw, magnitude=True)
    close(y, want["y"], size["y"], 30 * T + 50, "y")
    close(final, want["state"], size["state"], 30 * T + 35, "state")
    if dy is None:
        return y, final
    got = gradients((y, final), inputs, (dy, dfinal))
    assert set(got) == {k for k, v in values.items() if v is not None}
    for name, value in got.items():
        summands = T * B if name == "rates" else 2
        close(value, grads[name], grad_size[name], 60 * T + 150 + summands, f"d{name}")
    return y, final, got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_signals_and_gradients(gpu, shape, dtype):
    draw = Draw(gpu, sum(shape))
    values = operands(draw, *shape, dtype, gate=shape[0] % 2 == 1, state=shape[1] != 2)
    check(values, None, draw(*shape, dtype=dtype), draw(*shape[1:]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2500, 1, 37), (800, 2, 130), (2050, 1, 4200)])
def test_chunks(gpu, shape, dtype):
    """Long signals of few channels, whose time is cut into chunks, the last with two channels of
    16 bits to a lane."""
    draw = Draw(gpu, 3)
    T, B, N = shape
    check(operands(draw, T, B, N, dtype), None, draw(T, B, N, dtype=dtype), draw(B, N))


@pytest.mark.parametrize("lengths", [None, [17500, 16384, 9001]])
def test_more_chunks_than_wavefronts(gpu, lengths):
    """Many chunks.  Rates of 0.5 at least and gates of sigmoid(-1) at least let a channel
    forget by exp(-0.13) a tick, so terms older than 300 ticks, below exp(-40) of the others,
    count for nothing, and the bounds are those of 300 ticks."""
    draw = Draw(gpu, 13)
    T, B, N = 17500, 3, 2                        # 136 chunks
    values = operands(draw, T, B, N, torch.float32)
    values["rates"] = values["rates"].clamp(min=0.5)
    values["forget"] = values["forget"].clamp(min=-1)
    lengths = None if lengths is None else torch.tensor(lengths, device=gpu)
    dy, dfinal = draw(T, B, N), draw(B, N)
    inputs = leaves(values)
    y, final = gated_recurrence(**inputs, lengths=lengths)
    kw = dict(lengths=lengths, dy=dy, dfinal=dfinal)
    want, grads = bo.recurrence(**values, **kw)
    size, grad_size = bo.recurrence(**values, **kw, magnitude=True)
    close(y, want["y"], size["y"], 30 * 300 + 50, "y")
    close(final, want["state"], size["state"], 30 * 300 + 35, "state")
    for name, value in gradients((y, final), inputs, (dy, dfinal)).items():
        summands = T * B if name == "rates" else 2
        # dstate has passed every tick of its column.
        passed = 60 * T if name == "state" else 60 * 300
        close(value, grads[name], grad_size[name], passed + 150 + summands, f"d{name}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths_of_many_columns(gpu, dtype):
    """Many columns, each walked by workgroups of its own in one chunk."""
    draw = Draw(gpu, 15)
    T, B, N = 140, 256, 3
    values = operands(draw, T, B, N, dtype)
    lengths = torch.randint(0, T + 1, (B,), generator=draw.g, dtype=torch.int32).to(gpu)
    lengths[:6] = torch.tensor([0, 1, 31, 32, 33, T], dtype=torch.int32)
    dy = draw(T, B, N, dtype=dtype)
    past = torch.arange(T, device=gpu)[:, None] >= lengths
    for v in (values["x"], values["forget"], values["write"], values["z"], dy):
        v[past] = float("nan")
    y, _, got = check(values, lengths, dy, draw(B, N))
    for value in (y, *(got[k] for k in ("x", "forget", "write", "z"))):
        assert not value[past].any()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths(gpu, kind, dtype):
    """Columns of no, one, some, all and claimed more ticks, over several chunks and tiles;
    what stands past an end is NaN and never used."""
    draw = Draw(gpu, 5)
    T, B, N = 700, 8, 21
    values = operands(draw, T, B, N, dtype)
    lengths = torch.tensor([0, 1, 31, 32, 65, 333, T, T + 9], dtype=kind, device=gpu)
    dy = draw(T, B, N, dtype=dtype)
    for b, end in enumerate(lengths.tolist()):
        for k in ("x", "forget", "write", "z"):
            values[k][end:, b] = float("nan")
        dy[end:, b] = float("nan")
    y, _, got = check(values, lengths, dy, draw(B, N))
    for value in (y, *(got[k] for k in ("x", "forget", "write", "z"))):
        for b, end in enumerate(lengths.tolist()):
            assert not value[end:, b].any()


def test_no_ticks_and_no_columns(gpu):
    draw = Draw(gpu, 1)
    values = operands(draw, 0, 2, 5, torch.float32)
    inputs = leaves(values)
    y, final = gated_recurrence(**inputs)
    assert y.shape == (0, 2, 5) and torch.equal(final, values["state"])
    up = draw(2, 5)
    assert torch.equal(torch.autograd.grad(final, inputs["state"], up)[0], up)
    y, final = gated_recurrence(**operands(draw, 4, 0, 5, torch.float32))
    assert y.shape == (4, 0, 5) and final.shape == (0, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides(gpu, dtype):
    """[B, T, N] signals as transposed views, slices of a wider projection, spread columns."""
    draw = Draw(gpu, 9)
    T, B, N = 70, 3, 35
    values = operands(draw, T, B, N, dtype)
    wide = torch.cat([values[k] for k in ("forget", "write", "z")], -1)
    moved = dict(values, x=values["x"].transpose(0, 1).contiguous().transpose(0, 1))
    moved["forget"], moved["write"], moved["z"] = wide.split(N, -1)
    dy = draw(B, T, N, dtype=dtype).transpose(0, 1)
    ups = (dy, draw(B, N))
    one, two = leaves(values), None
    outs = gated_recurrence(**one)
    first = gradients(outs, one, ups)
    two = {k: v.detach().requires_grad_() for k, v in moved.items()}
    again = gated_recurrence(**two)
    assert torch.equal(outs[0], again[0]) and torch.equal(outs[1], again[1])
    for k, v in gradients(again, two, ups).items():
        assert torch.equal(v, first[k]), k
    spread = torch.stack((values["x"], values["x"]), -1)[..., 0]      # channels not dense
    assert torch.equal(gated_recurrence(**dict(values, x=spread))[0], outs[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_are_the_signal(gpu, dtype):
    draw = Draw(gpu, 4)
    T, B, N = 20, 3, 67
    values = operands(draw, T, B, N, dtype)
    y, final = gated_recurrence(**values)
    state = values["state"].clone()
    ticks = [gated_recurrence_step(values["x"][t], values["forget"][t], values["write"][t],
                                   values["rates"], z=values["z"][t], state=state)
             for t in range(T)]
    want, _ = bo.recurrence(**values)
    size, _ = bo.recurrence(**values, magnitude=True)
    close(torch.stack(ticks), want["y"], size["y"], 30 * T + 50, "y")
    close(state, want["state"], size["state"], 30 * T + 35, "state")
    # The signal in two parts carries on where the first one ends.
    cut = {k: v[:13] if v.dim() == 3 else v for k, v in values.items()}
    rest = {k: v[13:] if v.dim() == 3 else v for k, v in values.items()}
    one, middle = gated_recurrence(**cut)
    two, end = gated_recurrence(**dict(rest, state=middle))
    close(torch.cat((one, two)), want["y"], size["y"], 30 * T + 50, "y in parts")
    close(end, want["state"], size["state"], 30 * T + 35, "state in parts")


def test_ends_of_the_range(gpu):
    """Rates of zero, below zero and infinite, gates wide open and shut, and a slow channel over
    many ticks."""
    T, B, N = 90, 1, 6
    draw = Draw(gpu, 8)
    values = operands(draw, T, B, N, torch.float32)
    values["rates"] = torch.tensor([0.0, -1.0, float("inf"), 1.0, 1.0, 1e-6], device=gpu)
    values["forget"][:, :, 2] = 3.0
    values["forget"][:, :, 3] = 200.0            # sigmoid is 1
    values["forget"][:, :, 4] = -200.0           # sigmoid is below float32: nothing is forgotten
    inputs = leaves(values)
    y, final = gated_recurrence(**inputs)
    got = gradients((y, final), inputs, (draw(T, B, N), draw(B, N)))
    for value in (y, final, *got.values()):
        assert torch.isfinite(value).all()
    held = values["state"][0]
    for n in (0, 1, 4):                          # held as they are
        assert torch.equal(final[0, n], held[n])
    taken = torch.sigmoid(values["write"][:, 0, 2].double()) * values["x"][:, 0, 2].double()
    gate = torch.nn.functional.silu(values["z"][:, 0, 2].double())
    assert (y[:, 0, 2].double() - taken * gate).abs().max() < 1e-6
    want, _ = bo.recurrence(**{**values, "rates": values["rates"].clamp(min=0, max=1e9)})
    assert (final.double().cpu() - want["state"]).abs().max() < 1e-5


def test_not_a_number_stays_in_its_channel(gpu):
    draw = Draw(gpu, 2)
    values = operands(draw, 200, 2, 70, torch.bfloat16)
    values["x"][100, 1, 7] = float("nan")
    clean, _ = gated_recurrence(**dict(values, x=torch.nan_to_num(values["x"])))
    y, final = gated_recurrence(**values)
    assert torch.isnan(y[100:, 1, 7]).all() and torch.isnan(final[1, 7])
    y[100:, 1, 7] = clean[100:, 1, 7] = 0
    assert torch.equal(y, clean)


def test_other_streams_and_repeats(gpu):
    """On another stream, in two of them at once, and again: the same bits."""
    draw = Draw(gpu, 6)
    values = operands(draw, 600, 2, 90, torch.float32)
    dy, dfinal = draw(600, 2, 90), draw(2, 90)

    def passes():
        inputs = leaves(values)
        outs = gated_recurrence(**inputs)
        return (*outs, *gradients(outs, inputs, (dy, dfinal)).values())

    first = passes()
    torch.cuda.synchronize()
    streams, others = [torch.cuda.Stream() for _ in range(2)], []
    for stream in streams:
        with torch.cuda.stream(stream):
            others.append(passes())
    torch.cuda.synchronize()
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_captured_steps_and_signals(gpu):
    draw = Draw(gpu, 7)
    values = operands(draw, 150, 1, 33, torch.float32)
    tick = {k: values[k][0].clone() for k in ("x", "forget", "write", "z")}
    state = values["state"].clone()

    def once():
        y, final = gated_recurrence(**values)
        return y, final, gated_recurrence_step(tick["x"], tick["forget"], tick["write"],
                                               values["rates"], z=tick["z"], state=state)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = once()
    for k in range(4):
        values["x"].copy_(draw(150, 1, 33))
        state.copy_(draw(1, 33))
        kept = state.clone()
        graph.replay()
        torch.cuda.synchronize()
        y, final = gated_recurrence(**values)
        step = gated_recurrence_step(tick["x"], tick["forget"], tick["write"], values["rates"],
                                     z=tick["z"], state=kept)
        for a, b in zip((*outs, state), (y, final, step, kept)):
            assert torch.equal(a, b), k


def test_a_step_moves_the_version_of_its_state(gpu):
    draw = Draw(gpu, 1)
    values = operands(draw, 1, 2, 5, torch.float32)
    state = values["state"]
    leaf = torch.ones(2, 5, device=gpu, requires_grad=True)
    product = leaf * state
    gated_recurrence_step(values["x"][0], values["forget"][0], values["write"][0], values["rates"],
                          state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()


def test_refusals(gpu):
    draw = Draw(gpu, 0)
    good = operands(draw, 4, 2, 6, torch.float32)
    for change, message in (
            ({"x": good["x"].double()}, "float32, bfloat16 or float16"),
            ({"x": good["x"].cpu()}, "on a GPU"), ({"x": good["x"][0]}, r"\[T, B, N\]"),
            ({"forget": good["forget"][:3]}, "forget must be a tensor of shape"),
            ({"write": None}, "write must be a tensor"),
            ({"write": good["write"].half()}, "write must be float32"),
            ({"rates": good["rates"].double()}, "rates must be float32"),
            ({"rates": good["rates"][:5]}, "rates must be a tensor of shape"),
            ({"z": good["z"].cpu()}, "z must be on the signal's device"),
            ({"state": good["state"].half()}, "state must be float32"),
            ({"lengths": torch.zeros(3, dtype=torch.int32, device=gpu)}, "one int32 or int64"),
            ({"lengths": torch.zeros(2, dtype=torch.int32)}, "lengths must be on")):
        with pytest.raises(ValueError, match=message):
            gated_recurrence(**{**good, **change})
    tick = {k: good[k][0] for k in ("x", "forget", "write", "z")}
    with pytest.raises(ValueError, match="contiguous"):
        gated_recurrence_step(**tick, rates=good["rates"], state=draw(6, 2).t())
    with pytest.raises(ValueError, match="contiguous"):
        gated_recurrence_step(**tick, rates=good["rates"], state=None)
    with pytest.raises(ValueError, match="no gradients"):
        gated_recurrence_step(**dict(tick, x=tick["x"].clone().requires_grad_()),
                              rates=good["rates"], state=good["state"])
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            gated_recurrence(**dict(good, x=fwAD.make_dual(good["x"], torch.ones_like(good["x"]))))
