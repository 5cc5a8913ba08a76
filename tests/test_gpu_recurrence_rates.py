"""The gradient of rates below zero, which count as zero (MI355X).

What is computed does not depend on such a rate, so its gradient is zero: the same as the differences
of the outputs, which are exactly zero there.  Other gradients are those of a rate of zero, bit for bit."""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from test_gpu_recurrence import operands
from test_gpu_signal import Draw, gradients, leaves
from neurosim_gpu import gated_recurrence

pytestmark = pytest.mark.gpu

# T, B, N: a tile, chunks of time, many columns, two channels of 16 bits to a lane.
SHAPES = [(9, 2, 6), (2500, 1, 37), (70, 256, 7), (2050, 1, 4200)]


def passes(values, ups):
    inputs = leaves(values)
    outs = gated_recurrence(**inputs)
    return [v.detach() for v in outs], gradients(outs, inputs, ups)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_rates_below_zero_have_no_gradient(gpu, shape, dtype):
    draw = Draw(gpu, sum(shape))
    T, B, N = shape
    values, ups = operands(draw, *shape, dtype), (draw(*shape, dtype=dtype), draw(B, N))
    below = torch.zeros(N, dtype=torch.bool, device=gpu)
    below[::3] = True
    values["rates"][0], values["rates"][3] = -float("inf"), -1e-30
    values["rates"] = torch.where(below, -values["rates"].abs(), values["rates"])
    values["rates"][1] = 0.0
    outs, got = passes(values, ups)
    held, want = passes(dict(values, rates=values["rates"].clamp(min=0)), ups)
    assert all(torch.equal(a, b) for a, b in zip(outs, held))
    assert not got["rates"][below].any()
    assert torch.equal(got["rates"][~below], want["rates"][~below]) and got["rates"][1] != 0
    for name in ("x", "forget", "write", "z", "state"):
        assert torch.equal(got[name], want[name]), name


def test_against_differences(gpu):
    """Central differences of float64 outputs, a step that stays on the rate's own side."""
    draw = Draw(gpu, 1)
    T, B, N = 6, 2, 4
    values, ups = operands(draw, T, B, N, torch.float32), (draw(T, B, N), draw(B, N))
    values["rates"] = torch.tensor([-0.5, 0.7, -1e-3, 1.3], device=gpu)
    _, got = passes(values, ups)
    wide = {k: v.double().cpu() for k, v in values.items()}

    def total(rates):
        out, _ = bo.recurrence(**dict(wide, rates=rates))
        return float((out["y"] * ups[0].double().cpu()).sum() + (out["state"] * ups[1].double().cpu()).sum())

    step = 1e-5
    for n in range(N):
        move = torch.zeros(N, dtype=torch.float64)
        move[n] = step
        slope = (total(wide["rates"] + move) - total(wide["rates"] - move)) / (2 * step)
        # Differences: step^2 of a third derivative of some units, and 1e-16 / step; float32: 1e-6.
        assert abs(float(got["rates"][n]) - slope) <= 1e-5 * (1 + abs(slope)), n
    assert got["rates"][0] == 0 and got["rates"][2] == 0
