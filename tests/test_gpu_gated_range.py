"""Gradients of the gated projection in float16 whose dg = dy u f'(g) and du = dy f(g) are not in
float16's range, though the gradients are (MI355X).

Tolerances are those of test_gpu_block.py (block_oracle.gated_bounds: float32 sums, dg and du rounded
to 11 bits), without an allowance for numbers that vanish: dg and du are rounded as multiples of a
power of two for each row of [dg du], and for each column of either, that brings the largest one to
2^14 at least.  Below float16's normal numbers a rounding is then off by half of 2^-24, so by
2^-39 of the largest one, which passes through the products.
"""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from signal_oracle import wide
from test_gpu_block import operands, within
from test_gpu_signal import HALF_ULP, U, Draw, leaves
from neurosim_gpu import gated_projection

pytestmark = pytest.mark.gpu

SHAPES = [(3, 40, 20), (40, 130, 44), (300, 70, 90), (1030, 300, 700), (2100, 72, 2800), (40, 2100, 2820),
          (4120, 2900, 20)]


def gradients(values: dict, dy, activation="silu") -> dict:
    inputs = leaves(values)
    y = gated_projection(**inputs, activation=activation)
    return dict(zip(inputs, torch.autograd.grad(y, list(inputs.values()), dy)))


def check(values: dict, dy, activation="silu", rows=None, columns=None):
    """Gradients within their bounds (``rows`` of dx, ``columns`` of the weights': those that are)."""
    got = gradients(values, dy, activation)
    finite = torch.nan_to_num(dy, nan=0.0, posinf=0.0, neginf=0.0)
    _, want = bo.gated(**values, activation=activation, dy=finite)
    bounds = bo.gated_bounds(**values, activation=activation, dy=finite, u=U, half=HALF_ULP[torch.float16])
    x, gate, up = (wide(values[k]) for k in ("x", "gate", "up"))
    g, w, d = x @ gate.t(), x @ up.t(), wide(finite)
    value, slope = bo.activated(g, activation)
    dg, du = (d * w * slope).abs(), (d * value).abs()
    vanish = 1.01 * 2.0 ** -39             # a hundredth for the errors of the largest ones themselves
    largest = torch.maximum(dg, du).amax(1, keepdim=True)
    low = {"x": vanish * largest * (gate.abs() + up.abs()).sum(0),
           "gate": vanish * dg.amax(0)[:, None] * x.abs().sum(0),
           "up": vanish * du.amax(0)[:, None] * x.abs().sum(0)}
    for name, grad in got.items():
        keep = rows if name == "x" else columns
        keep = slice(None) if keep is None else keep
        assert float(want[name].abs().max()) <= 65504        # in range, or the case is no such one
        within(grad[keep], want[name][keep], (bounds[name] + low[name])[keep], f"d{name}")
    return got


@pytest.mark.parametrize("shape", SHAPES)
def test_small_products(gpu, shape):
    """dy of 1e-4 and products of 1e-3: dg and du of 1e-7 and less, near the least of float16."""
    M, K, F = shape
    draw = Draw(gpu, sum(shape))
    values = operands(draw, M, K, F, torch.float16)
    values = {**values, "gate": values["gate"] * 1e-3, "up": values["up"] * 1e-3}
    check(values, draw(M, F, scale=1e-4, dtype=torch.float16))


@pytest.mark.parametrize("shape", SHAPES)
def test_small_products_of_one_sign(gpu, shape):
    """Nothing cancels: sums over many rows of what rounds to zero."""
    M, K, F = shape
    draw = Draw(gpu, sum(shape))
    values = operands(draw, M, K, F, torch.float16)
    values = {"x": values["x"].abs(), "gate": values["gate"].abs(),
              "up": values["up"].abs() * (2e-4 * K ** -0.5)}
    dy = (draw(M, F).abs() * 1e-4).half()
    check(values, dy, "gelu")


@pytest.mark.parametrize("shape", SHAPES)
def test_large_products(gpu, shape):
    """Products dy u of up to some 1e6, whose sums over small x and gate are in float16's range."""
    M, K, F = shape
    draw = Draw(gpu, sum(shape))
    values = {"x": draw(M, K, scale=1e-3, dtype=torch.float16),
              "gate": draw(F, K, scale=1e-3, dtype=torch.float16),
              "up": draw(F, K, scale=min(2e4, 2e5 * K ** -0.5)).clamp(-6e4, 6e4).half()}
    dy = draw(M, F, scale=1000.0, dtype=torch.float16)
    dg = 0.5 * wide(dy) * (wide(values["x"]) @ wide(values["up"]).t())     # silu's slope at 0
    assert float(dg.abs().max()) > 1.1 * 65504
    check(values, dy)


def test_rows_and_columns_of_their_own_size(gpu):
    """Rows of dy from 60,000 down to 1e-7, columns of weights from 1 to 1e-4, an empty row and
    an empty column; an infinity, a NaN, and no other row or column touched by them."""
    draw = Draw(gpu, 4)
    M, K, F = 200, 96, 150
    values = operands(draw, M, K, F, torch.float16)
    values["x"] = values["x"] * 0.05
    values["up"] = (values["up"].float() * torch.logspace(0, -4, F, device=gpu)[:, None]).half()
    dy = draw(M, F) * torch.logspace(4, -6, M, device=gpu)[:, None]
    dy = dy.clamp(-6e4, 6e4).half()
    dy[7], dy[:, 9] = 0, 0
    got = check(values, dy)
    assert not got["x"][7].any() and not got["gate"][9].any() and not got["up"][9].any()
    dy[11, 3], dy[60, 140] = float("inf"), float("nan")
    rows = torch.tensor([m for m in range(M) if m not in (11, 60)])
    columns = torch.tensor([f for f in range(F) if f not in (3, 140)])
    got = check(values, dy, rows=rows, columns=columns)
    for name, keep in (("x", (11, 60)), ("gate", (3, 140)), ("up", (3, 140))):
        assert not torch.isfinite(got[name][list(keep)]).any(), name


@pytest.mark.parametrize("shape", [(40, 130, 44), (4400, 1000, 50)])
def test_gradients_of_some_and_again(gpu, shape):
    """Asked for one at a time, or again, they are the same bits."""
    M, K, F = shape
    draw = Draw(gpu, M)
    values, dy = operands(draw, M, K, F, torch.float16), draw(M, F, scale=1e-5, dtype=torch.float16)
    want = gradients(values, dy)
    for _ in range(2):
        for name, value in gradients(values, dy).items():
            assert torch.equal(value, want[name]), name
    for name in values:
        inputs = {k: v.clone().requires_grad_(k == name) for k, v in values.items()}
        got = torch.autograd.grad(gated_projection(**inputs), inputs[name], dy)[0]
        assert torch.equal(got, want[name]), name
