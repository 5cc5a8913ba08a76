"""Float32 projections that take one float32 matrix instruction a product: up to 16 rows, and those too
small to repay three bfloat16 parts (MI355X).

Their sums have no more than K products, so block_oracle.gated_bounds holds without the six times that
it allows for parts (which it does where ``half`` is zero: y's own bound has no other use for it)."""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from test_gpu_block import operands, within
from test_gpu_signal import U, Draw, leaves
from neurosim_gpu import block_ops, gated_projection

pytestmark = pytest.mark.gpu

# M, K, F with whole 16-byte rows: laid out anew they would be in parts.
SHAPES = [(1, 64, 16), (1, 4096, 200), (7, 1032, 70), (16, 200, 33), (17, 32, 32), (65, 96, 40), (130, 256, 100),
          (64, 4096, 256), (200, 1000, 77), (1030, 72, 1700), (700, 512, 120)]


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES)
def test_float32_products(gpu, shape, activation):
    M, K, F = shape
    draw = Draw(gpu, sum(shape))
    values = operands(draw, M, K, F, torch.float32)
    args = block_ops._gated_args(values["x"], values["gate"], values["up"], 0)
    assert block_ops._library().ns_gated_forward_bytes(args) == 0
    none = torch.zeros(M, F)
    want, _ = bo.gated(**values, activation=activation)
    bounds = bo.gated_bounds(**values, activation=activation, dy=none, u=U, half=U)
    within(gated_projection(**values, activation=activation), want, bounds["y"], "y")
    # The kept products themselves: 2 u an addition, of which a product has K.
    y = gated_projection(**leaves(values), activation=activation)
    pre = y.grad_fn.saved_tensors[3]
    x = values["x"].double().cpu()
    for k, name in enumerate(("gate", "up")):
        w = values[name].double().cpu()
        within(pre[k], x @ w.t(), 2 * (K + 2) * U * (x.abs() @ w.abs().t()), name)
