"""The tests' float64 gradient formulas against autograd through the same equations."""

from __future__ import annotations

import pytest
import torch

import signal_oracle as so


def leaf(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).requires_grad_()


@pytest.mark.parametrize("activation", ["silu", None])
def test_conv_formulas(activation):
    g = torch.Generator().manual_seed(3)
    x, w, b, hist = leaf(g, 9, 3, 5), leaf(g, 5, 4), leaf(g, 5), leaf(g, 3, 3, 5)
    dy, dlast = (torch.randn(9, 3, 5, generator=g, dtype=torch.float64),
                 torch.randn(3, 3, 5, generator=g, dtype=torch.float64))
    line = torch.cat((hist, x))
    pre = b + sum(w[:, k] * line[k:k + 9] for k in range(4))
    y = torch.nn.functional.silu(pre) if activation else pre
    want = torch.autograd.grad((y, line[9:]), (x, w, b, hist), (dy, dlast))
    out, grads = so.conv(x, w, b, hist, activation=activation, dy=dy, dlast=dlast)
    assert torch.allclose(out["y"], y.detach(), rtol=1e-12, atol=1e-14)
    for name, value in zip(("x", "weight", "bias", "history"), want):
        assert torch.allclose(grads[name], value, rtol=1e-11, atol=1e-13), name


@pytest.mark.parametrize("soft", [True, False])
def test_scan_formulas(soft):
    g = torch.Generator().manual_seed(4)
    T, Bt, N, S, G = 7, 2, 6, 3, 2
    x, delta, z = leaf(g, T, Bt, N), leaf(g, T, Bt, N, scale=0.3), leaf(g, T, Bt, N)
    A, D, bias = leaf(g, N, S), leaf(g, N), leaf(g, N)
    B, C, state = leaf(g, T, Bt, G, S), leaf(g, T, Bt, G, S), leaf(g, Bt, N, S)
    dy, dh = (torch.randn(T, Bt, N, generator=g, dtype=torch.float64),
              torch.randn(Bt, N, S, generator=g, dtype=torch.float64))
    raw = delta + bias
    dt = torch.nn.functional.softplus(raw) if soft else raw
    h, ys = state, []
    for t in range(T):
        write, read = (v[t].repeat_interleave(N // G, 1) for v in (B, C))
        h = torch.exp(dt[t][..., None] * A) * h + (dt[t] * x[t])[..., None] * write
        ys.append(((read * h).sum(-1) + D * x[t]) * torch.nn.functional.silu(z[t]))
    leaves = {"x": x, "delta": delta, "A": A, "B": B, "C": C, "D": D, "z": z, "delta_bias": bias,
              "state": state}
    want = dict(zip(leaves, torch.autograd.grad((torch.stack(ys), h), list(leaves.values()), (dy, dh))))
    out, grads = so.scan(x, delta, A, B, C, D, z, bias, soft, state, dy=dy, dfinal=dh)
    assert torch.allclose(out["state"], h.detach(), rtol=1e-12, atol=1e-14)
    for name, value in want.items():
        assert torch.allclose(grads[name], value, rtol=1e-10, atol=1e-12), name


def test_mx_codes_of_the_grid():
    """Levels map to themselves, midpoints to the even code, larger values saturate."""
    levels = so.LEVELS
    middle = (levels[1:] + levels[:-1]) / 2
    row = torch.zeros(32, dtype=torch.float64)
    row[:8], row[8:15], row[15], row[16] = levels, middle, 7.9, -levels[3]
    codes, scales = so.mx_quantize(row)
    assert scales.tolist() == [127]
    assert codes[:8].tolist() == list(range(8))
    assert codes[8:15].tolist() == [0, 2, 2, 4, 4, 6, 6]
    assert codes[15] == 7 and codes[16] == 8 + 3
