"""Plain float64 restatements of the gated block's operators, for the tests.

``magnitude=True`` takes every term with its absolute value: the sum of the absolute values of
the terms that make up a result, to which rounding errors are proportional.
"""

from __future__ import annotations

import math

import torch

from signal_oracle import ends_of, silu, wide


def recurrence(x, forget, write, rates, z=None, state=None, lengths=None, dy=None, dfinal=None,
               magnitude=False):
    """(outputs, gradients) of the gated linear recurrence, one tick at a time."""
    x, forget, write, rates, z, state, dy, dfinal = (
        wide(v) for v in (x, forget, write, rates, z, state, dy, dfinal))
    ticks, batch, n = x.shape
    size = torch.abs if magnitude else (lambda v: v)
    zero = torch.zeros((), dtype=torch.float64)
    live = (torch.arange(ticks)[:, None] < torch.tensor(ends_of(lengths, ticks, batch)))[:, :, None]
    x, forget, write = (torch.where(live, v, zero) for v in (x, forget, write))
    gated = torch.ones_like(x) if z is None else torch.where(live, z, zero)
    gate, slope = (torch.ones_like(x), torch.zeros_like(x)) if z is None else silu(gated)
    if z is not None and magnitude:
        s = torch.sigmoid(gated)
        slope = s * (1 + gated.abs() * (1 - s))
    s, i = torch.sigmoid(forget), torch.sigmoid(write)
    u = torch.where(live, rates.clamp(min=0) * s, zero)
    a, m = torch.exp(-u), torch.sqrt(-torch.expm1(-2 * u))
    h = torch.zeros(batch, n, dtype=torch.float64) if state is None else size(state)
    y, before = torch.zeros_like(x), []
    for t in range(ticks):
        before.append(h)
        h = a[t] * h + size(m[t] * i[t] * x[t])
        y[t] = torch.where(live[t], h * size(gate[t]), zero)
    out = {"y": y, "state": h}
    if dy is None:
        return out, {}
    dy = torch.where(live, dy, zero)
    g = torch.zeros(batch, n, dtype=torch.float64) if dfinal is None else size(dfinal)
    grads = {k: torch.zeros_like(x) for k in ("x", "forget", "write", "z")}
    grads["rates"] = torch.zeros(n, dtype=torch.float64)
    after = h
    for t in range(ticks - 1, -1, -1):
        grads["z"][t] = size(dy[t] * slope[t]) * after
        g = g + size(dy[t] * gate[t])
        grads["x"][t] = g * m[t] * i[t]
        grads["write"][t] = g * m[t] * i[t] * (1 - i[t]) * size(x[t])
        to_m = torch.where(m[t] > 0, a[t] * a[t] / m[t], zero)
        kept = -before[t] if not magnitude else before[t]
        by_u = g * (to_m * i[t] * size(x[t]) + a[t] * kept)
        grads["forget"][t] = by_u * u[t] * (1 - s[t])
        grads["rates"] += torch.where(live[t], by_u * s[t], zero).sum(0)
        g, after = a[t] * g, before[t]
    grads["state"] = g
    return out, grads
