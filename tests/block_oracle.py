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


def activated(x, activation: str):
    """(value, slope) of an activation."""
    if activation == "silu":
        return silu(x)
    below = 0.5 * torch.special.erfc(-x * math.sqrt(0.5))
    return x * below, below + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def gated(x, gate, up, activation="silu", dy=None):
    """y and its gradients (without dy: none)."""
    x, gate, up, dy = (wide(v) for v in (x, gate, up, dy))
    g, u = x @ gate.t(), x @ up.t()
    value, slope = activated(g, activation)
    if dy is None:
        return value * u, {}
    dg, du = dy * u * slope, dy * value
    return value * u, {"x": dg @ gate + du @ up, "gate": dg.t() @ x, "up": du.t() @ x}


def gated_bounds(x, gate, up, activation, dy, u, half):
    """How far y and the gradients may be off for sums in arithmetic of half unit ``u`` and
    operands rounded to a type of half unit ``half`` (see the tests)."""
    x, gate, up, dy = (wide(v) for v in (x, gate, up, dy))
    K = x.shape[1]
    # Float32 operands go in as three parts, six products of which are summed: six times the
    # additions, and 2 u of a product left out.
    times = 6 if half == 0 else 1
    sums = 2 * times * (K + 2) * u
    g, w = x @ gate.t(), x @ up.t()
    eg, ew = sums * (x.abs() @ gate.abs().t()), sums * (x.abs() @ up.abs().t())
    value, slope = activated(g, activation)
    # |f'| <= 1.13 and |f''| <= 0.8 for both.  A value's own operations: silu's exponential is off
    # by |g| u and its other steps by 5 u; gelu's erfc is off by 8 u and, its argument by 2 u, by
    # twice g^2 u below zero.  The slope's are off by 16 u of 1 + |g|.
    ev = 1.13 * eg + (12 + g.abs() + 2 * g * g) * u * value.abs()
    es = 0.8 * eg + 16 * u * (1 + g.abs())
    bounds = {"y": ev * (w.abs() + ew) + value.abs() * ew + 2 * u * (value * w).abs()}
    dg, du = dy * w * slope, dy * value
    edg = dy.abs() * (ew * slope.abs() + (w.abs() + ew) * es) + 3 * u * dg.abs()
    edu = dy.abs() * ev + 2 * u * du.abs()
    edg, edu = edg + half * (dg.abs() + edg), edu + half * (du.abs() + edu)
    M, F = dy.shape
    bounds["x"] = (edg @ gate.abs() + edu @ up.abs()
                   + 2 * times * (2 * F + 2) * u * (dg.abs() @ gate.abs() + du.abs() @ up.abs()))
    bounds["gate"] = edg.t() @ x.abs() + 2 * times * (M + 2) * u * (dg.abs().t() @ x.abs())
    bounds["up"] = edu.t() @ x.abs() + 2 * times * (M + 2) * u * (du.abs().t() @ x.abs())
    return bounds


def philox(counter: int, offset: int, seed: int) -> list[int]:
    """Eight 16-bit numbers of one counter: Philox4x32, 10 rounds, in Python's integers."""
    word = 0xFFFFFFFF
    c = [counter & word, counter >> 32 & word, offset & word, offset >> 32 & word]
    k = [seed & word, seed >> 32 & word]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & word, (p >> 32) ^ c[3] ^ k[1], p & word]
        k = [(k[0] + 0x9E3779B9) & word, (k[1] + 0xBB67AE85) & word]
    return [part for v in c for part in (v & 0xFFFF, v >> 16)]


def kept(count: int, p: float, seed: int, offset: int = 0):
    numbers = [n for c in range(-(-count // 8)) for n in philox(c, offset, seed)][:count]
    return torch.tensor([n >= round(p * 65536) for n in numbers], dtype=torch.bool)


def q4_codes(x, group: int, symmetric: bool, dtype):
    """(codes, scales, zeros) of rows, step by step as the format says: float32 arithmetic, whose
    division is exactly rounded, and scales rounded to their type."""
    x = x.detach().float().cpu()
    rows, columns = x.shape
    groups = -(-columns // group)
    wide_x = torch.zeros(rows, groups * group)
    wide_x[:, :columns] = x
    parts = wide_x.view(rows, groups, group)
    low, high = parts.amin(-1).clamp(max=0), parts.amax(-1).clamp(min=0)
    finite = torch.isfinite(parts).all(-1)
    scale = torch.maximum(high, -low) / 7 if symmetric else high / 15 - low / 15
    scale = scale.to(dtype).float()
    good = finite & torch.isfinite(scale)
    some = good & (scale > 0)
    safe = torch.where(some, scale, torch.ones_like(scale))
    zero = torch.full_like(scale, 8.0) if symmetric else torch.where(
        some, torch.round(-low / safe).clamp(0, 15), torch.zeros_like(scale))
    zero_of = zero.unsqueeze(-1)
    codes = torch.where(some.unsqueeze(-1), (torch.round(parts / safe.unsqueeze(-1)) + zero_of)
                        .clamp(0, 15), torch.where(good.unsqueeze(-1), zero_of, 0.0))
    codes = torch.nan_to_num(codes).view(rows, -1)[:, :columns]
    scale = torch.where(good, scale, torch.full_like(scale, math.nan))
    return codes.to(torch.uint8), scale.to(dtype), zero.to(torch.uint8)


def q4_pack(codes):
    """Codes [N, K] as bytes [N, ceil(K/32) * 16]."""
    rows, columns = codes.shape
    room = torch.zeros(rows, -(-columns // 32) * 32, dtype=torch.uint8)
    room[:, :columns] = codes
    return room[:, 0::2] | (room[:, 1::2] << 4)


def q4_values(codes, scales, zeros, group: int):
    """Values [N, K] in float64 (zeros None: 8)."""
    columns = codes.shape[1]
    spread = lambda v: v.double().cpu().repeat_interleave(group, 1)[:, :columns]  # noqa: E731
    return (codes.double().cpu() - (8.0 if zeros is None else spread(zeros))) * spread(scales)
