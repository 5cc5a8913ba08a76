"""Plain float64 restatements of the signal operators, for the tests.

``conv`` and ``scan`` give outputs and, for upstream gradients, the gradients of every
input from the formulas, one tick at a time.  With ``magnitude=True`` every term enters
with its absolute value: the sum of the absolute values of all the terms that make up a
result, to which rounding errors are proportional.
"""

from __future__ import annotations

import torch


def wide(value):
    return None if value is None else value.detach().double().cpu()


def ends_of(lengths, ticks: int, batch: int) -> list[int]:
    if lengths is None:
        return [ticks] * batch
    return [min(max(int(v), 0), ticks) for v in lengths.tolist()]


def silu(x):
    """(value, slope)."""
    gate = torch.sigmoid(x)
    return x * gate, gate * (1 + x * (1 - gate))


def softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def conv(x, weight, bias=None, history=None, lengths=None, activation="silu", dy=None, dlast=None,
         magnitude=False):
    x, weight, bias, history, dy, dlast = (wide(v) for v in (x, weight, bias, history, dy, dlast))
    (ticks, batch, n), taps = x.shape, weight.shape[1]
    bias = torch.zeros(n, dtype=torch.float64) if bias is None else bias
    history = torch.zeros(taps - 1, batch, n, dtype=torch.float64) if history is None else history
    size = torch.abs if magnitude else (lambda v: v)
    out = {"y": torch.zeros_like(x), "history": torch.zeros_like(history)}
    grads = {"x": torch.zeros_like(x), "weight": torch.zeros_like(weight),
             "bias": torch.zeros_like(bias), "history": torch.zeros_like(history)}
    for b, end in enumerate(ends_of(lengths, ticks, batch)):
        line = torch.cat((history[:, b], x[:end, b]))
        pre = bias + sum(weight[:, k] * line[k:k + end] for k in range(taps))
        value, slope = silu(pre) if activation == "silu" else (pre, torch.ones_like(pre))
        if magnitude:
            # The slope of silu is at most 1.1, so this bounds what errors of pre become.
            value = bias.abs() + sum((weight[:, k] * line[k:k + end]).abs() for k in range(taps))
        out["y"][:end, b] = value
        out["history"][:, b] = line[end:]
        if dy is None:
            continue
        q = size(dy[:end, b] * slope)
        if magnitude and activation == "silu":
            # The second derivative is at most 1/2: an error of pre moves the slope by that.
            q = size(dy[:end, b]) * (slope.abs() + value)
        dline = torch.zeros_like(line)
        for k in range(taps):
            dline[k:k + end] += size(weight[:, k]) * q
            grads["weight"][:, k] += (q * size(line[k:k + end])).sum(0)
        grads["bias"] += q.sum(0)
        if dlast is not None:
            dline[end:] += size(dlast[:, b])
        grads["history"][:, b], grads["x"][:end, b] = dline[:taps - 1], dline[taps - 1:]
    return out, grads


def scan(x, delta, A, B, C, D=None, z=None, delta_bias=None, soft=True, state=None, lengths=None,
         dy=None, dfinal=None, magnitude=False):
    x, delta, A, B, C, D, z, delta_bias, state, dy, dfinal = (
        wide(v) for v in (x, delta, A, B, C, D, z, delta_bias, state, dy, dfinal))
    ticks, batch, n = x.shape
    shape = B.shape
    B, C = (v if v.dim() == 4 else v.unsqueeze(2) for v in (B, C))
    groups, states = B.shape[2:]
    size = torch.abs if magnitude else (lambda v: v)
    ends = torch.tensor(ends_of(lengths, ticks, batch))
    live = (torch.arange(ticks)[:, None] < ends)[:, :, None]
    zero = torch.zeros((), dtype=torch.float64)
    x, delta = torch.where(live, x, zero), torch.where(live, delta, zero)
    B, C = (torch.where(live[..., None], v, zero).repeat_interleave(n // groups, 2) for v in (B, C))
    raw = delta + (0 if delta_bias is None else delta_bias)
    dt = torch.where(live, softplus(raw) if soft else raw, zero)
    slope = torch.sigmoid(raw) if soft else torch.ones_like(raw)
    gate, gate_slope = ((torch.ones_like(x), torch.zeros_like(x)) if z is None
                        else silu(torch.where(live, z, zero)))
    decay = torch.exp(dt[..., None] * A)
    skip = torch.zeros(n, dtype=torch.float64) if D is None else D
    h = torch.zeros(batch, n, states, dtype=torch.float64) if state is None else state
    h, x, B, C, skip = size(h), size(x), size(B), size(C), size(skip)
    step, gate, gate_slope, rate = size(dt), size(gate), size(gate_slope), size(A)
    kept, inner = [h], []
    for t in range(ticks):
        h = decay[t] * h + (step[t] * x[t])[..., None] * B[t]
        kept.append(h)
        inner.append((C[t] * h).sum(-1) + skip * x[t])
    inner = torch.stack(inner) if ticks else torch.zeros_like(x)
    out = {"y": torch.where(live, inner * gate, zero), "state": h}
    if dy is None:
        return out, None
    dy = size(torch.where(live, dy, zero))
    gy = dy * gate
    grads = {"x": torch.zeros_like(x), "delta": torch.zeros_like(x), "A": torch.zeros_like(A),
             "B": torch.zeros(ticks, batch, groups, states, dtype=torch.float64),
             "C": torch.zeros(ticks, batch, groups, states, dtype=torch.float64),
             "D": (gy * x).sum((0, 1)), "z": dy * inner * gate_slope}
    g = torch.zeros_like(h) if dfinal is None else size(dfinal)
    for t in range(ticks - 1, -1, -1):
        g = g + gy[t][..., None] * C[t]
        grads["C"][t] = (gy[t][..., None] * kept[t + 1]).unflatten(1, (groups, -1)).sum(2)
        grads["B"][t] = (g * (step[t] * x[t])[..., None]).unflatten(1, (groups, -1)).sum(2)
        through = (g * B[t]).sum(-1)
        grads["x"][t] = step[t] * through + skip * gy[t]
        flow = g * kept[t] * decay[t]
        grads["A"] += (flow * step[t][..., None]).sum(0)
        d_raw = ((flow * rate).sum(-1) + x[t] * through) * slope[t]
        grads["delta"][t] = torch.where(live[t], d_raw, zero)
        g = g * decay[t]
    grads |= {"delta_bias": grads["delta"].sum((0, 1)), "state": g}
    grads["B"], grads["C"] = grads["B"].reshape(shape), grads["C"].reshape(shape)
    return out, grads


# ---- microscaled 4-bit rows ------------------------------------------------------------

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def mx_quantize(x):
    """(codes uint8 [..., blocks * 32] one per value, scale bytes [..., blocks]), value by value."""
    x = wide(x)
    width = x.shape[-1]
    blocks = -(-width // 32)
    x = torch.nn.functional.pad(x, (0, 32 * blocks - width)).unflatten(-1, (blocks, 32))
    bad = ~torch.isfinite(x).all(-1)
    peak = torch.where(bad, torch.ones((), dtype=torch.float64), x.abs().amax(-1))
    # Powers of two found by comparison: the largest one not above the peak.
    powers = torch.exp2(torch.arange(-149, 128, dtype=torch.float64))
    place = torch.searchsorted(powers, peak, right=True) - 1            # -1: peak 0
    exponent = (place - 149 - 2).clamp(-127, 127)
    exponent = torch.where(place < 0, torch.full_like(exponent, -127), exponent)
    size = x.abs() / torch.exp2(exponent.double()).unsqueeze(-1)
    gap = (size.unsqueeze(-1) - LEVELS).abs()
    best = gap.amin(-1, keepdim=True)
    tied = gap == best                                                  # one or two levels
    code = torch.arange(8).where(tied, 8 + torch.arange(8))
    even = torch.where(tied & (torch.arange(8) % 2 == 0), torch.arange(8), 99).amin(-1)
    first = code.amin(-1)
    code = torch.where((tied.sum(-1) == 2) & (even < 99), even, first)
    code = code + 8 * torch.signbit(x)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    scales = torch.where(bad, torch.full_like(exponent, 255), exponent + 127)
    return code.to(torch.uint8).flatten(-2), scales.to(torch.uint8)


def mx_values(codes, scales, width: int):
    """Values of one-per-value codes and scale bytes."""
    codes, scales = codes.cpu(), scales.cpu()
    sign = torch.where(codes >= 8, -1.0, 1.0).double()
    unit = torch.exp2(scales.double() - 127)
    unit = torch.where(scales == 255, torch.full_like(unit, float("nan")), unit)
    values = (sign * LEVELS[(codes & 7).long()]).unflatten(-1, (scales.shape[-1], 32))
    return (values * unit.unsqueeze(-1)).flatten(-2)[..., :width]


def unpack(codes):
    """One code per value of packed bytes (even value low)."""
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
