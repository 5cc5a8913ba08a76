"""Workloads of the signal path around the network: convolution, scan and 4-bit products.

A signal becomes per-tick drives through dense projections in microscaled 4-bit
floating point, a short causal convolution per channel and a selective state space
scan; the network's rates are read out by another 4-bit projection.  Each pass is one
operator as a program calls it, in one of these kinds:

* ``conv_step`` / ``scan_step``: one tick, the carried history or state updated in place;
* ``conv`` / ``scan``: a whole signal of T ticks, outputs and the state it leaves;
* ``conv_train`` / ``scan_train``: the same with the gradients of every input;
* ``quantize``: float rows to 4-bit codes and block scales, and back to values;
* ``product``: float rows times a 4-bit weight (the rows are quantised on the way).

``own`` chooses between the package's kernels and the plain form: elementary torch
operations in float32, rounded once at the end.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PACKAGE = str(Path(__file__).resolve().parent.parent / "neurosim-gpu_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DEVICE = "cuda"
BLOCK = 32                                   # values per scale of the 4-bit format
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
# Magnitudes of the eight e2m1 codes; bit 3 of a code is the sign.
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases ---------------------------------------------------------------------------

def _signal(kind: str, ticks: int, batch: int, channels: int, dtype: str, **more) -> dict:
    return {"kind": kind, "ticks": ticks, "batch": batch, "channels": channels, "dtype": dtype,
            "ragged": False, **more}


def _rows(kind: str, rows: int, columns: int, dtype: str, **more) -> dict:
    return {"kind": kind, "rows": rows, "columns": columns, "dtype": dtype, **more}


def listed() -> list[dict]:
    def named(name: str, case: dict) -> dict:
        return {"name": name, **case}

    return [
        # One tick of a small encoder in closed loop with its network: latency only.
        named("conv_step_1k_b1", _signal("conv_step", 1, 1, 1024, "float32", taps=4)),
        # A batch of whole signals filtered for serving.
        named("conv_4k_b4", _signal("conv", 4096, 4, 4096, "bfloat16", taps=4)),
        # Fitting the filters on recordings of different lengths, odd sizes, float32.
        named("conv_train_ragged", _signal("conv_train", 1500, 7, 1031, "float32", taps=3,
                                           ragged=True)),
        # One tick of 32 encoders stepped side by side.
        named("scan_step_4k_b32", _signal("scan_step", 1, 32, 4096, "bfloat16", states=16,
                                          groups=1)),
        # One long recording, a single column: few rows, all of the work along time.
        named("scan_2k_t16k_b1", _signal("scan", 16384, 1, 2048, "bfloat16", states=16,
                                         groups=1)),
        # Fitting the integrators on a batch of signals: the largest scan.
        named("scan_train_4k_b8", _signal("scan_train", 2048, 8, 4096, "bfloat16", states=16,
                                          groups=1)),
        # The same on recordings of different lengths, three groups of channels, odd sizes, float32.
        named("scan_train_ragged", _signal("scan_train", 777, 5, 1500, "float32", states=8,
                                           groups=3, ragged=True)),
        # A chunk of rates of a data-derived network on its way to the read-out: odd width.
        named("quantize_31k_r64", _rows("quantize", 64, 31_013, "float32")),
        # Activations of a batch of signals before a projection.
        named("quantize_8k_r16k", _rows("quantize", 16384, 8192, "bfloat16")),
        # The drive of one tick of a 50,000-neuron network from 1024 channels: one row.
        named("product_50k_r1", _rows("product", 1, 1024, "float32", outputs=50_000)),
        # Rates of 50,000 neurons over 33 ticks read out to 1000 signals: few rows, long sums.
        named("product_readout_r33", _rows("product", 33, 50_000, "float32", outputs=1000)),
        # A batch of whole signals projected: the matrix cores' case.
        named("product_8k_r8k", _rows("product", 8192, 8192, "bfloat16", outputs=8192)),
    ]


def draw(rng) -> dict:
    def log_uniform(low: float, high: float) -> int:
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(("conv_step", "conv", "conv_train", "scan_step", "scan", "scan", "scan_train",
                       "scan_train", "quantize", "product", "product", "product"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    if kind == "quantize":
        columns = log_uniform(17, 60_000)
        rows = log_uniform(1, max(1, min(20_000, 100_000_000 // columns)))
        return _rows(kind, rows, columns, dtype)
    if kind == "product":
        columns, outputs = log_uniform(33, 50_000), log_uniform(17, 50_000)
        weight = columns * outputs
        if weight > 200_000_000:
            outputs = max(17, 200_000_000 // columns)
            weight = columns * outputs
        rows = min(rng.choice((1, 1, log_uniform(2, 64), log_uniform(65, 8000))),
                   max(1, 400_000_000_000 // weight))
        return _rows(kind, rows, columns, dtype, outputs=outputs)
    groups = rng.choice((1, 1, 1, 2, 3))
    channels = groups * max(1, log_uniform(64, 5000) // groups)
    more: dict = {"taps": rng.choice((2, 3, 4, 4))}
    if kind.startswith("scan"):
        more = {"states": rng.choice((4, 8, 16, 16, 16, 32)), "groups": groups}
    if kind.endswith("step"):
        return _signal(kind, 1, log_uniform(1, 128), channels, dtype, **more)
    batch = rng.choice((1, 1, 2, 3, 4, 5, 8, 16))
    most = {"conv": 60_000_000, "conv_train": 30_000_000, "scan": 30_000_000,
            "scan_train": 20_000_000}[kind] * (16 if "states" in more else 1)
    cost = batch * channels * more.get("states", 1)
    ticks = log_uniform(2, max(3, min(16_384, most // cost)))
    return _signal(kind, ticks, batch, channels, dtype, **{**more, "ragged": rng.random() < 0.3})


# ---- inputs, from the seed alone -----------------------------------------------------

class _Random:
    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed * 7919 + 23)

    def normal(self, *shape: int, scale: float = 1.0, dtype: torch.dtype = torch.float32):
        return (torch.randn(shape, generator=self.g, device=DEVICE) * scale).to(dtype)

    def uniform(self, *shape: int, low: float, high: float):
        return torch.rand(shape, generator=self.g, device=DEVICE) * (high - low) + low


def _lengths(case: dict, random: _Random):
    """Ticks of each column: whole, or (ragged) a spread with an empty and a one-tick column."""
    if not case["ragged"]:
        return None
    ticks, batch = case["ticks"], case["batch"]
    lengths = random.uniform(batch, low=0.3, high=1.0).mul(ticks).ceil().to(torch.int32)
    lengths = lengths.clamp_(0, ticks)
    if batch > 2:
        lengths[0], lengths[1] = 0, 1
    return lengths


def _quantized(x: torch.Tensor):
    """(codes uint8 [..., blocks * 16], scales uint8 [..., blocks]) of float rows."""
    width = x.shape[-1]
    blocks = -(-width // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - width)).unflatten(-1, (blocks, BLOCK))
    peak = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    # frexp: peak = m 2^k with m in [1/2, 1), so floor(log2 peak) = k - 1; 6 = 1.5 * 2^2.
    exponent = torch.where(peak > 0, torch.frexp(peak)[1] - 3, -127).clamp(-127, 127)
    scaled = torch.ldexp(x, -exponent.unsqueeze(-1))
    size = scaled.abs()
    # Each stretch of the grid is uniform; rounding half to even there is to the even code.
    code = torch.where(size < 2, torch.round(size * 2),
                       torch.where(size < 4, torch.round(size) + 2, torch.round(size / 2) + 4))
    code = code.clamp(max=7).to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)
    code = torch.where(finite.unsqueeze(-1), code, torch.zeros_like(code)).flatten(-2)
    scales = torch.where(finite, exponent + 127, 255).to(torch.uint8)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), scales.contiguous()


def _values(codes: torch.Tensor, scales: torch.Tensor, width: int, dtype=torch.float32):
    """The values that codes and scales stand for."""
    levels = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), dtype=dtype, device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    exponent = scales.to(torch.int32) - 127
    unit = torch.ldexp(torch.ones_like(exponent, dtype=dtype), exponent)
    unit = torch.where(scales == 255, torch.full_like(unit, math.nan), unit)
    values = levels[nibbles.long()].unflatten(-1, (scales.shape[-1], BLOCK)) * unit.unsqueeze(-1)
    return values.flatten(-2)[..., :width]


def prepare(case: dict, seed: int) -> dict:
    random, kind = _Random(seed), case["kind"]
    dtype = _DTYPES[case["dtype"]]
    if kind in ("quantize", "product"):
        # Rows of one signal differ in scale, and some channels stand out.
        x = random.normal(case["rows"], case["columns"])
        x *= torch.exp(random.normal(case["rows"], 1, scale=0.5))
        x *= torch.exp(random.normal(1, case["columns"], scale=0.7))
        state = {"case": case, "x": x.to(dtype)}
        if kind == "product":
            weight = random.normal(case["outputs"], case["columns"],
                                   scale=1 / math.sqrt(case["columns"]))
            # The weight as it is kept: packed codes, two to a byte, and block scales.
            state["codes"], state["scales"] = _quantized(weight)
            state["bias"] = random.normal(case["outputs"], scale=0.1)
        return state
    ticks, batch, n = case["ticks"], case["batch"], case["channels"]
    state = {"case": case, "lengths": _lengths(case, random)}
    if kind.startswith("conv"):
        taps = case["taps"]
        state |= {"x": random.normal(ticks, batch, n, dtype=dtype),
                  "weight": random.normal(n, taps, scale=1 / math.sqrt(taps)),
                  "bias": random.normal(n, scale=0.1),
                  "history": random.normal(taps - 1, batch, n, dtype=dtype)}
    else:
        s, groups = case["states"], case["groups"]
        # Decay rates 1..S, time steps from about 1e-3 to 0.1 moved by the signal.
        rates = torch.arange(1, s + 1, device=DEVICE, dtype=torch.float32).expand(n, s)
        base = torch.exp(random.uniform(n, low=math.log(1e-3), high=math.log(1e-1)))
        state |= {"x": random.normal(ticks, batch, n, dtype=dtype),
                  "delta": random.normal(ticks, batch, n, scale=0.5, dtype=dtype),
                  "z": random.normal(ticks, batch, n, dtype=dtype),
                  "A": -rates * torch.exp(random.normal(n, s, scale=0.1)),
                  "B": random.normal(ticks, batch, groups, s, dtype=dtype),
                  "C": random.normal(ticks, batch, groups, s, dtype=dtype),
                  "D": 1 + random.normal(n, scale=0.1),
                  "delta_bias": base + torch.log(-torch.expm1(-base)),
                  "state": random.normal(batch, n, s, scale=0.5)}
    if kind.endswith("train"):
        state["dy"] = random.normal(ticks, batch, n, dtype=dtype)
        if kind == "scan_train":
            state["dstate"] = random.normal(batch, n, case["states"], scale=0.1)
    return state


# ---- the plain form ------------------------------------------------------------------

def _valid(lengths, ticks: int, batch: int):
    """[T, B, 1] truth values: the ticks that belong to their column."""
    if lengths is None:
        return torch.ones(ticks, batch, 1, dtype=torch.bool, device=DEVICE)
    return (torch.arange(ticks, device=DEVICE).unsqueeze(1) < lengths).unsqueeze(-1)


def _silu_slope(x: torch.Tensor) -> torch.Tensor:
    gate = torch.sigmoid(x)
    return gate * (1 + x * (1 - gate))


def _plain_conv(state: dict, gradients: bool) -> dict:
    x, w, history = state["x"], state["weight"], state["history"]
    (ticks, batch, _), taps, dtype = x.shape, w.shape[1], x.dtype
    valid = _valid(state["lengths"], ticks, batch)
    longer = torch.cat((history, x)).float()
    windows = longer.unfold(0, taps, 1)                             # [T, B, N, W]
    pre = (windows * w).sum(-1) + state["bias"]
    y = torch.where(valid, pre * torch.sigmoid(pre), 0.0)
    ends = valid.sum(0).flatten()                                   # ticks of each column
    last = torch.arange(taps - 1, device=DEVICE).unsqueeze(1) + ends
    out = {"y": y.to(dtype),
           "history": longer[last, torch.arange(batch, device=DEVICE)].to(dtype)}
    if gradients:
        dpre = torch.where(valid, state["dy"].float() * _silu_slope(pre), 0.0)
        padded = torch.nn.functional.pad(dpre, (0, 0, 0, 0, taps - 1, taps - 1))
        dlonger = (padded.unfold(0, taps, 1) * w.flip(1)).sum(-1)
        out |= {"dx": dlonger[taps - 1:].to(dtype), "dhistory": dlonger[:taps - 1].to(dtype),
                "dweight": (dpre.unsqueeze(-1) * windows).sum((0, 1)), "dbias": dpre.sum((0, 1))}
    return out


def _prefix(decay: torch.Tensor, inject: torch.Tensor) -> torch.Tensor:
    """h[t] = decay[t] h[t-1] + inject[t] from h = 0, by doubling the stretch joined."""
    step = 1
    while step < decay.shape[0]:
        inject = torch.cat((inject[:step], torch.addcmul(inject[step:], decay[step:],
                                                         inject[:-step])))
        decay = torch.cat((decay[:step], decay[step:] * decay[:-step]))
        step *= 2
    return inject


def _plain_scan(state: dict, gradients: bool) -> dict:
    dtype, (ticks, batch, n) = state["x"].dtype, state["x"].shape
    A, skip, start = state["A"], state["D"], state["state"]
    valid = _valid(state["lengths"], ticks, batch)
    x, z, raw = (torch.where(valid, state[k].float(), 0.0) for k in ("x", "z", "delta"))
    raw = raw + state["delta_bias"]
    step = torch.where(valid, torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())), 0.0)
    groups = state["B"].shape[2]
    write, read = (torch.where(valid.unsqueeze(-1), state[k].float(), 0.0)
                   .repeat_interleave(n // groups, 2) for k in ("B", "C"))    # [T, B, N, S]
    decay = torch.exp(step.unsqueeze(-1) * A)
    inject = (step * x).unsqueeze(-1) * write
    inject[0] += decay[0] * start
    h = _prefix(decay, inject)
    del inject
    read_out = (h * read).sum(-1) + skip * x
    gate = z * torch.sigmoid(z)
    out = {"y": (read_out * gate).to(dtype), "state": h[-1].clone()}
    if not gradients:
        return out
    dy = torch.where(valid, state["dy"].float(), 0.0)
    gy = dy * gate

    def over_groups(value: torch.Tensor) -> torch.Tensor:
        return value.unflatten(2, (groups, n // groups)).sum(3).to(dtype)

    out |= {"dz": (dy * read_out * _silu_slope(z)).to(dtype), "dD": (gy * x).sum((0, 1)),
            "dC": over_groups(gy.unsqueeze(-1) * h)}
    back = gy.unsqueeze(-1) * read
    back[-1] += state["dstate"]
    # The adjoint runs from the last tick to the first, tick t taking the decay of tick t + 1.
    g = _prefix(torch.cat((torch.ones_like(decay[:1]), decay.flip(0)[:-1])), back.flip(0)).flip(0)
    del back
    out["dB"] = over_groups(g * (step * x).unsqueeze(-1))
    through = (g * write).sum(-1)
    out["dx"] = (step * through + skip * gy).to(dtype)
    out["dstate0"] = decay[0] * g[0]
    flow = g * torch.cat((start.unsqueeze(0), h[:-1])) * decay
    del g, h, decay
    draw_ = torch.where(valid, ((flow * A).sum(-1) + through * x) * torch.sigmoid(raw), 0.0)
    out["ddelta"], out["ddelta_bias"] = draw_.to(dtype), draw_.sum((0, 1))
    out["dA"] = (flow * step.unsqueeze(-1)).sum((0, 1))
    return out


def _plain(state: dict) -> dict:
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        dtype = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
        return {"values": _values(*_quantized(state["x"]), case["columns"]).to(dtype)}
    if kind == "product":
        width = case["columns"]
        rows = _values(*_quantized(state["x"]), width)
        weight = _values(state["codes"], state["scales"], width)
        return {"y": (rows @ weight.t() + state["bias"]).to(state["x"].dtype)}
    plain = _plain_conv if kind.startswith("conv") else _plain_scan
    out = plain(state, kind.endswith("train"))
    if kind.endswith("step"):
        carried = "history" if kind == "conv_step" else "state"
        out[carried] = state[carried].copy_(out[carried])
    return out


# ---- the package's operators ---------------------------------------------------------

def _own(state: dict) -> dict:
    import neurosim_gpu as ns

    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        dtype = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
        return {"values": ns.mx_dequantize(ns.mx_quantize(state["x"]), dtype)}
    if kind == "product":
        weight = ns.MXTensor(state["codes"], state["scales"], case["columns"])
        return {"y": ns.mx_product(state["x"], weight, bias=state["bias"])}
    if kind == "conv_step":
        y = ns.causal_conv_step(state["x"][0], state["weight"], state["bias"],
                                history=state["history"])
        return {"y": y.unsqueeze(0), "history": state["history"]}
    if kind == "scan_step":
        now = {k: state[k][0] for k in ("x", "delta", "B", "C", "z")}
        y = ns.selective_scan_step(now["x"], now["delta"], state["A"], now["B"], now["C"],
                                   state["D"], z=now["z"], delta_bias=state["delta_bias"],
                                   state=state["state"])
        return {"y": y.unsqueeze(0), "state": state["state"]}
    names = (("x", "weight", "bias", "history") if kind.startswith("conv") else
             ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"))
    leaves = {k: state[k] for k in names}
    if kind.endswith("train"):
        leaves = {k: v.detach().requires_grad_() for k, v in leaves.items()}
    if kind.startswith("conv"):
        y, history = ns.causal_conv(leaves["x"], leaves["weight"], leaves["bias"],
                                    history=leaves["history"], lengths=state["lengths"])
        out = {"y": y, "history": history}
    else:
        y, final = ns.selective_scan(leaves["x"], leaves["delta"], leaves["A"], leaves["B"],
                                     leaves["C"], leaves["D"], z=leaves["z"],
                                     delta_bias=leaves["delta_bias"], state=leaves["state"],
                                     lengths=state["lengths"])
        out = {"y": y, "state": final}
    if kind.endswith("train"):
        ends = (y,) if kind == "conv_train" else (y, final)
        seeds = (state["dy"],) if kind == "conv_train" else (state["dy"], state["dstate"])
        grads = dict(zip(names, torch.autograd.grad(ends, list(leaves.values()), seeds)))
        out = {k: v.detach() for k, v in out.items()}
        out |= {"dstate0" if k == "state" else "d" + k: v for k, v in grads.items()}
    return out


def run(state: dict) -> dict:
    out = _own(state) if own else _plain(state)
    return {k: out[k] for k in sorted(out)}


# ---- what a pass cannot do without -----------------------------------------------------

def work(case: dict) -> dict:
    kind, e = case["kind"], _BYTES[case["dtype"]]
    if kind == "quantize":
        values = case["rows"] * case["columns"]
        back = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": values * (e + back), "flops": 4 * values}
    if kind == "product":
        m, k, n = case["rows"], case["columns"], case["outputs"]
        blocks = -(-k // BLOCK)
        return {"bytes": m * k * e + n * blocks * 17 + 4 * n + m * n * e, "flops": 2 * m * n * k}
    t, b, n = case["ticks"], case["batch"], case["channels"]
    cells, train = t * b * n, kind.endswith("train")
    if kind.startswith("conv"):
        taps = case["taps"]
        carried = 2 * (taps - 1) * b * n * e
        return {"bytes": (4 if train else 2) * cells * e + (1 + train) * (carried + 4 * n * (taps + 1)),
                "flops": cells * ((6 * taps + 12) if train else 2 * taps + 4)}
    s, groups = case["states"], case["groups"]
    carried = 2 * 4 * b * n * s
    shared = 2 * t * b * groups * s * e
    return {"bytes": (8 if train else 4) * cells * e + (1 + train) * (shared + carried + 4 * n * (s + 2)),
            "flops": cells * (s * (20 if train else 7) + (40 if train else 12))}


# ---- the definitions in 64 bits --------------------------------------------------------

def _exact_block_values(x: torch.Tensor) -> torch.Tensor:
    """Rows rounded to the 4-bit format, each value by its distance to the sixteen levels."""
    rows, width = x.shape
    x = x.double()
    out = torch.empty_like(x)
    whole = width // BLOCK * BLOCK
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=x.device)
    ends = (levels[1:] + levels[:-1]) / 2

    def rounded(blocks: torch.Tensor) -> torch.Tensor:
        peak = blocks.abs().amax(-1, keepdim=True)
        power = torch.floor(torch.log2(peak))
        power = power - (torch.exp2(power) > peak).double() + (torch.exp2(power + 1) <= peak).double()
        unit = torch.exp2((power - 2).clamp(-127, 127))
        size = blocks.abs() / unit
        # At a midpoint the even code wins: below it for even codes, above it for odd ones.
        low = torch.bucketize(size, ends)
        up = (low < 7) & (low % 2 == 1) & (size == ends[low.clamp(max=6)])
        return torch.where(blocks < 0, -1.0, 1.0) * levels[low + up.long()] * unit

    if whole:
        out[:, :whole] = rounded(x[:, :whole].unflatten(1, (-1, BLOCK))).flatten(1)
    if whole < width:
        out[:, whole:] = rounded(x[:, whole:].unsqueeze(1)).squeeze(1)
    return out


def _exact_conv(state: dict, gradients: bool) -> dict:
    x, w = state["x"].double(), state["weight"].double()
    history, bias = state["history"].double(), state["bias"].double()
    (ticks, batch, _), taps = x.shape, w.shape[1]
    ends = [ticks] * batch if state["lengths"] is None else state["lengths"].tolist()
    out = {"y": torch.zeros_like(x), "history": torch.zeros_like(history)}
    if gradients:
        out |= {"dx": torch.zeros_like(x), "dhistory": torch.zeros_like(history),
                "dweight": torch.zeros_like(w), "dbias": torch.zeros_like(bias)}
    for b, end in enumerate(ends):
        line = torch.cat((history[:, b], x[:end, b]))
        pre = bias + sum(w[:, k] * line[k:k + end] for k in range(taps))
        gate = 1 / (1 + torch.exp(-pre))
        out["y"][:end, b] = pre * gate
        out["history"][:, b] = line[end:]
        if gradients:
            dpre = state["dy"][:end, b].double() * (gate + pre * gate * (1 - gate))
            dline = torch.zeros_like(line)
            for k in range(taps):
                dline[k:k + end] += w[:, k] * dpre
                out["dweight"][:, k] += (dpre * line[k:k + end]).sum(0)
            out["dbias"] += dpre.sum(0)
            out["dhistory"][:, b], out["dx"][:end, b] = dline[:taps - 1], dline[taps - 1:]
    return out


def _exact_scan(state: dict, gradients: bool) -> dict:
    wide = {k: state[k].double() for k in ("x", "delta", "z", "A", "B", "C", "D", "delta_bias",
                                           "state")}
    ticks, batch, n = wide["x"].shape
    groups = wide["B"].shape[2]
    of = torch.arange(n, device=DEVICE) // (n // groups)            # each channel's group
    ends = torch.full((batch,), ticks, device=DEVICE) if state["lengths"] is None else state["lengths"]
    h = wide["state"].clone()
    y = torch.zeros_like(wide["x"])
    kept = torch.empty(ticks if gradients else 0, *h.shape, dtype=torch.float64, device=DEVICE)

    def tick(t: int):
        live = (t < ends)[:, None]
        raw = wide["delta"][t] + wide["delta_bias"]
        step = torch.where(live, torch.logaddexp(raw, torch.zeros_like(raw)), 0.0)
        return live, raw, step, torch.exp(step[..., None] * wide["A"])

    def sloped(z):
        gate = 1 / (1 + torch.exp(-z))
        return z * gate, gate * (1 + z * (1 - gate))

    for t in range(ticks):
        live, _, step, decay = tick(t)
        if gradients:
            kept[t] = h
        h = decay * h + (step * wide["x"][t])[..., None] * wide["B"][t][:, of]
        inner = (wide["C"][t][:, of] * h).sum(-1) + wide["D"] * wide["x"][t]
        y[t] = torch.where(live, inner * sloped(wide["z"][t])[0], 0.0)
    out = {"y": y, "state": h.clone()}
    if not gradients:
        return out
    grads = {k: torch.zeros_like(wide[k]) for k in wide if k != "state"}
    g = state["dstate"].double().clone()
    for t in range(ticks - 1, -1, -1):
        live, raw, step, decay = tick(t)
        x, before = wide["x"][t], kept[t]
        write, read = wide["B"][t][:, of], wide["C"][t][:, of]
        gate, slope = sloped(wide["z"][t])
        dy = torch.where(live, state["dy"][t].double(), 0.0)
        gy = dy * gate
        inner = (read * h).sum(-1) + wide["D"] * x
        grads["z"][t] = dy * inner * slope
        grads["D"] += (gy * x).sum(0)
        grads["C"][t] = (gy[..., None] * h).unflatten(1, (groups, -1)).sum(2)
        g = g + gy[..., None] * read
        grads["B"][t] = (g * (step * x)[..., None]).unflatten(1, (groups, -1)).sum(2)
        grads["x"][t] = step * (g * write).sum(-1) + wide["D"] * gy
        flow = g * before * decay
        grads["A"] += (flow * step[..., None]).sum(0)
        d_raw = ((flow * wide["A"]).sum(-1) + x * (g * write).sum(-1)) / (1 + torch.exp(-raw))
        grads["delta"][t] = torch.where(live, d_raw, 0.0)
        g, h = decay * g, before
    out |= {"d" + k: v for k, v in grads.items()}
    out |= {"ddelta_bias": grads["delta"].sum((0, 1)), "dstate0": g}
    return out


def exact(case: dict, seed: int):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        out = {"values": _exact_block_values(state["x"])}
    elif kind == "product":
        weight = _values(state["codes"], state["scales"], case["columns"], torch.float64)
        out = {"y": _exact_block_values(state["x"]) @ weight.t() + state["bias"].double()}
    else:
        form = _exact_conv if kind.startswith("conv") else _exact_scan
        out = form(state, kind.endswith("train"))
    return {k: out[k] for k in sorted(out)}
