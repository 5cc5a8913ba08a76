"""Workloads of a gated block in the signal path: recurrence, projection, dropout, 4-bit groups.

A block turns a signal [T, B, N] into per-tick drives: a gated linear recurrence over time,
a gated projection of each tick, dropout while it is fitted, and, served, projections whose
weights are 4-bit integers with a scale per group of columns while the rows stay floats.
Each pass is one operator as a program calls it, in one of these kinds:

* ``recur_step``: one tick, the carried state updated in place;
* ``recur`` / ``recur_train``: a whole signal of T ticks; with the gradients of every input;
* ``gated`` / ``gated_train``: activation(x gate^T) * (x up^T); with all gradients;
* ``drop`` / ``drop_train``: residual + dropped x; with the gradient of x;
* ``q4``: float rows times a weight of 4-bit groups.

``own`` chooses between the package's kernels and the plain form: elementary torch
operations in float32, rounded once at the end.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

_PACKAGE = str(Path(__file__).resolve().parent.parent / "neurosim-gpu_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DEVICE = "cuda"
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---- cases ---------------------------------------------------------------------------

def _recur(kind: str, ticks: int, batch: int, channels: int, dtype: str, *, gate: bool = True,
           ragged: bool = False) -> dict:
    return {"kind": kind, "ticks": ticks, "batch": batch, "channels": channels, "dtype": dtype,
            "gate": gate, "ragged": ragged}


def _gated(kind: str, rows: int, columns: int, width: int, dtype: str,
           activation: str = "silu") -> dict:
    return {"kind": kind, "rows": rows, "columns": columns, "width": width, "dtype": dtype,
            "activation": activation}


def _drop(kind: str, rows: int, columns: int, dtype: str, p: float, residual: bool) -> dict:
    return {"kind": kind, "rows": rows, "columns": columns, "dtype": dtype, "p": p,
            "residual": residual}


def _q4(rows: int, columns: int, outputs: int, group: int, dtype: str, zeros: bool = True) -> dict:
    return {"kind": "q4", "rows": rows, "columns": columns, "outputs": outputs, "group": group,
            "dtype": dtype, "zeros": zeros}


def listed() -> list[dict]:
    def named(name: str, case: dict) -> dict:
        return {"name": name, **case}

    return [
        # One tick of a small encoder in closed loop with its network: latency only.
        named("recur_step_1k_b1", _recur("recur_step", 1, 1, 1024, "float32")),
        # One long recording, a single column: all of the parallel work lies along time.
        named("recur_2k_t16k_b1", _recur("recur", 16384, 1, 2048, "bfloat16")),
        # Fitting the recurrence on a batch of signals: the largest scan.
        named("recur_train_4k_b8", _recur("recur_train", 2048, 8, 4096, "bfloat16")),
        # The same on recordings of different lengths, odd sizes, no output gate, float32.
        named("recur_train_ragged", _recur("recur_train", 777, 5, 1500, "float32", gate=False,
                                           ragged=True)),
        # Activations of that batch dropped and added to the residual stream, and back.
        named("drop_train_16k", _drop("drop_train", 16384, 4096, "bfloat16", 0.1, True)),
        # A ragged batch's activations, odd width, no residual.
        named("drop_4k_odd", _drop("drop", 3885, 1031, "float32", 0.25, False)),
        # One tick of the served block: one row, bound by the weights.
        named("gated_8k_r1", _gated("gated", 1, 4096, 8192, "bfloat16")),
        # Fitting the block in float32 on a ragged batch's ticks, odd sizes.
        named("gated_train_odd", _gated("gated_train", 3885, 1031, 1500, "float32", "gelu")),
        # Fitting the block on a batch of whole signals: the matrix cores' case.
        named("gated_train_8k_r8k", _gated("gated_train", 8192, 4096, 8192, "bfloat16")),
        # The drive of one tick of a 50,000-neuron network from 1024 channels: one row.
        named("q4_50k_r1", _q4(1, 1024, 50_000, 128, "float32")),
        # Rates of 50,000 neurons over 33 ticks read out to 1000 signals: long sums.
        named("q4_readout_r33", _q4(33, 50_000, 1000, 64, "bfloat16")),
        # One tick of 16 encoders side by side, symmetric codes, small groups.
        named("q4_8k_r16", _q4(16, 8192, 8192, 32, "float16", zeros=False)),
    ]


def draw(rng) -> dict:
    def log_uniform(low: float, high: float) -> int:
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(("recur_step", "recur", "recur", "recur_train", "recur_train", "drop",
                       "drop_train", "gated", "gated", "gated_train", "gated_train", "q4", "q4",
                       "q4"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    if kind.startswith("drop"):
        columns = log_uniform(17, 20_000)
        rows = log_uniform(1, max(2, min(20_000, 60_000_000 // columns)))
        return _drop(kind, rows, columns, dtype, rng.choice((0.05, 0.1, 0.3, 0.5)),
                     rng.random() < 0.5)
    if kind.startswith("gated"):
        columns, width = log_uniform(33, 8000), log_uniform(17, 10_000)
        most = (60_000_000_000 if dtype == "float32" else 250_000_000_000) // (columns * width)
        rows = rng.choice((1, log_uniform(2, 64), log_uniform(65, 9000))) if kind == "gated" \
            else log_uniform(2, 9000)
        return _gated(kind, max(1, min(rows, most)), columns, width, dtype,
                      rng.choice(("silu", "silu", "gelu")))
    if kind == "q4":
        columns, outputs = log_uniform(33, 50_000), log_uniform(17, 50_000)
        outputs = max(17, min(outputs, 200_000_000 // columns))
        rows = rng.choice((1, 1, log_uniform(2, 16), log_uniform(17, 64), log_uniform(65, 2000)))
        rows = max(1, min(rows, 100_000_000_000 // (columns * outputs)))
        return _q4(rows, columns, outputs, rng.choice((32, 64, 128, 128)), dtype,
                   rng.random() < 0.7)
    channels, batch = log_uniform(64, 6000), rng.choice((1, 1, 2, 3, 4, 5, 8, 16))
    gate = rng.random() < 0.6
    if kind == "recur_step":
        return _recur(kind, 1, log_uniform(1, 128), channels, dtype, gate=gate)
    most = 60_000_000 // (batch * channels)
    ticks = log_uniform(2, max(3, min(16_384, most)))
    return _recur(kind, ticks, batch, channels, dtype, gate=gate, ragged=rng.random() < 0.3)


# ---- inputs, from the seed alone -----------------------------------------------------

class _Random:
    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed * 6151 + 41)

    def normal(self, *shape: int, scale: float = 1.0, dtype: torch.dtype = torch.float32):
        return (torch.randn(shape, generator=self.g, device=DEVICE) * scale).to(dtype)

    def uniform(self, *shape: int, low: float = 0.0, high: float = 1.0):
        return torch.rand(shape, generator=self.g, device=DEVICE) * (high - low) + low


def _lengths(case: dict, random: _Random):
    """Ticks of each column: whole, or (ragged) a spread with an empty and a one-tick column."""
    if not case["ragged"]:
        return None
    ticks, batch = case["ticks"], case["batch"]
    lengths = random.uniform(batch, low=0.3).mul(ticks).ceil().to(torch.int32).clamp_(0, ticks)
    if batch > 2:
        lengths[0], lengths[1] = 0, 1
    return lengths


def prepare(case: dict, seed: int) -> dict:
    random, kind, dtype = _Random(seed), case["kind"], _DTYPES[case["dtype"]]
    state = {"case": case}
    if kind.startswith("recur"):
        shape = (case["ticks"], case["batch"], case["channels"])
        # Channels forget over three ticks to a few thousand, moved by the signal.
        rates = torch.exp(random.uniform(shape[2], low=math.log(1e-3), high=math.log(2.0)))
        state |= {"x": random.normal(*shape, dtype=dtype),
                  "forget": random.normal(*shape, dtype=dtype),
                  "write": random.normal(*shape, dtype=dtype),
                  "rates": rates, "z": random.normal(*shape, dtype=dtype) if case["gate"] else None,
                  "state": random.normal(*shape[1:], scale=0.5),
                  "lengths": _lengths(case, random)}
        if kind == "recur_train":
            state |= {"dy": random.normal(*shape, dtype=dtype),
                      "dstate": random.normal(*shape[1:], scale=0.1)}
    elif kind.startswith("gated"):
        rows, columns, width = case["rows"], case["columns"], case["width"]
        state |= {"x": random.normal(rows, columns, dtype=dtype),
                  "gate": random.normal(width, columns, scale=columns ** -0.5, dtype=dtype),
                  "up": random.normal(width, columns, scale=columns ** -0.5, dtype=dtype)}
        if kind == "gated_train":
            state["dy"] = random.normal(rows, width, dtype=dtype)
    elif kind.startswith("drop"):
        shape = (case["rows"], case["columns"])
        state |= {"x": random.normal(*shape, dtype=dtype), "seed": seed * 2_654_435_761 + 99,
                  "offset": seed % 1000,
                  "residual": random.normal(*shape, dtype=dtype) if case["residual"] else None}
        if kind == "drop_train":
            state["dy"] = random.normal(*shape, dtype=dtype)
    else:
        rows, columns, outputs = case["rows"], case["columns"], case["outputs"]
        groups, blocks = -(-columns // case["group"]), -(-columns // 32)
        # The weight as it is kept: codes two to a byte around their zero point, bf16 scales.
        zero = torch.randint(6, 10, (outputs, groups), generator=random.g, device=DEVICE,
                             dtype=torch.uint8)
        spread = torch.randn(outputs, blocks * 32, generator=random.g, device=DEVICE,
                             dtype=torch.bfloat16).mul_(2.7).add_(8).round_().clamp_(0, 15)
        code = spread.to(torch.uint8)
        # Rates and activations: few channels stand out, and the mean is not zero.
        x = random.normal(rows, columns) * torch.exp(random.normal(1, columns, scale=0.7)) + 0.2
        state |= {"x": x.to(dtype), "codes": code[:, 0::2] | (code[:, 1::2] << 4),
                  "scales": (torch.exp(random.normal(outputs, groups, scale=0.3))
                             * (0.4 * columns ** -0.5)).to(torch.bfloat16),
                  "zeros": zero if case["zeros"] else None,
                  "bias": random.normal(outputs, scale=0.1)}
    return state


# ---- the plain form ------------------------------------------------------------------

def _silu_slope(x: torch.Tensor) -> torch.Tensor:
    gate = torch.sigmoid(x)
    return gate * (1 + x * (1 - gate))


def _prefix(decay: torch.Tensor, inject: torch.Tensor) -> torch.Tensor:
    """h[t] = decay[t] h[t-1] + inject[t] from h = 0, by doubling the stretch joined."""
    step = 1
    while step < decay.shape[0]:
        inject = torch.cat((inject[:step], torch.addcmul(inject[step:], decay[step:],
                                                         inject[:-step])))
        decay = torch.cat((decay[:step], decay[step:] * decay[:-step]))
        step *= 2
    return inject


def _plain_recur(state: dict, gradients: bool) -> dict:
    dtype, (ticks, batch, _) = state["x"].dtype, state["x"].shape
    start, z = state["state"], state["z"]
    valid = torch.ones(ticks, batch, 1, dtype=torch.bool, device=DEVICE) \
        if state["lengths"] is None \
        else (torch.arange(ticks, device=DEVICE).unsqueeze(1) < state["lengths"]).unsqueeze(-1)
    x = torch.where(valid, state["x"].float(), 0.0)
    opened, written = torch.sigmoid(state["forget"].float()), torch.sigmoid(state["write"].float())
    fade = torch.where(valid, opened * state["rates"], 0.0)       # -log of the decay
    decay, room = torch.exp(-fade), torch.sqrt(-torch.expm1(-2 * fade))
    inject = room * written * x
    inject[0] += decay[0] * start
    h = _prefix(decay, inject)
    gate = 1.0 if z is None else torch.nn.functional.silu(z.float())
    out = {"y": torch.where(valid, h * gate, 0.0).to(dtype), "state": h[-1].clone()}
    if not gradients:
        return out
    dy = torch.where(valid, state["dy"].float(), 0.0)
    if z is not None:
        out["dz"] = torch.where(valid, dy * h * _silu_slope(z.float()), 0.0).to(dtype)
    back = dy * gate
    back[-1] += state["dstate"]
    # The adjoint runs from the last tick to the first, tick t taking the decay of tick t + 1.
    g = _prefix(torch.cat((torch.ones_like(decay[:1]), decay.flip(0)[:-1])), back.flip(0)).flip(0)
    before = torch.cat((start.unsqueeze(0), h[:-1]))
    out["dx"] = (g * room * written).to(dtype)
    out["dwrite"] = (g * room * x * written * (1 - written)).to(dtype)
    slope = torch.where(valid, decay * decay / room.clamp(min=1e-30), 0.0) * written * x
    dfade = g * (slope - decay * before)
    out["dforget"] = (dfade * fade * (1 - opened)).to(dtype)
    out["drates"] = torch.where(valid, dfade * opened, 0.0).sum((0, 1))
    out["dstate0"] = decay[0] * g[0]
    return out


def _activated(x: torch.Tensor, activation: str):
    """(value, slope) of the activation."""
    if activation == "silu":
        return x * torch.sigmoid(x), _silu_slope(x)
    below = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    return x * below, below + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))


def _plain_gated(state: dict, gradients: bool) -> dict:
    dtype = state["x"].dtype
    x, gate, up = (state[k].float() for k in ("x", "gate", "up"))
    raised = x @ up.t()
    value, slope = _activated(x @ gate.t(), state["case"]["activation"])
    out = {"y": (value * raised).to(dtype)}
    if gradients:
        dy = state["dy"].float()
        draised, dgated = dy * value, dy * raised * slope
        out |= {"dx": (dgated @ gate + draised @ up).to(dtype),
                "dgate": (dgated.t() @ x).to(dtype), "dup": (draised.t() @ x).to(dtype)}
    return out


_WORD = 0xFFFFFFFF


def _wide_product(a: torch.Tensor, m: int):
    """(high, low) words of a * m for 32-bit words held in int64."""
    low, high = (a & 0xFFFF) * m, (a >> 16) * m              # each below 2^48
    total = (low >> 16) + high
    return total >> 16, ((total & 0xFFFF) << 16) | (low & 0xFFFF)


def _kept(count: int, p: float, seed: int, offset: int) -> torch.Tensor:
    """Truth values of ``count`` elements: eight 16-bit numbers from each counter of
    Philox4x32 with 10 rounds (Salmon et al. 2011), kept from p on."""
    at = torch.arange(-(-count // 8), device=DEVICE)
    c = [at & _WORD, at >> 32, torch.full_like(at, offset & _WORD),
         torch.full_like(at, offset >> 32 & _WORD)]
    key = [seed & _WORD, seed >> 32 & _WORD]
    for _ in range(10):
        high0, low0 = _wide_product(c[0], 0xD2511F53)
        high1, low1 = _wide_product(c[2], 0xCD9E8D57)
        c = [high1 ^ c[1] ^ key[0], low1, high0 ^ c[3] ^ key[1], low0]
        key = [(key[0] + 0x9E3779B9) & _WORD, (key[1] + 0xBB67AE85) & _WORD]
    halves = torch.stack([part for word in c for part in (word & 0xFFFF, word >> 16)], -1)
    return halves.flatten()[:count] >= round(p * 65536)


def _plain_drop(state: dict, gradients: bool) -> dict:
    x, case = state["x"], state["case"]
    kept = _kept(x.numel(), case["p"], state["seed"], state["offset"]).view_as(x)
    scale = 65536 / (65536 - round(case["p"] * 65536))
    y = torch.where(kept, x.float() * scale, 0.0)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    out = {"y": y.to(x.dtype)}
    if gradients:
        out["dx"] = torch.where(kept, state["dy"].float() * scale, 0.0).to(x.dtype)
    return out


def _plain_q4(state: dict) -> dict:
    case, codes = state["case"], state["codes"]
    columns, group = case["columns"], case["group"]
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[:, :columns].to(torch.float32)
    zero = 8.0 if state["zeros"] is None \
        else state["zeros"].float().repeat_interleave(group, 1)[:, :columns]
    scale = state["scales"].float().repeat_interleave(group, 1)[:, :columns]
    weight = (code - zero) * scale
    return {"y": (state["x"].float() @ weight.t() + state["bias"]).to(state["x"].dtype)}


def _plain(state: dict) -> dict:
    kind = state["case"]["kind"]
    if kind == "q4":
        return _plain_q4(state)
    form = {"r": _plain_recur, "g": _plain_gated, "d": _plain_drop}[kind[0]]
    out = form(state, kind.endswith("train"))
    if kind == "recur_step":
        out["state"] = state["state"].copy_(out["state"])
    return out


# ---- the package's operators ---------------------------------------------------------

def _with_gradients(names, state: dict, call, seeds) -> dict:
    """Outputs of ``call`` on the named inputs, and the inputs' gradients."""
    leaves = {k: state[k].detach().requires_grad_() for k in names if state[k] is not None}
    ends = call({k: leaves.get(k) for k in names})
    grads = torch.autograd.grad(ends, list(leaves.values()), seeds)
    return {k: v for k, v in zip(("y", "state"), (v.detach() for v in ends))} \
        | {"dstate0" if k == "state" else "d" + k: v for k, v in zip(leaves, grads)}


def _own(state: dict) -> dict:
    import neurosim_gpu as ns

    case, kind = state["case"], state["case"]["kind"]
    if kind == "q4":
        weight = ns.Q4Tensor(state["codes"], state["scales"], state["zeros"], case["columns"],
                             case["group"])
        return {"y": ns.q4_product(state["x"], weight, bias=state["bias"])}
    if kind == "recur_step":
        z = state["z"]
        y = ns.gated_recurrence_step(state["x"][0], state["forget"][0], state["write"][0],
                                     state["rates"], z=None if z is None else z[0],
                                     state=state["state"])
        return {"y": y.unsqueeze(0), "state": state["state"]}
    if kind.startswith("recur"):
        def recur(v):
            return ns.gated_recurrence(v["x"], v["forget"], v["write"], v["rates"], z=v["z"],
                                       state=v["state"], lengths=state["lengths"])

        names = ("x", "forget", "write", "rates", "z", "state")
        if kind == "recur_train":
            return _with_gradients(names, state, recur, (state["dy"], state["dstate"]))
        return dict(zip(("y", "state"), recur(state)))
    if kind.startswith("gated"):
        def gated(v):
            return (ns.gated_projection(v["x"], v["gate"], v["up"],
                                        activation=case["activation"]),)

        if kind == "gated_train":
            return _with_gradients(("x", "gate", "up"), state, gated, (state["dy"],))
        return {"y": gated(state)[0]}

    def drop(v):
        return (ns.dropout(v["x"], case["p"], seed=state["seed"], offset=state["offset"],
                           residual=state["residual"]),)

    if kind == "drop_train":
        return _with_gradients(("x",), state, drop, (state["dy"],))
    return {"y": drop(state)[0]}


def run(state: dict) -> dict:
    out = _own(state) if own else _plain(state)
    return {k: out[k] for k in sorted(out)}


# ---- what a pass cannot do without -----------------------------------------------------

def work(case: dict) -> dict:
    kind, e, train = case["kind"], _BYTES[case["dtype"]], case["kind"].endswith("train")
    if kind.startswith("recur"):
        lines = case["batch"] * case["channels"]
        cells, streams = case["ticks"] * lines, 4 + case["gate"]
        # Backwards the inputs are read once more with dy, and each has a gradient.
        bytes_ = cells * e * (streams + train * (2 * streams - 1)) + (8 + 8 * train) * lines
        return {"bytes": bytes_ + 4 * case["channels"] * (1 + train),
                "flops": cells * (60 if train else 20)}
    if kind.startswith("gated"):
        m, k, f = case["rows"], case["columns"], case["width"]
        bytes_ = (m * k + 2 * f * k + m * f) * e
        return {"bytes": bytes_ * (2 if train else 1), "flops": 4 * m * k * f * (3 if train else 1)}
    cells = case["rows"] * case["columns"]
    if kind.startswith("drop"):
        return {"bytes": cells * e * (2 + case["residual"] + 2 * train),
                "flops": cells * (30 if train else 15)}
    k, n = case["columns"], case["outputs"]
    groups = -(-k // case["group"])
    return {"bytes": cells * e + n * -(-k // 32) * 16 + n * groups * (3 if case["zeros"] else 2)
            + 4 * n + case["rows"] * n * e, "flops": 2 * cells * n}


# ---- the definitions in 64 bits --------------------------------------------------------

def _exact_recur(state: dict, gradients: bool) -> dict:
    x, forget, write, rates = (state[k].double() for k in ("x", "forget", "write", "rates"))
    ticks, batch, n = x.shape
    z = None if state["z"] is None else state["z"].double()
    ends = torch.full((batch,), ticks, device=DEVICE) if state["lengths"] is None \
        else state["lengths"]

    def tick(t: int):
        live = (t < ends)[:, None]
        r, i = 1 / (1 + torch.exp(-forget[t])), 1 / (1 + torch.exp(-write[t]))
        a = torch.exp(-rates * r)
        return live, r, i, a, torch.sqrt((1 - a) * (1 + a))

    def gated(t: int):
        if z is None:
            return torch.ones_like(x[t]), torch.zeros_like(x[t])
        s = 1 / (1 + torch.exp(-z[t]))
        return z[t] * s, s + z[t] * s * (1 - s)

    h, y = state["state"].double(), torch.zeros_like(x)
    kept = []
    for t in range(ticks):
        live, _, i, a, room = tick(t)
        if gradients:
            kept.append(h)
        h = torch.where(live, a * h + room * i * x[t], h)
        y[t] = torch.where(live, h * gated(t)[0], 0.0)
    out = {"y": y, "state": h}
    if not gradients:
        return out
    grads = {k: torch.zeros_like(x) for k in ("dx", "dforget", "dwrite", "dz")}
    drates, g, after = torch.zeros_like(rates), state["dstate"].double(), h
    for t in range(ticks - 1, -1, -1):
        live, r, i, a, room = tick(t)
        gate, slope = gated(t)
        dy = torch.where(live, state["dy"][t].double(), 0.0)
        grads["dz"][t] = dy * after * slope
        g = g + dy * gate
        grads["dx"][t] = torch.where(live, g * room * i, 0.0)
        grads["dwrite"][t] = torch.where(live, g * room * x[t] * i * (1 - i), 0.0)
        # With a = exp(-rate r): da = -a d(rate r), d sqrt(1 - a^2) = a^2 / room d(rate r).
        dfade = torch.where(live, g * (a * a / room * i * x[t] - a * kept[t]), 0.0)
        grads["dforget"][t] = dfade * rates * r * (1 - r)
        drates += (dfade * r).sum(0)
        g, after = torch.where(live, a * g, g), kept[t]
    if z is None:
        del grads["dz"]
    return out | grads | {"drates": drates, "dstate0": g}


def _exact_gated(state: dict, gradients: bool) -> dict:
    x, gate, up = (state[k].double() for k in ("x", "gate", "up"))
    pre, raised = torch.matmul(x, gate.T), torch.matmul(x, up.T)
    if state["case"]["activation"] == "silu":
        s = 1 / (1 + torch.exp(-pre))
        value, slope = pre * s, s + pre * s * (1 - s)
    else:
        s = torch.special.ndtr(pre)
        value, slope = pre * s, s + pre * torch.exp(-pre.square() / 2) / math.sqrt(2 * math.pi)
    out = {"y": value * raised}
    if gradients:
        dy = state["dy"].double()
        dpre, draised = dy * raised * slope, dy * value
        out |= {"dx": torch.matmul(dpre, gate) + torch.matmul(draised, up),
                "dgate": torch.matmul(x.T, dpre).T, "dup": torch.matmul(x.T, draised).T}
    return out


def _exact_drop(state: dict, gradients: bool) -> dict:
    x, p = state["x"], state["case"]["p"]
    count = x.numel()
    mask, low32 = np.uint64(_WORD), np.uint64(32)
    at = np.arange(-(-count // 8), dtype=np.uint64)
    words = [at & mask, at >> low32, np.full_like(at, state["offset"] & _WORD),
             np.full_like(at, state["offset"] >> 32 & _WORD)]
    k0, k1 = state["seed"] & _WORD, state["seed"] >> 32 & _WORD
    for _ in range(10):
        p0, p1 = words[0] * np.uint64(0xD2511F53), words[2] * np.uint64(0xCD9E8D57)
        words = [(p1 >> low32) ^ words[1] ^ np.uint64(k0), p1 & mask,
                 (p0 >> low32) ^ words[3] ^ np.uint64(k1), p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & _WORD, (k1 + 0xBB67AE85) & _WORD
    numbers = np.stack(words, 1).astype("<u4").view("<u2").reshape(-1)[:count]
    first = int(p * 65536 + 0.5)
    factor = torch.from_numpy(numbers >= first).to(DEVICE).view(x.shape).double() \
        / (1 - first / 65536)
    rest = 0 if state["residual"] is None else state["residual"].double()
    out = {"y": rest + x.double() * factor}
    if gradients:
        out["dx"] = state["dy"].double() * factor
    return out


def _exact_q4(state: dict) -> dict:
    case, x = state["case"], state["x"].double()
    columns, group = case["columns"], case["group"]
    out = state["bias"].double().expand(case["rows"], -1).clone()
    for g, first in enumerate(range(0, columns, group)):
        last = min(first + group, columns)
        bytes_ = state["codes"][:, first // 2:(last + 1) // 2].long()
        whole = torch.empty(bytes_.shape[0], 2 * bytes_.shape[1], dtype=torch.float64,
                            device=DEVICE)
        whole[:, 0::2], whole[:, 1::2] = (bytes_ % 16).double(), (bytes_ // 16).double()
        whole = whole[:, :last - first]
        zero = 8 if state["zeros"] is None else state["zeros"][:, g:g + 1].double()
        out += (x[:, first:last] @ (whole - zero).T) * state["scales"][:, g].double()
    return {"y": out}


def exact(case: dict, seed: int):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "q4":
        out = _exact_q4(state)
    else:
        form = {"r": _exact_recur, "g": _exact_gated, "d": _exact_drop}[kind[0]]
        out = form(state, kind.endswith("train"))
    return {k: out[k] for k in sorted(out)}
