"""Signals into per-tick drives, and rates into read-outs.

``SignalEncoder`` turns a signal [T, B, F] into the somatic drives [T, B, N] of a network:

    projection F -> 2C (values and gates), a short causal convolution per channel, a
    projection to each channel's time step and the shared B and C, a selective scan, and
    a projection C -> N.

With ``mixer="gated"`` a gated linear recurrence takes the scan's place (and the projection
gives each channel's two gates), and with ``feed_forward`` W a gated block of that width,
y + W_down (silu(W_gate y) * (W_up y)), follows it; a ``Dropout`` passed to ``drives`` drops
parts of what the block adds while the encoder is fitted.

It runs in two forms.  With its float32 parameters every step has gradients, so it is
fitted through recorded ticks of a ``NativeDendriticMatrixRuntime``; ``quantized()`` gives
the serving form, whose projections hold their weights in 4 bits (microscaled floats, whose
products quantise the signal too, or integers with a scale per group, whose do not; the
block's two gated projections stay as they are), with whole signals (``drives``, staged into a
``MatrixRollout``) and single ticks in closed loop (``step``).  ``ReadOut`` is a 4-bit
projection of rates.

    python -m neurosim_gpu.signal_encoder [--neurons 1024 ...]

fits an encoder so that a network's rates follow a target, quantises it, rolls the network
out under both forms' drives and prints what the 4 bits change, as JSON.
"""

from __future__ import annotations

import argparse
import json
import math

import torch

from .block_ops import dropout, gated_projection
from .compartmental import DendriticDynamics
from .dynamics import Dynamics
from .group_scaled import q4_product, q4_quantize
from .microscaled import mx_product, mx_quantize
from .native_compartmental import NativeDendriticMatrixRuntime
from .rollout import MatrixRollout
from .signal_ops import (causal_conv, causal_conv_step, gated_recurrence, gated_recurrence_step,
                         selective_scan, selective_scan_step)
from .topology import random_topology

_PROJECTIONS = ("project_in", "project_step", "project_down", "project_out")
MIXERS = ("scan", "gated")
# How a weight is held in 4 bits, and what multiplies it.
FORMATS = {"mx": (mx_quantize, mx_product), "q4": (q4_quantize, q4_product)}


class Dropout:
    """What a fit drops: each element with probability ``p``, by masks of its own in every pass
    (``next`` moves on to another one's)."""

    def __init__(self, p: float, seed: int = 0) -> None:
        self.p, self.seed, self.offset = p, seed, 0

    def next(self) -> None:
        self.offset += 1

    def __call__(self, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        return dropout(x, self.p, seed=self.seed, offset=self.offset, residual=residual)


class _Encoder:
    """What the float and the 4-bit form share; ``_project`` is theirs."""

    def __init__(self, parameters: dict, channels: int, states: int, groups: int,
                 mixer: str = "scan") -> None:
        self.parameters = parameters
        self.channels, self.states, self.groups, self.mixer = channels, states, groups, mixer

    @property
    def device(self) -> torch.device:
        return self.parameters["conv_weight"].device

    @property
    def taps(self) -> int:
        return self.parameters["conv_weight"].shape[1]

    def _project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        raise NotImplementedError

    def initial(self, batch: int, dtype: torch.dtype = torch.float32
                ) -> tuple[torch.Tensor, torch.Tensor]:
        """The carried (history, state) before a signal of type ``dtype``: zeros."""
        state = (batch, self.channels) if self.mixer == "gated" else (batch, self.channels, self.states)
        return (torch.zeros(self.taps - 1, batch, self.channels, dtype=dtype, device=self.device),
                torch.zeros(state, device=self.device))

    def _scan_inputs(self, x: torch.Tensor):
        """(delta, B, C) of filtered values [..., C]: slices of one projection, not copied."""
        both = self._project("project_step", x)
        lead, wide = x.shape[:-1], self.groups * self.states
        delta, write, read = both.split((self.channels, wide, wide), -1)
        shape = (*lead, self.groups, self.states)
        return delta, write.unflatten(-1, shape[-2:]), read.unflatten(-1, shape[-2:])

    def _block(self, y: torch.Tensor, drop: Dropout | None = None) -> torch.Tensor:
        """The gated block after the mixer, where there is one."""
        p = self.parameters
        if "block_gate" not in p:
            if drop is not None:
                raise ValueError("dropout acts on the gated block, which this encoder lacks")
            return y
        inner = gated_projection(y.to(p["block_gate"].dtype), p["block_gate"], p["block_up"])
        more = self._project("project_down", inner).to(y.dtype)
        return y + more if drop is None else drop(more, y)

    def drives(self, signal: torch.Tensor, carried=None, lengths: torch.Tensor | None = None,
               drop: Dropout | None = None):
        """Drives [T, B, N] of a signal [T, B, F], and the carried (history, state) after it."""
        p = self.parameters
        history, state = (self.initial(signal.shape[1], signal.dtype) if carried is None
                          else carried)
        x, gate = self._project("project_in", signal).chunk(2, -1)
        x, history = causal_conv(x, p["conv_weight"], p["conv_bias"], history=history,
                                 lengths=lengths)
        if self.mixer == "gated":
            forget, write = self._project("project_step", x).chunk(2, -1)
            y, state = gated_recurrence(x, forget, write, torch.exp(p["log_rates"]), z=gate,
                                        state=state, lengths=lengths)
        else:
            delta, write, read = self._scan_inputs(x)
            y, state = selective_scan(x, delta, -torch.exp(p["log_rates"]), write, read, p["skip"],
                                      z=gate, delta_bias=p["step_bias"], state=state,
                                      lengths=lengths)
        return self._project("project_out", self._block(y, drop)), (history, state)


class SignalEncoder(_Encoder):
    """Float32 encoder with gradients (see the module); parameters are drawn from ``seed``."""

    def __init__(self, features: int, channels: int, neurons: int, *, states: int = 16,
                 groups: int = 1, taps: int = 4, mixer: str = "scan", feed_forward: int = 0,
                 device="cuda", seed: int = 0) -> None:
        if min(features, channels, neurons, states, groups, taps) <= 0 or channels % groups:
            raise ValueError("sizes must be positive and the groups divide the channels")
        if mixer not in MIXERS or feed_forward < 0:
            raise ValueError("the mixer is 'scan' or 'gated', the feed-forward width not negative")
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, scale):
            return torch.randn(shape, generator=g) * scale

        # Time steps from 1e-3 to 0.1 and decay rates 1 .. S per channel.
        steps = torch.exp(torch.rand(channels, generator=g) * math.log(100) + math.log(1e-3))
        values = {
            "project_in": normal(2 * channels, features, scale=features ** -0.5),
            "conv_weight": normal(channels, taps, scale=taps ** -0.5),
            "conv_bias": torch.zeros(channels),
            "project_step": normal(channels + 2 * groups * states, channels,
                                   scale=channels ** -0.5),
            "step_bias": steps + torch.log(-torch.expm1(-steps)),
            "log_rates": torch.log(torch.arange(1, states + 1.0)).repeat(channels, 1),
            "skip": torch.ones(channels),
            "project_out": normal(neurons, channels, scale=0.3 * channels ** -0.5),
        }
        if mixer == "gated":
            # Gates half open: channels forget over two to a thousand ticks.
            values["project_step"] = normal(2 * channels, channels, scale=channels ** -0.5)
            spread = torch.rand(channels, generator=g) * math.log(500)
            values["log_rates"] = spread + math.log(2e-3)
            del values["step_bias"], values["skip"]
        if feed_forward:
            values |= {"block_gate": normal(feed_forward, channels, scale=channels ** -0.5),
                       "block_up": normal(feed_forward, channels, scale=channels ** -0.5),
                       "project_down": normal(channels, feed_forward,
                                              scale=0.5 * feed_forward ** -0.5)}
        super().__init__({k: v.to(device).requires_grad_() for k, v in values.items()},
                         channels, states, groups, mixer)

    def _project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return x @ self.parameters[name].t()

    def quantized(self, weights: str = "mx", *, block: torch.dtype = torch.float32
                  ) -> "QuantizedEncoder":
        """The serving form of the present parameters, its projections in 4 bits: "mx"
        (microscaled floats) or "q4" (integers with group scales).  ``block`` is the type of
        the gated block's two gated projections."""
        if weights not in FORMATS:
            raise ValueError("weights are held as 'mx' or 'q4'")
        quantize = FORMATS[weights][0]
        values = {k: quantize(v.detach()) if k in _PROJECTIONS else v.detach().clone()
                  for k, v in self.parameters.items()}
        values |= {k: values[k].to(block) for k in ("block_gate", "block_up") if k in values}
        return QuantizedEncoder(values, self.channels, self.states, self.groups, self.mixer, weights)


class QuantizedEncoder(_Encoder):
    """Encoder with 4-bit projections, for serving."""

    def __init__(self, parameters: dict, channels: int, states: int, groups: int,
                 mixer: str = "scan", weights: str = "mx") -> None:
        super().__init__(parameters, channels, states, groups, mixer)
        rates = torch.exp(parameters["log_rates"])
        self._rates = rates if mixer == "gated" else -rates
        self._product = FORMATS[weights][1]

    def _project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return self._product(x, self.parameters[name])

    def step(self, signal: torch.Tensor, carried) -> torch.Tensor:
        """Drives [B, N] of one tick [B, F]; ``carried`` (``initial``) moves on in place."""
        p, (history, state) = self.parameters, carried
        x, gate = self._project("project_in", signal).chunk(2, -1)
        x = causal_conv_step(x, p["conv_weight"], p["conv_bias"], history=history)
        if self.mixer == "gated":
            forget, write = self._project("project_step", x).chunk(2, -1)
            y = gated_recurrence_step(x, forget, write, self._rates, z=gate, state=state)
        else:
            delta, write, read = self._scan_inputs(x)
            y = selective_scan_step(x, delta, self._rates, write, read, p["skip"], z=gate,
                                    delta_bias=p["step_bias"], state=state)
        return self._project("project_out", self._block(y))


class ReadOut:
    """Outputs [..., K] of rates [..., N]: a projection ``weight`` [K, N] held in 4 bits, "mx" or
    "q4" (see ``SignalEncoder.quantized``)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 weights: str = "mx") -> None:
        if weights not in FORMATS:
            raise ValueError("weights are held as 'mx' or 'q4'")
        quantize, self._product = FORMATS[weights]
        self.weight = quantize(weight.detach())
        self.bias = bias

    def __call__(self, rates: torch.Tensor) -> torch.Tensor:
        return self._product(rates, self.weight, bias=self.bias)


# ---- the example ---------------------------------------------------------------------

def _network(neurons: int, edges: int, batch: int, device, seed: int):
    def constant(value):
        return torch.full((neurons,), value, device=device)

    graph = random_topology(neurons, edges, device=device, seed=seed)
    model = DendriticDynamics.from_time_constants(
        Dynamics(constant(0.72), constant(0.8)), dt=1.0, tau_dendrite=4.0, tau_adaptation=25.0,
        coupling=0.5, adaptation_strength=0.2)
    return NativeDendriticMatrixRuntime(graph, model, torch.zeros(batch, neurons, device=device))


def fit(encoder: SignalEncoder, runtime, signal, target, steps: int, rate: float,
        drop: Dropout | None = None) -> list[float]:
    """Losses of ``steps`` updates of the encoder through recorded ticks: the mean squared
    distance of the rates after every tick from ``target`` [T, B, N]."""
    start = runtime.state, runtime.dendritic_state, runtime.adaptation_state
    optimizer = torch.optim.Adam(list(encoder.parameters.values()), lr=rate)
    losses = []
    for _ in range(steps):
        runtime.state, runtime.dendritic_state, runtime.adaptation_state = start
        drives, _ = encoder.drives(signal, drop=drop)
        rates = []
        for drive in drives.unbind(0):
            runtime.step(drive)
            rates.append(runtime.state)
        loss = (torch.stack(rates) - target).square().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        if drop is not None:
            drop.next()
        losses.append(float(loss.detach()))
    runtime.state, runtime.dendritic_state, runtime.adaptation_state = start
    return losses


def rollout_rates(runtime, drives: torch.Tensor) -> torch.Tensor:
    """Rates [T, B, N] of the network under staged drives (an even number of ticks)."""
    with torch.inference_mode():
        rollout = MatrixRollout(runtime, drives.shape[0], drive=drives.contiguous(), trace=True)
        rollout.run()
        return rollout.trace.clone()


def run(args: argparse.Namespace) -> dict:
    device, g = torch.device("cuda"), torch.Generator().manual_seed(args.seed)
    signal = torch.randn(args.ticks, args.batch, args.features, generator=g).cumsum(0).to(device)
    signal = signal / signal.abs().amax()
    runtime = _network(args.neurons, args.edges, args.batch, device, args.seed)
    # Rates to follow: a random projection of the signal, within the rates' range.
    mixing = torch.randn(args.neurons, args.features, generator=g).to(device)
    target = torch.sigmoid(2 * signal @ mixing.t() / args.features ** 0.5) * 0.6
    encoder = SignalEncoder(args.features, args.channels, args.neurons, mixer=args.mixer,
                            feed_forward=args.feed_forward, device=device, seed=args.seed)
    drop = Dropout(args.dropout, args.seed) if args.dropout else None
    losses = fit(encoder, runtime, signal, target, args.steps, args.rate, drop)
    served = encoder.quantized(args.weights)
    with torch.no_grad():
        exact = rollout_rates(runtime, encoder.drives(signal)[0])
        drives, _ = served.drives(signal)
        rates = rollout_rates(runtime, drives)
        carried = served.initial(args.batch)
        ticked = torch.stack([served.step(x, carried) for x in signal])
        read = ReadOut(torch.linalg.pinv(mixing), weights=args.weights)
        outputs = read(rates)
    return {"losses": [losses[0], losses[-1]],
            "rates_4bit_rms": float((rates - exact).square().mean().sqrt()),
            "ticks_against_signal": float((ticked - drives).abs().max()),
            "read_out": list(outputs.shape), "finite": bool(torch.isfinite(outputs).all())}


def parser() -> argparse.ArgumentParser:
    cli = argparse.ArgumentParser(description=__doc__,
                                  formatter_class=argparse.RawDescriptionHelpFormatter)
    for flag, default in (("neurons", 1024), ("edges", 16_384), ("batch", 4), ("ticks", 32),
                          ("features", 24), ("channels", 256), ("steps", 30), ("seed", 0)):
        cli.add_argument(f"--{flag}", type=int, default=default)
    cli.add_argument("--rate", type=float, default=3e-3, help="Adam's learning rate")
    cli.add_argument("--mixer", choices=MIXERS, default="scan")
    cli.add_argument("--feed-forward", type=int, default=0, help="width of the gated block (0: none)")
    cli.add_argument("--dropout", type=float, default=0.0, help="of what the gated block adds")
    cli.add_argument("--weights", choices=tuple(FORMATS), default="mx", help="4-bit form served")
    return cli


def main(argv=None) -> None:
    args = parser().parse_args(argv)
    if args.ticks % 2:
        raise SystemExit("--ticks must be even")
    if args.dropout and not args.feed_forward:
        raise SystemExit("--dropout needs --feed-forward")
    print(json.dumps(run(args)))


if __name__ == "__main__":
    main()
