"""Signals into per-tick drives, and rates into read-outs.

``SignalEncoder`` turns a signal [T, B, F] into the somatic drives [T, B, N] of a network:

    projection F -> 2C (values and gates), a short causal convolution per channel, a
    projection to each channel's time step and the shared B and C, a selective scan, and
    a projection C -> N.

It runs in two forms.  With its float32 parameters every step has gradients, so it is
fitted through recorded ticks of a ``NativeDendriticMatrixRuntime``; ``quantized()`` gives
the serving form, whose three projections hold their weights in microscaled 4 bits, with
whole signals (``drives``, staged into a ``MatrixRollout``) and single ticks in closed loop
(``step``).  ``ReadOut`` is a 4-bit projection of rates.

    python -m neurosim_gpu.signal_encoder [--neurons 1024 ...]

fits an encoder so that a network's rates follow a target, quantises it, rolls the network
out under both forms' drives and prints what the 4 bits change, as JSON.
"""

from __future__ import annotations

import argparse
import json
import math

import torch

from .compartmental import DendriticDynamics
from .dynamics import Dynamics
from .microscaled import MXTensor, mx_product, mx_quantize
from .native_compartmental import NativeDendriticMatrixRuntime
from .rollout import MatrixRollout
from .signal_ops import causal_conv, causal_conv_step, selective_scan, selective_scan_step
from .topology import random_topology

_PROJECTIONS = ("project_in", "project_step", "project_out")


class _Encoder:
    """What the float and the 4-bit form share; ``_project`` is theirs."""

    def __init__(self, parameters: dict, channels: int, states: int, groups: int) -> None:
        self.parameters = parameters
        self.channels, self.states, self.groups = channels, states, groups

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
        return (torch.zeros(self.taps - 1, batch, self.channels, dtype=dtype, device=self.device),
                torch.zeros(batch, self.channels, self.states, device=self.device))

    def _scan_inputs(self, x: torch.Tensor):
        """(delta, B, C) of filtered values [..., C]: slices of one projection, not copied."""
        both = self._project("project_step", x)
        lead, wide = x.shape[:-1], self.groups * self.states
        delta, write, read = both.split((self.channels, wide, wide), -1)
        shape = (*lead, self.groups, self.states)
        return delta, write.unflatten(-1, shape[-2:]), read.unflatten(-1, shape[-2:])

    def drives(self, signal: torch.Tensor, carried=None, lengths: torch.Tensor | None = None):
        """Drives [T, B, N] of a signal [T, B, F], and the carried (history, state) after it."""
        p = self.parameters
        history, state = (self.initial(signal.shape[1], signal.dtype) if carried is None
                          else carried)
        x, gate = self._project("project_in", signal).chunk(2, -1)
        x, history = causal_conv(x, p["conv_weight"], p["conv_bias"], history=history,
                                 lengths=lengths)
        delta, write, read = self._scan_inputs(x)
        y, state = selective_scan(x, delta, -torch.exp(p["log_rates"]), write, read, p["skip"],
                                  z=gate, delta_bias=p["step_bias"], state=state, lengths=lengths)
        return self._project("project_out", y), (history, state)


class SignalEncoder(_Encoder):
    """Float32 encoder with gradients (see the module); parameters are drawn from ``seed``."""

    def __init__(self, features: int, channels: int, neurons: int, *, states: int = 16,
                 groups: int = 1, taps: int = 4, device="cuda", seed: int = 0) -> None:
        if min(features, channels, neurons, states, groups, taps) <= 0 or channels % groups:
            raise ValueError("sizes must be positive and the groups divide the channels")
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
        super().__init__({k: v.to(device).requires_grad_() for k, v in values.items()},
                         channels, states, groups)

    def _project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return x @ self.parameters[name].t()

    def quantized(self) -> "QuantizedEncoder":
        """The serving form of the present parameters, its projections in 4 bits."""
        values = {k: mx_quantize(v.detach()) if k in _PROJECTIONS else v.detach().clone()
                  for k, v in self.parameters.items()}
        return QuantizedEncoder(values, self.channels, self.states, self.groups)


class QuantizedEncoder(_Encoder):
    """Encoder with microscaled 4-bit projections, for serving."""

    def __init__(self, parameters: dict, channels: int, states: int, groups: int) -> None:
        super().__init__(parameters, channels, states, groups)
        self._rates = -torch.exp(parameters["log_rates"])

    def _project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return mx_product(x, self.parameters[name])

    def step(self, signal: torch.Tensor, carried) -> torch.Tensor:
        """Drives [B, N] of one tick [B, F]; ``carried`` (``initial``) moves on in place."""
        p, (history, state) = self.parameters, carried
        x, gate = self._project("project_in", signal).chunk(2, -1)
        x = causal_conv_step(x, p["conv_weight"], p["conv_bias"], history=history)
        delta, write, read = self._scan_inputs(x)
        y = selective_scan_step(x, delta, self._rates, write, read, p["skip"], z=gate,
                                delta_bias=p["step_bias"], state=state)
        return self._project("project_out", y)


class ReadOut:
    """Outputs [..., K] of rates [..., N]: a projection ``weight`` [K, N] held in 4 bits."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None) -> None:
        self.weight: MXTensor = mx_quantize(weight.detach())
        self.bias = bias

    def __call__(self, rates: torch.Tensor) -> torch.Tensor:
        return mx_product(rates, self.weight, bias=self.bias)


# ---- the example ---------------------------------------------------------------------

def _network(neurons: int, edges: int, batch: int, device, seed: int):
    def constant(value):
        return torch.full((neurons,), value, device=device)

    graph = random_topology(neurons, edges, device=device, seed=seed)
    model = DendriticDynamics.from_time_constants(
        Dynamics(constant(0.72), constant(0.8)), dt=1.0, tau_dendrite=4.0, tau_adaptation=25.0,
        coupling=0.5, adaptation_strength=0.2)
    return NativeDendriticMatrixRuntime(graph, model, torch.zeros(batch, neurons, device=device))


def fit(encoder: SignalEncoder, runtime, signal, target, steps: int, rate: float) -> list[float]:
    """Losses of ``steps`` updates of the encoder through recorded ticks: the mean squared
    distance of the rates after every tick from ``target`` [T, B, N]."""
    start = runtime.state, runtime.dendritic_state, runtime.adaptation_state
    optimizer = torch.optim.Adam(list(encoder.parameters.values()), lr=rate)
    losses = []
    for _ in range(steps):
        runtime.state, runtime.dendritic_state, runtime.adaptation_state = start
        drives, _ = encoder.drives(signal)
        rates = []
        for drive in drives.unbind(0):
            runtime.step(drive)
            rates.append(runtime.state)
        loss = (torch.stack(rates) - target).square().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
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
    encoder = SignalEncoder(args.features, args.channels, args.neurons, device=device, seed=args.seed)
    losses = fit(encoder, runtime, signal, target, args.steps, args.rate)
    served = encoder.quantized()
    with torch.no_grad():
        exact = rollout_rates(runtime, encoder.drives(signal)[0])
        drives, _ = served.drives(signal)
        rates = rollout_rates(runtime, drives)
        carried = served.initial(args.batch)
        ticked = torch.stack([served.step(x, carried) for x in signal])
        read = ReadOut(torch.linalg.pinv(mixing))
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
    return cli


def main(argv=None) -> None:
    args = parser().parse_args(argv)
    if args.ticks % 2:
        raise SystemExit("--ticks must be even")
    print(json.dumps(run(args)))


if __name__ == "__main__":
    main()
