"""The encoder example: its operators together, fitted and served (MI355X)."""

from __future__ import annotations

import pytest
import torch

import signal_oracle as so
from neurosim_gpu import mx_quantize, signal_encoder
from neurosim_gpu.signal_encoder import ReadOut, SignalEncoder

pytestmark = pytest.mark.gpu


def make(gpu, seed=0, **more):
    return SignalEncoder(10, 48, 70, states=8, groups=2, device=gpu, seed=seed, **more)


def signal(gpu, T, B, seed=1):
    return torch.randn(T, B, 10, generator=torch.Generator().manual_seed(seed)).to(gpu)


def test_drives_and_gradients_against_float64(gpu):
    """Drives and the gradients of every parameter, against the same encoder in float64
    through the oracle's equations (autograd over torch operations).  Float32 throughout:
    some hundred roundings of 6e-8 along a path, so 1e-4 of each tensor's largest value."""
    encoder, x = make(gpu), signal(gpu, 12, 3)
    drives, _ = encoder.drives(x)
    up = torch.randn(drives.shape, generator=torch.Generator().manual_seed(2)).to(gpu)
    got = torch.autograd.grad(drives, list(encoder.parameters.values()), up)
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in encoder.parameters.items()}
    values, gate = (so.wide(x) @ p["project_in"].t()).chunk(2, -1)
    line = torch.cat((torch.zeros(3, 3, 48, dtype=torch.float64), values))
    pre = p["conv_bias"] + sum(p["conv_weight"][:, k] * line[k:k + 12] for k in range(4))
    values = torch.nn.functional.silu(pre)
    delta, write, read = (values @ p["project_step"].t()).split((48, 16, 16), -1)
    write, read = (v.unflatten(-1, (2, 8)).repeat_interleave(24, -2) for v in (write, read))
    dt = torch.nn.functional.softplus(delta + p["step_bias"])
    h, ys = torch.zeros(3, 48, 8, dtype=torch.float64), []
    for t in range(12):
        h = (torch.exp(-dt[t][..., None] * torch.exp(p["log_rates"])) * h
             + (dt[t] * values[t])[..., None] * write[t])
        ys.append(((read[t] * h).sum(-1) + p["skip"] * values[t])
                  * torch.nn.functional.silu(gate[t]))
    want = torch.stack(ys) @ p["project_out"].t()
    assert (drives.detach().double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()
    grads = torch.autograd.grad(want, list(p.values()), up.double().cpu())
    for name, a, b in zip(p, got, grads):
        assert (a.double().cpu() - b).abs().max() <= 1e-4 * b.abs().max(), name


def test_served_ticks_are_the_served_signal(gpu):
    """One tick at a time against the whole signal, both in 4 bits.  The forms differ in the
    last bits of the scan's float32 outputs; where that moves a value across a rounding
    boundary of the last projection's 4 bits it changes by one step, at most 1/3 of a value of
    the block's upper half, here one of 48 that a drive sums: rarely, so most drives agree to
    float32 rounding and all to a quarter of the largest."""
    encoder = make(gpu).quantized()
    x = signal(gpu, 20, 4)
    with torch.no_grad():
        whole, (history, state) = encoder.drives(x)
        carried = encoder.initial(4)
        ticks = torch.stack([encoder.step(v, carried) for v in x])
    scale = float(whole.abs().max())
    apart = (ticks - whole).abs()
    assert float((apart <= 1e-5 * scale).float().mean()) >= 0.9
    assert float(apart.max()) <= 0.25 * scale
    assert (carried[0] - history).abs().max() <= 1e-5 * history.abs().max()
    assert (carried[1] - state).abs().max() <= 1e-4 * state.abs().max()


def test_columns_of_their_own_length(gpu):
    encoder, x = make(gpu).quantized(), signal(gpu, 9, 3)
    with torch.no_grad():
        short, carried = encoder.drives(x, lengths=torch.tensor([9, 4, 0], device=gpu))
        alone, _ = encoder.drives(x[:4, 1:2])
    # Past a column's end the scan gives zeros, whose projection is zero.
    assert torch.equal(short[4:, 1], torch.zeros_like(short[4:, 1]))
    assert torch.equal(short[:, 2], torch.zeros_like(short[:, 2]))
    assert (short[:4, 1:2] - alone).abs().max() <= 0.25 * alone.abs().max()
    assert torch.equal(carried[1][2], torch.zeros_like(carried[1][2]))


def test_read_out(gpu):
    weight = torch.randn(5, 200, generator=torch.Generator().manual_seed(4)).to(gpu)
    rates = torch.rand(6, 3, 200, generator=torch.Generator().manual_seed(5)).to(gpu)
    got = ReadOut(weight)(rates)
    want = mx_quantize(rates).dequantize().double() @ mx_quantize(weight).dequantize().double().t()
    assert got.shape == (6, 3, 5)
    assert (got.double() - want).abs().max() <= 200 * 2.0 ** -23 * 200


def test_example_fits_and_serves(gpu):
    """The module's example, small: the loss falls, and 4 bits move the rates little."""
    args = signal_encoder.parser().parse_args(
        ["--neurons", "256", "--edges", "4096", "--channels", "64", "--ticks", "16", "--steps",
         "25", "--batch", "2"])
    report = signal_encoder.run(args)
    assert report["losses"][1] < 0.7 * report["losses"][0]
    assert report["finite"] and report["read_out"] == [16, 2, 24]
    assert report["rates_4bit_rms"] < 0.1


def test_refusals(gpu):
    with pytest.raises(ValueError, match="groups divide"):
        SignalEncoder(4, 10, 8, groups=3, device=gpu)
    with pytest.raises(ValueError, match="positive"):
        SignalEncoder(0, 10, 8, device=gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_signals_of_fewer_bits_are_served(gpu, dtype):
    """The carried history has the signal's type, also where the encoder makes it.  The bounds
    are those of float32 signals, with the type's rounding in place of float32's."""
    encoder = make(gpu).quantized()
    x = signal(gpu, 20, 4).to(dtype)
    with torch.no_grad():
        whole, (history, state) = encoder.drives(x)
        first, carried = encoder.drives(x[:7])
        second, _ = encoder.drives(x[7:], carried)
        carried = encoder.initial(4, dtype)
        ticks = torch.stack([encoder.step(v, carried) for v in x])
    assert whole.dtype == history.dtype == dtype and state.dtype == torch.float32
    assert (carried[0] - history).abs().max() <= 2.0 ** -7 * history.abs().max()   # one rounding
    scale = float(whole.float().abs().max())
    for other in (torch.cat((first, second)), ticks):
        apart = (other.float() - whole.float()).abs()
        assert float((apart <= 0.02 * scale).float().mean()) >= 0.9
        assert float(apart.max()) <= 0.25 * scale
