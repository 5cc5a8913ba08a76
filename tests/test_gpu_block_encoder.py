"""The encoder with a gated recurrence, a gated block, dropout and 4-bit groups: the operators
together, fitted and served (MI355X)."""

from __future__ import annotations

import json

import pytest
import torch

import block_oracle as bo
import signal_oracle as so
from neurosim_gpu import signal_encoder
from neurosim_gpu.signal_encoder import Dropout, ReadOut, SignalEncoder

pytestmark = pytest.mark.gpu


def make(gpu, mixer="gated", seed=0, **more):
    return SignalEncoder(10, 48, 70, states=8, groups=2, mixer=mixer, feed_forward=60, device=gpu,
                         seed=seed, **more)


def signal(gpu, T, B, seed=1):
    return torch.randn(T, B, 10, generator=torch.Generator().manual_seed(seed)).to(gpu)


def test_drives_and_gradients_against_float64(gpu):
    """Drives and the gradients of every parameter, with a mask in force, against the same
    encoder in float64 (autograd over torch operations).  Float32 throughout: some hundred
    roundings of 6e-8 along a path, so 1e-4 of each tensor's largest value."""
    encoder, x, drop = make(gpu), signal(gpu, 12, 3), Dropout(0.3, seed=5)
    drop.next()
    drives, _ = encoder.drives(x, drop=drop)
    up = torch.randn(drives.shape, generator=torch.Generator().manual_seed(2)).to(gpu)
    got = torch.autograd.grad(drives, list(encoder.parameters.values()), up)
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in encoder.parameters.items()}
    values, gate = (so.wide(x) @ p["project_in"].t()).chunk(2, -1)
    line = torch.cat((torch.zeros(3, 3, 48, dtype=torch.float64), values))
    pre = p["conv_bias"] + sum(p["conv_weight"][:, k] * line[k:k + 12] for k in range(4))
    values = torch.nn.functional.silu(pre)
    forget, write = (values @ p["project_step"].t()).chunk(2, -1)
    fade = torch.exp(p["log_rates"]) * torch.sigmoid(forget)
    h, ys = torch.zeros(3, 48, dtype=torch.float64), []
    for t in range(12):
        h = (torch.exp(-fade[t]) * h
             + torch.sqrt(1 - torch.exp(-2 * fade[t])) * torch.sigmoid(write[t]) * values[t])
        ys.append(h * torch.nn.functional.silu(gate[t]))
    y = torch.stack(ys)
    inner = torch.nn.functional.silu(y @ p["block_gate"].t()) * (y @ p["block_up"].t())
    kept = bo.kept(y.numel(), 0.3, 5, 1).view(y.shape)
    y = y + torch.where(kept, inner @ p["project_down"].t(), 0.0) * (65536 / (65536 - round(0.3 * 65536)))
    want = y @ p["project_out"].t()
    assert (drives.detach().double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()
    grads = torch.autograd.grad(want, list(p.values()), up.double().cpu())
    for name, a, b in zip(p, got, grads):
        assert (a.double().cpu() - b).abs().max() <= 1e-4 * b.abs().max(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mixer", ["scan", "gated"])
def test_served_ticks_are_the_served_signal(gpu, mixer, dtype):
    """One tick at a time, in parts and as a whole, with integer weights.  Nothing but the last
    bits differ, since rows stay floats: some hundred roundings of the type's half unit."""
    encoder = make(gpu, mixer).quantized("q4", block=dtype)
    x = signal(gpu, 20, 4).to(dtype)
    with torch.no_grad():
        whole, (history, state) = encoder.drives(x)
        first, carried = encoder.drives(x[:7])
        second, _ = encoder.drives(x[7:], carried)
        carried = encoder.initial(4, dtype)
        ticks = torch.stack([encoder.step(v, carried) for v in x])
    assert whole.dtype == dtype
    bound = (1e-5 if dtype == torch.float32 else 0.05) * float(whole.float().abs().max())
    for other in (ticks, torch.cat((first, second))):
        assert (other.float() - whole.float()).abs().max() <= bound
    assert (carried[0] - history).abs().max() <= 2.0 ** -7 * history.abs().max()
    assert (carried[1] - state).abs().max() <= bound / float(whole.float().abs().max()) * state.abs().max()


def test_integer_weights_are_the_weights_values(gpu):
    """The encoder served in 4-bit groups is the float encoder with the weights read back."""
    encoder, x = make(gpu), signal(gpu, 9, 2)
    served = encoder.quantized("q4")
    with torch.no_grad():
        for name, value in served.parameters.items():
            encoder.parameters[name].copy_(value if isinstance(value, torch.Tensor) else value.dequantize())
        want, _ = encoder.drives(x)
        got, _ = served.drives(x)
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()


def test_columns_of_their_own_length(gpu):
    encoder, x = make(gpu).quantized("q4"), signal(gpu, 9, 3)
    with torch.no_grad():
        short, carried = encoder.drives(x, lengths=torch.tensor([9, 4, 0], device=gpu))
        alone, _ = encoder.drives(x[:4, 1:2])
    assert not short[4:, 1].any() and not short[:, 2].any() and not carried[1][2].any()
    assert (short[:4, 1:2] - alone).abs().max() <= 1e-5 * alone.abs().max()


def test_dropout_moves_on(gpu):
    encoder, x, drop = make(gpu), signal(gpu, 5, 2), Dropout(0.5)
    with torch.no_grad():
        first = encoder.drives(x, drop=drop)[0]
        assert torch.equal(first, encoder.drives(x, drop=drop)[0])
        drop.next()
        assert not torch.equal(first, encoder.drives(x, drop=drop)[0])
        none = encoder.drives(x, drop=Dropout(0.0))[0]
        assert (none - encoder.drives(x)[0]).abs().max() <= 1e-5 * none.abs().max()


def test_read_out(gpu):
    weight = torch.randn(5, 200, generator=torch.Generator().manual_seed(4)).to(gpu)
    rates = torch.rand(6, 3, 200, generator=torch.Generator().manual_seed(5)).to(gpu)
    read = ReadOut(weight, weights="q4")
    want = rates.double() @ read.weight.dequantize().double().t()
    assert (read(rates).double() - want).abs().max() <= 1e-5 * want.abs().max()


@pytest.mark.parametrize("mixer", ["scan", "gated"])
def test_example_runs(gpu, mixer, capsys):
    signal_encoder.main(["--neurons", "256", "--edges", "4096", "--channels", "64", "--ticks", "16",
                         "--steps", "4", "--batch", "2", "--mixer", mixer, "--feed-forward", "96",
                         "--dropout", "0.1", "--weights", "q4"])
    report = json.loads(capsys.readouterr().out)
    assert report["finite"] and report["read_out"] == [16, 2, 24]
    assert all(v == v for v in report["losses"]) and report["ticks_against_signal"] < 1e-4


def test_refusals(gpu):
    for more, message in (({"mixer": "mean"}, "mixer is"), ({"feed_forward": -1}, "not negative")):
        with pytest.raises(ValueError, match=message):
            SignalEncoder(4, 10, 8, device=gpu, **more)
    plain = SignalEncoder(10, 16, 8, device=gpu)
    with pytest.raises(ValueError, match="'mx' or 'q4'"):
        plain.quantized("int8")
    with pytest.raises(ValueError, match="'mx' or 'q4'"):
        ReadOut(torch.ones(2, 2, device=gpu), weights="int8")
    with pytest.raises(ValueError, match="which this encoder lacks"):
        plain.drives(signal(gpu, 2, 1), drop=Dropout(0.1))
    with pytest.raises(SystemExit, match="needs --feed-forward"):
        signal_encoder.main(["--dropout", "0.1"])
