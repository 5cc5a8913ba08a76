"""The oracle of the gated block's operators: its gradients against differences of its outputs."""

from __future__ import annotations

import torch

import block_oracle as bo


def draw(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def against_differences(form, operands: dict, ups: dict, tolerance=1e-6):
    """form(operands) -> outputs; the gradients of sum(outputs * ups), by central differences."""
    def total(values):
        out = form(values)
        return sum(float((out[k] * up).sum()) for k, up in ups.items())

    step, found = 1e-5, {}
    for name, value in operands.items():
        grad = torch.zeros_like(value)
        for k in range(value.numel()):
            ends = []
            for sign in (1, -1):
                moved = value.clone()
                moved.view(-1)[k] += sign * step
                ends.append(total({**operands, name: moved}))
            grad.view(-1)[k] = (ends[0] - ends[1]) / (2 * step)
        found[name] = grad
    return found


def test_recurrence_gradients():
    g = torch.Generator().manual_seed(1)
    T, B, N = 5, 3, 2
    operands = {"x": draw(g, T, B, N), "forget": draw(g, T, B, N), "write": draw(g, T, B, N),
                "z": draw(g, T, B, N), "rates": draw(g, N).abs() + 0.1, "state": draw(g, B, N)}
    ups = {"y": draw(g, T, B, N), "state": draw(g, B, N)}
    lengths = torch.tensor([5, 0, 2])
    found = against_differences(lambda v: bo.recurrence(**v, lengths=lengths)[0], operands, ups)
    _, grads = bo.recurrence(**operands, lengths=lengths, dy=ups["y"], dfinal=ups["state"])
    for name, value in found.items():
        assert (grads[name] - value).abs().max() < 1e-7, name
    sizes = bo.recurrence(**operands, lengths=lengths, dy=ups["y"], dfinal=ups["state"],
                          magnitude=True)[1]
    for name in found:
        assert (grads[name].abs() <= sizes[name] + 1e-12).all(), name


def test_gated_gradients():
    g = torch.Generator().manual_seed(2)
    for activation in ("silu", "gelu"):
        operands = {"x": draw(g, 4, 3), "gate": draw(g, 5, 3), "up": draw(g, 5, 3)}
        dy = draw(g, 4, 5)
        found = against_differences(lambda v: {"y": bo.gated(**v, activation=activation)[0]},
                                    operands, {"y": dy})
        _, grads = bo.gated(**operands, activation=activation, dy=dy)
        for name, value in found.items():
            assert (grads[name] - value).abs().max() < 1e-7, name


def test_philox_known_answers():
    """Known answers that the generator's authors publish for Philox4x32 with 10 rounds."""
    def words(counter, offset, seed):
        n = bo.philox(counter, offset, seed)
        return [n[2 * k] | n[2 * k + 1] << 16 for k in range(4)]

    assert words(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert words(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
