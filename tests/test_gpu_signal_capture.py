"""The backward of the signal operators under graph capture (MI355X)."""

from __future__ import annotations

import pytest
import torch

from neurosim_gpu import causal_conv, selective_scan

pytestmark = pytest.mark.gpu


def outputs(gpu):
    x = torch.ones(3, 2, 4, device=gpu, requires_grad=True)
    narrow = torch.ones(3, 2, 5, device=gpu)
    return {"causal_conv": causal_conv(x, torch.ones(4, 3, device=gpu)),
            "selective_scan": selective_scan(x, x, -torch.ones(4, 5, device=gpu), narrow, narrow)}


@pytest.mark.parametrize("which", [0, 1])      # y, and the carried history or state
@pytest.mark.parametrize("name", ["causal_conv", "selective_scan"])
def test_no_backward_under_capture(gpu, monkeypatch, name, which):
    """Refused from the query alone: no stream is captured here."""
    out = outputs(gpu)[name][which]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match=f"the backward of {name} cannot be captured"):
        out.sum().backward()


@pytest.mark.parametrize("name", ["causal_conv", "selective_scan"])
def test_a_backward_beside_it_runs(gpu, name):
    y, carried = outputs(gpu)[name]
    (y.sum() + carried.sum()).backward()
