"""What the signal operators' size queries say; they touch no device."""

from __future__ import annotations

import ctypes

import pytest

from neurosim_gpu import native, signal_ops


@pytest.fixture(scope="module")
def lib():
    return native.load_library()


SHAPES = [  # T, B, N, G, S
    (16_384, 1, 2048, 1, 16), (777, 5, 1500, 3, 8), (2048, 8, 4096, 1, 16), (260, 2, 5, 1, 4),
    (1, 1, 1, 1, 1), (300, 1, 70, 2, 33), (0, 2, 8, 1, 4),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_scan_plan(shape):
    """Both directions cut time alike; states are padded to four times a power of two per
    channel and kept before every tile; partial sums belong to the backward alone."""
    T, B, N, G, S = shape
    forward = list(signal_ops._plan((T, B, N), G, S, False))
    backward = list(signal_ops._plan((T, B, N), G, S, True))
    assert forward[:3] == backward[:3]
    chunks, ends, checkpoints, partials = backward
    padded = next(p for p in (4, 8, 16, 32, 64) if S <= p)
    tile = 16 if padded <= 16 else 256 // padded
    tiles = -(-T // tile)
    assert 1 <= chunks <= max(1, tiles // 2)
    assert ends == (chunks * B * N * (padded + 1) if chunks > 1 else 0)
    assert checkpoints == tiles * B * N * padded
    blocks = -(-(N // G) // 64)
    assert partials == chunks * B * N * (S + 2) + blocks * T * B * G * 2 * padded
    assert forward[3] == 0


def test_scan_plan_refuses(lib):
    fn, sizes = signal_ops._library().ns_scan_plan, (ctypes.c_int64 * 4)()
    for shape, text in (((4, -1, 8, 1, 4), "[T, B, N]"), ((4, 1, 8, 3, 4), "divide"),
                        ((4, 1, 8, 1, 65), "1 to 64 states"), ((2 ** 31, 1, 8, 1, 4), "2^31 ticks")):
        assert fn(*shape, 0, ctypes.addressof(sizes)) == 1
        assert text.encode() in lib.ns_last_error()
    assert fn(4, 1, 8, 1, 4, 0, None) == 1
