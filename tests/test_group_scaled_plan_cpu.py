"""Every kernel that a 4-bit product's plan can choose is reached by a shape of the GPU tests.

``plan`` restates the rule of csrc/q4_product.hip; that it is the library's is seen from the size of
the workspace, which tells how many parts K is cut into, for every shape here and some thousand others."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

import test_gpu_group_scaled as values
import test_gpu_group_scaled_tiles as tiles
from neurosim_gpu import native

FLOAT, HALF = 0, 1


def ceil(a, b):
    return -(-a // b)


def plan(m, n, k, kind):
    """(kernel, tiles of rows, strips; wavefronts a strip, parts of K, chunks a part)."""
    if kind != FLOAT and m <= 16:
        stages = ceil(k, 128)
        strips = 1 if n <= 4096 else 2 if m <= 8 or n < 12_288 else 4
        parts = 1
        while parts < 8 and stages >= 8 * parts:
            parts *= 2
        groups, splits = ceil(ceil(n, 16 * strips) * parts, 8), 1
        if groups < 128:
            splits = max(1, min(512 // groups, stages // (4 * parts)))
        per = ceil(stages, splits)
        return ("rows", 1, strips), parts, ceil(stages, per), per
    count = ceil(m, 4 if kind == FLOAT else 16)
    own = count if count <= 2 else 3 if count == 3 and kind != FLOAT else 4
    m_tiles, chunks = ceil(count, own), ceil(k, 1024 if own == 1 else 512)
    few = kind != FLOAT and m_tiles * ceil(n, 16) * chunks <= 2048
    strips = 1 if own == 1 or few else 2
    lines, parts = ceil(n, 16 * strips), 1
    while parts * 2 <= 4 // own and m_tiles * lines * parts < 2048:
        parts *= 2
    waves = m_tiles * lines * parts
    per = ceil(chunks, min(2048 // waves if waves < 2048 else 1, chunks))
    return ("tiles", own, strips), parts, ceil(chunks, per), per


def products_run():
    """(kind, shape, group) of the GPU tests of products."""
    for shape in values.SHAPES:
        for group in (32, 64, 128, 256):
            yield FLOAT, shape, group
            yield HALF, shape, group
    for dtype, shape in tiles.CASES:
        for group in tiles.GROUPS:
            yield FLOAT if dtype == torch.float32 else HALF, shape, group


def test_every_kernel_is_reached():
    seen, more = set(), {}
    for kind, (m, n, k), group in products_run():
        kernel, parts, splits, per = plan(m, n, k, kind)
        seen.add((kind, *kernel, min(group, 128)))
        facts = more.setdefault((kind, *kernel), set())
        facts |= {f"{splits > 24} past 24 parts", f"{splits > 1} split", f"{parts > 1} shared strip"}
        facts.add(f"{kernel[0] == 'tiles' and per > 1} several chunks")
        facts.add(f"{m > kernel[1] * (4 if kind == FLOAT else 16)} tiles of rows")
    kernels = {(HALF, "rows", 1, s) for s in (1, 2, 4)}
    kernels |= {(HALF, "tiles", t, s) for t in (2, 3, 4) for s in (1, 2)}
    kernels |= {(FLOAT, "tiles", 1, 1), (FLOAT, "tiles", 2, 2), (FLOAT, "tiles", 4, 2)}
    assert seen == {(*kernel, group) for kernel in kernels for group in (32, 64, 128)}
    # Both ends of what a kernel does, where it can be at both.
    for kernel in ((FLOAT, "tiles", 1, 1), (FLOAT, "tiles", 2, 2), (FLOAT, "tiles", 4, 2), (HALF, "tiles", 2, 2),
                   (HALF, "tiles", 3, 2), (HALF, "tiles", 4, 2)):
        assert "True several chunks" in more[kernel], kernel
    for fact in ("True past 24 parts", "True shared strip"):
        for kind in (FLOAT, HALF):
            assert any(fact in facts for kernel, facts in more.items() if kernel[0] == kind), fact
    for kernel in ((FLOAT, "tiles", 4, 2), (HALF, "tiles", 4, 1), (HALF, "tiles", 4, 2)):
        assert "True tiles of rows" in more[kernel], kernel


def test_the_rule_is_the_library_s():
    fn = native.load_library().ns_q4_product_floats
    fn.restype, fn.argtypes = ctypes.c_int64, [ctypes.c_int64] * 3 + [ctypes.c_int32]
    rng = random.Random(5)
    shapes = [(kind, shape) for kind, shape, _ in products_run()]
    for _ in range(4000):
        size = [int(2 ** rng.uniform(0, top)) for top in (11, 16, 16)]
        shapes.append((rng.choice((FLOAT, HALF, 2)), tuple(size)))
    for kind, (m, n, k) in shapes:
        splits = plan(m, n, k, kind)[2]
        assert fn(m, n, k, kind) == (splits * m * n if splits > 1 else 0), (kind, m, n, k)


@pytest.mark.parametrize("around_one", [False, True])
def test_exact_rows_are_exact(around_one):
    """The premise of the GPU test: a float32 row's parts, and their sums, as it says."""
    g = torch.Generator().manual_seed(1)
    x = tiles.exact_rows(g, 3, 128, torch.float32, around_one).double()
    mean = x.mean(-1, keepdim=True)
    assert torch.equal(mean, torch.full_like(mean, float(around_one)))
    rest, grids = x - mean, (2.0 ** -9, 2.0 ** -16, 0) if around_one else (2.0 ** -7, 2.0 ** -16, 2.0 ** -23)
    for grid in grids:
        part = rest.bfloat16().double()
        rest = rest - part
        if grid:
            assert torch.equal((part / grid).round() * grid, part)
            assert float(part.abs().sum()) * 31 < 2.0 ** 24 * grid
        else:
            assert not part.any()
    assert not rest.any()
