"""Gated projection and dropout against float64 formulas (MI355X).

Tolerances of the projection (block_oracle.gated_bounds).  With u = 2^-24, a sum of K products
in float32 is off by at most 2 (K + 2) u times the sum of their sizes (2 u an addition, since the
matrix cores may cut off instead of rounding), six times that in float32, whose products are
summed in six parts (and the three left out are at most 2 u of a product).  The activation carries its argument's error
times its slope, and its own operations.  The gradients' operands dg and du are rounded to
the operands' type, half a unit each, which passes through their products like the errors
before.  Outputs are then rounded once to their type.
"""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from test_gpu_signal import HALF_ULP, SMALLEST, U, Draw, leaves
from neurosim_gpu import dropout, gated_projection, gated_recurrence

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def within(got, want, bound, what: str):
    assert got.shape == want.shape, what
    # A rounding below the type's normal numbers is off by half the smallest one's unit.
    bound = bound + HALF_ULP[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    assert torch.isfinite(got).all(), what
    worst = float(((got.detach().double().cpu() - want).abs() / bound).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} of its bound"


def check_gated(values: dict, activation: str, dy):
    inputs = leaves(values)
    y = gated_projection(**inputs, activation=activation)
    alone = gated_projection(**values, activation=activation)
    assert torch.equal(y.detach(), alone)          # keeping the products changes nothing
    half = 0.0 if y.dtype == torch.float32 else HALF_ULP[y.dtype]
    want, grads = bo.gated(**values, activation=activation, dy=dy)
    bounds = bo.gated_bounds(**values, activation=activation, dy=dy, u=U, half=half)
    within(y, want, bounds["y"], "y")
    got = torch.autograd.grad(y, list(inputs.values()), dy)
    for name, value in zip(inputs, got):
        assert value.dtype == y.dtype
        # Below the type's normal numbers the operands' rounding is off by a fixed amount.
        low = SMALLEST[y.dtype] * (dy.shape[0] + 2 * dy.shape[1]) * float(
            max(v.abs().max() for v in values.values()))
        within(value, grads[name], bounds[name] + low, f"d{name}")


def operands(draw, M, K, F, dtype):
    return {"x": draw(M, K, dtype=dtype), "gate": draw(F, K, scale=K ** -0.5, dtype=dtype),
            "up": draw(F, K, scale=K ** -0.5, dtype=dtype)}


SHAPES = [  # M, K, F: few rows, small, middle and large tiles, odd ends each way
    (1, 1, 1), (1, 64, 16), (3, 200, 33), (16, 1031, 70), (5, 4100, 9), (17, 32, 32),
    (20, 7, 130), (64, 64, 32), (65, 96, 40), (130, 257, 100), (200, 1000, 77), (33, 4096, 24),
    (1030, 72, 1700),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_projection(gpu, shape, dtype):
    draw = Draw(gpu, sum(shape))
    M, K, F = shape
    check_gated(operands(draw, M, K, F, dtype), "silu" if K % 2 else "gelu", draw(M, F, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2100, 72, 2800), (40, 2100, 2820), (4120, 2900, 20)])
def test_large_tiles(gpu, shape, dtype):
    """The largest tiles: of the forward, of the weights' gradients, of x's."""
    draw = Draw(gpu, 3)
    M, K, F = shape
    check_gated(operands(draw, M, K, F, dtype), "silu", draw(M, F, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kept_products_leave_the_result_alone(gpu, dtype):
    """Many large tiles with long sums, whose wavefronts end at their own pace: the result with
    the two products kept beside it is the one without, again and again."""
    draw = Draw(gpu, 8)
    values = operands(draw, 4100, 1024, 4000, dtype)
    want = gated_projection(**values)
    inputs = leaves(values)
    for _ in range(5):
        y = gated_projection(**inputs)
        assert torch.equal(y.detach(), want)
        pre = y.grad_fn.saved_tensors[3]
        assert torch.equal((torch.nn.functional.silu(pre[0].double()) * pre[1].double()).isfinite(),
                           torch.ones_like(y, dtype=torch.bool))
        assert (pre[1] - values["x"].float() @ values["up"].float().t()).abs().max() < 1e-3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,F", [(7, 130, 44), (150, 130, 44), (1500, 2500, 410)])
def test_gated_strides(gpu, rows, K, F, dtype):
    """Rows at any stride and alignment, a shared row, more dimensions, dense or not: the same
    bits as dense copies."""
    draw = Draw(gpu, rows)
    dense = operands(draw, rows, K, F, dtype)
    dy = draw(rows, F, dtype=dtype)

    def passes(values, up):
        inputs = {k: v.detach().requires_grad_() for k, v in values.items()}
        y = gated_projection(**inputs)
        return (y, *torch.autograd.grad(y, list(inputs.values()), up))

    def spread(v, before, behind):
        room = torch.full((v.shape[0], before + v.shape[1] + behind), float("nan"), dtype=v.dtype,
                          device=v.device)
        out = room[:, before:before + v.shape[1]]
        return out.copy_(v)

    want = passes(dense, dy)
    for change in ({"x": spread(dense["x"], 1, 2)}, {"gate": spread(dense["gate"], 3, 0)},
                   {"x": spread(dense["x"], 8, 6), "up": spread(dense["up"], 8, 8)},
                   {"x": dense["x"].t().contiguous().t()}, {"up": dense["up"].t().contiguous().t()}):
        for a, b in zip(passes({**dense, **change}, dy), want):
            assert torch.equal(a, b), list(change)
    for up in (spread(dy, 1, 1), dy.t().contiguous().t()):
        for a, b in zip(passes(dense, up), want):
            assert torch.equal(a, b)
    shared = {**dense, "x": dense["x"][:1].expand(rows, K)}
    plain = {**dense, "x": shared["x"].contiguous()}
    assert torch.equal(gated_projection(**shared), gated_projection(**plain))
    cubes = {**dense, "x": dense["x"].view(1, rows, K)}
    assert torch.equal(gated_projection(**cubes), want[0].detach().view(1, rows, F))


def test_many_float32_rows(gpu):
    """A float32 forward in thirds, odd sizes each way."""
    draw = Draw(gpu, 6)
    M, K, F = 1290, 2301, 525
    check_gated(operands(draw, M, K, F, torch.float32), "gelu", draw(M, F))


@pytest.mark.parametrize("rows,width", [(5, 2), (200, 2), (4100, 400)])
def test_float32_is_multiplied_as_float32(gpu, rows, width):
    """Values whose parts matter: all 24 bits set, far apart in size, as large and as small as
    float32 has them.  Against float64, a product is off by its own rounding and the three parts
    left out, a sum of two by one rounding more: 2^-22 of the sizes is more than both.  What
    float32 has no number for, 3.4e38 times more than one, is an infinity of its sign."""
    g = torch.Generator().manual_seed(3)
    pad = torch.nn.functional.pad if width > 300 else (lambda v, _: v)
    x = torch.randn(rows, 2, generator=g)
    x[0] = torch.tensor([1 + 2.0 ** -23, 0.0])
    x[1] = torch.tensor([2.0 - 2.0 ** -23, 0.0])
    x[2] = torch.tensor([3.4e38, 0.0])           # rounds past the largest bfloat16
    x[3] = torch.tensor([1e-30, 1e10])
    up = torch.tensor([[1 + 2.0 ** -22, 2.0 ** -12 + 2.0 ** -30], [0.75, -1.0]])
    up = torch.cat((up, torch.randn(width - 2, 2, generator=g)))
    gate = torch.zeros_like(up)
    # Columns of zeros make the products many enough to be worth thirds.
    inputs = [pad(v, (500, 500)).to(gpu).requires_grad_() for v in (x, gate, up)]
    y = gated_projection(*inputs)
    pre = y.grad_fn.saved_tensors[3][1]
    want = x.double() @ up.double().t()
    size = x.double().abs() @ up.double().abs().t()
    pre, past = pre.cpu(), want.abs() > torch.finfo(torch.float32).max
    assert torch.equal(pre[past], torch.where(want[past] > 0, torch.inf, -torch.inf).float())
    pre, want, size = pre[~past], want[~past], size[~past]
    assert ((pre.double() - want).abs() <= 2.0 ** -22 * size + 2.0 ** -126).all()


@pytest.mark.parametrize("rows,dtype", [(9, torch.float32), (90, torch.float32), (9, torch.bfloat16),
                                        (90, torch.bfloat16)])
def test_infinities_stay_infinities(gpu, rows, dtype):
    """An infinity of x in a row makes infinities of its products with nonzero weights."""
    draw = Draw(gpu, 5)
    values = operands(draw, rows, 70, 20, dtype)
    clean = gated_projection(**values)
    values["x"][4, 69] = float("inf")
    kept = gated_projection(**leaves(values))
    pre = kept.grad_fn.saved_tensors[3]
    assert torch.equal(pre[:, 4], torch.stack([torch.where(values[k][:, 69] > 0, torch.inf, -torch.inf)
                                               for k in ("gate", "up")]))
    y = gated_projection(**values)
    y[4] = clean[4]
    assert torch.equal(y, clean)


def test_infinities_of_many_float32_rows(gpu):
    """Multiplied in parts of either sign, an infinity is none of a sign: its row or column is not
    finite, and no other one is touched."""
    draw = Draw(gpu, 5)
    values = operands(draw, 2000, 2500, 310, torch.float32)
    clean = gated_projection(**values)
    values["x"][4, 2499] = float("inf")
    values["up"][7, 3] = float("-inf")
    y = gated_projection(**values)
    assert not torch.isfinite(y[4]).any() and not torch.isfinite(y[:, 7]).any()
    y[4], y[:, 7] = clean[4], clean[:, 7]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("sizes", [(0, 5, 4), (3, 5, 0), (3, 0, 4), (30, 0, 4)])
def test_gated_of_nothing(gpu, sizes):
    M, K, F = sizes
    values = leaves({"x": torch.ones(M, K, device=gpu), "gate": torch.ones(F, K, device=gpu),
                     "up": torch.ones(F, K, device=gpu)})
    y = gated_projection(**values)
    assert y.shape == (M, F) and not y.any()
    for value, grad in zip(values.values(), torch.autograd.grad(y.sum(), list(values.values()))):
        assert grad.shape == value.shape and not grad.any()


@pytest.mark.parametrize("rows", [6, 70])
def test_not_a_number_stays_in_its_row_and_column(gpu, rows):
    draw = Draw(gpu, 1)
    values = operands(draw, rows, 100, 50, torch.bfloat16)
    clean = gated_projection(**values)
    values["x"][rows - 1, 99] = float("nan")
    values["up"][3, 0] = float("inf")
    y = gated_projection(**values)
    assert torch.isnan(y[rows - 1]).all() and not torch.isfinite(y[:, 3]).any()
    y[rows - 1], y[:, 3] = clean[rows - 1], clean[:, 3]
    assert torch.equal(y, clean)


def test_only_the_gradients_asked_for(gpu):
    draw = Draw(gpu, 2)
    values, dy = operands(draw, 40, 64, 48, torch.bfloat16), draw(40, 48, dtype=torch.bfloat16)
    inputs = leaves(values)
    every = torch.autograd.grad(gated_projection(**inputs), list(inputs.values()), dy)
    for k, name in enumerate(values):
        one = {**values, name: values[name].detach().requires_grad_()}
        got = torch.autograd.grad(gated_projection(**one), one[name], dy)[0]
        assert torch.equal(got, every[k]), name


def test_gated_streams_and_captures(gpu):
    """In two streams at once, and in replays of a captured forward: the same bits."""
    draw = Draw(gpu, 4)
    for shape in ((4, 500, 60), (300, 260, 90)):
        values, dy = operands(draw, *shape, torch.float32), draw(shape[0], shape[2])

        def passes():
            inputs = leaves(values)
            y = gated_projection(**inputs)
            return (y, *torch.autograd.grad(y, list(inputs.values()), dy))

        first, others = passes(), []
        torch.cuda.synchronize()
        for stream in [torch.cuda.Stream() for _ in range(2)]:
            with torch.cuda.stream(stream):
                others.append(passes())
        torch.cuda.synchronize()
        for other in others:
            assert all(torch.equal(a, b) for a, b in zip(first, other))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = gated_projection(**values)
        for k in range(4):
            values["x"].copy_(draw(*shape[:2]))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, gated_projection(**values)), k


def test_gated_refusals(gpu):
    draw = Draw(gpu, 0)
    good = operands(draw, 4, 6, 5, torch.float32)
    for change, message in (
            ({"x": good["x"].double()}, "float32, bfloat16 or float16"),
            ({"x": good["x"].cpu()}, "on a GPU"), ({"gate": good["gate"][:, :5]}, "gate must be a"),
            ({"up": good["up"].half()}, "up must be float32"), ({"up": None}, "up must be a"),
            ({"gate": good["gate"].cpu()}, "gate must be on x's device"),
            ({"up": good["up"][:4]}, "the same shape"), ({"activation": "relu"}, "silu' or 'gelu")):
        with pytest.raises(ValueError, match=message):
            gated_projection(**{**good, **change})
    tall = torch.zeros(1, 1, device=gpu, requires_grad=True).expand((1 << 21) + 1, 1)
    with pytest.raises(ValueError, match="up to 2097152 rows"):
        gated_projection(tall, torch.ones(1, 1, device=gpu), torch.ones(1, 1, device=gpu))


# ---- dropout -------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9, 1), (3, 5, 11), (4096, 3), (2049,)])
def test_dropout_follows_the_generator(gpu, shape, dtype):
    """The mask number by number, and the values: one product, one sum, one rounding."""
    draw = Draw(gpu, len(shape))
    x, residual, dy = (draw(*shape, dtype=dtype) for _ in range(3))
    for p, seed, offset, more in ((0.3, 12345, 0, residual), (0.5, -1, 1 << 40, None),
                                  (0.0, 7, 3, residual), (1.0, 7, 3, residual)):
        mask = bo.kept(x.numel(), p, seed, offset).view(shape)
        inputs = [v.detach().requires_grad_() for v in ((x, more) if more is not None else (x,))]
        y = dropout(inputs[0], p, seed=seed, offset=offset,
                    residual=inputs[1] if more is not None else None)
        scale = 65536 / max(1, 65536 - round(p * 65536))
        rest = 0 if more is None else more.double().cpu()
        kept = torch.where(mask, x.double().cpu() * scale, 0.0)
        want = kept + rest
        # The scale and the product are rounded, then the sum.
        within(y, want, 2 * U * kept.abs() + U * (kept.abs() + (rest.abs() if more is not None else 0)),
               f"p={p}")
        grads = torch.autograd.grad(y, inputs, dy)
        want = torch.where(mask, dy.double().cpu() * scale, 0.0)
        within(grads[0], want, 2 * U * want.abs(), f"dx, p={p}")
        if more is not None:
            assert torch.equal(grads[1], dy)


def test_dropout_drops_as_many_as_asked(gpu):
    """Of n = 2^22 elements a share p within five standard deviations, and no two neighbouring
    seeds or offsets alike."""
    n = 1 << 22
    ones = torch.ones(n, device=gpu)
    masks = [dropout(ones, 0.25, seed=s, offset=o) > 0 for s, o in ((1, 0), (2, 0), (1, 1))]
    for mask in masks:
        assert abs(float(mask.double().mean()) - 0.75) < 5 * (0.25 * 0.75 / n) ** 0.5
    both = [float((masks[0] & m).double().mean()) for m in masks[1:]]
    for share in both:
        assert abs(share - 0.75 ** 2) < 5 * (0.5625 * 0.4375 / n) ** 0.5


def test_dropout_does_not_look_at_what_it_drops(gpu):
    x = torch.full((1000,), float("nan"), device=gpu)
    mask = bo.kept(1000, 0.4, 9).to(gpu)
    y = dropout(x, 0.4, seed=9, residual=torch.ones(1000, device=gpu))
    assert torch.equal(torch.isnan(y), mask) and (y[~mask] == 1).all()


def test_dropout_of_views(gpu):
    """The mask goes by the place in x's own order, whatever its strides and alignment."""
    draw = Draw(gpu, 5)
    x, residual = draw(30, 41), draw(30, 41)
    want = dropout(x, 0.2, seed=3, residual=residual)
    turned = x.t().contiguous().t()
    assert torch.equal(dropout(turned, 0.2, seed=3, residual=residual), want)
    late = torch.cat((x.new_zeros(1), x.flatten()))[1:].view(30, 41)   # 4 bytes past 16
    assert torch.equal(dropout(late, 0.2, seed=3, residual=residual), want)
    assert dropout(x[:0], 0.2, seed=3).shape == (0, 41)


def test_dropout_seed_on_the_gpu(gpu):
    """A seed tensor gives the integer's mask, replays follow it, and a backward notices a
    changed one."""
    draw = Draw(gpu, 6)
    x = draw(500)
    seed = torch.tensor([77], device=gpu)
    assert torch.equal(dropout(x, 0.5, seed=seed), dropout(x, 0.5, seed=77))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.5, seed=seed, offset=2)
    for value in (77, -5, 1 << 50):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dropout(x, 0.5, seed=value, offset=2))
    leaf = x.clone().requires_grad_()
    y = dropout(leaf, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_refusals(gpu):
    x = torch.ones(4, device=gpu)
    for args, message in (
            (dict(x=x.double(), p=0.1, seed=1), "float32, bfloat16 or float16"),
            (dict(x=x.cpu(), p=0.1, seed=1), "on a GPU"), (dict(x=x, p=1.5, seed=1), "probability"),
            (dict(x=x, p=float("nan"), seed=1), "probability"),
            (dict(x=x, p=0.1, seed=1.5), "seed must be"), (dict(x=x, p=0.1, seed=None), "seed must be"),
            (dict(x=x, p=0.1, seed=torch.ones(1, device=gpu)), "one int64"),
            (dict(x=x, p=0.1, seed=torch.ones(1, dtype=torch.int64)), "one int64"),
            (dict(x=x, p=0.1, seed=1, offset=0.5), "offset must be"),
            (dict(x=x, p=0.1, seed=1, residual=x[:3]), "like x"),
            (dict(x=x, p=0.1, seed=1, residual=x.half()), "like x")):
        with pytest.raises(ValueError, match=message):
            dropout(**args)


def test_no_backward_under_capture(gpu, monkeypatch):
    """Refused from the query alone: no stream is captured here."""
    x = torch.ones(3, 4, device=gpu, requires_grad=True)
    w = torch.ones(5, 4, device=gpu)
    signal = torch.ones(2, 1, 4, device=gpu, requires_grad=True)
    outs = {"dropout": dropout(x, 0.1, seed=1), "gated_projection": gated_projection(x, w, w),
            "gated_recurrence": gated_recurrence(signal, signal, signal, torch.ones(4, device=gpu))[0]}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for name, out in outs.items():
        with pytest.raises(RuntimeError, match=f"{name} cannot be captured"):
            out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,F", [(40, 130, 44), (4400, 1000, 50)])
def test_gated_gradients_of_some(gpu, rows, K, F, dtype):
    """Gradients asked for one at a time, or two, are those of all three, bit for bit."""
    draw = Draw(gpu, rows)
    values = operands(draw, rows, K, F, dtype)
    dy = draw(rows, F, dtype=dtype)

    def gradients(names):
        inputs = {k: v.clone().requires_grad_(k in names) for k, v in values.items()}
        return torch.autograd.grad(gated_projection(**inputs), [inputs[k] for k in names], dy)

    want = dict(zip(values, gradients(list(values))))
    for names in (["x"], ["gate"], ["up"], ["gate", "up"], ["x", "up"]):
        for name, got in zip(names, gradients(names)):
            assert torch.equal(got, want[name]), names
