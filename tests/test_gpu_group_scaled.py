"""4-bit integer groups: quantisation bit for bit, products against float64 (MI355X).

Tolerance of a product.  With u = 2^-24, over a group of G columns the matrix cores sum
x (16 + u) exactly as products, with at most 2 u of error an addition (they may cut off), and
(16 + zero) times the sum of x, itself off by G u of the sum of sizes, is taken off: at most
(2 G + G + 6) u times 2 (16 + 15) the sum of |x| in the group, twice that where zero points pass 15.
Float32 rows are taken around their mean, whose part is exact but for its own few roundings, so
the same holds with |x - mean| in place of |x|, and (G + 8) u of |mean| |sum (u - zero)|.  The
scaled groups are then summed, (groups + 3) u of their sizes, and rounded once.
"""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from signal_oracle import wide
from test_gpu_block import within
from test_gpu_signal import U, Draw
from neurosim_gpu import Q4Tensor, q4_dequantize, q4_product, q4_quantize

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


# ---- quantisation --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (4, 200), (7, 256), (2, 1000)])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("symmetric", [False, True])
def test_quantisation(gpu, shape, group, symmetric, dtype):
    draw = Draw(gpu, sum(shape) + group)
    x = draw(*shape, dtype=dtype) + 0.3
    x[0, 0] = 0
    if shape[0] > 2:
        x[1] = x[1].abs() + 0.1                 # one sign only
        x[2] = 0
    for scales in (torch.bfloat16, torch.float32, torch.float16):
        got = q4_quantize(x, group, symmetric=symmetric, dtype=scales)
        codes, scale, zero = bo.q4_codes(x, group, symmetric, scales)
        assert torch.equal(got.codes.cpu(), bo.q4_pack(codes))
        assert torch.equal(got.scales.cpu(), scale)
        assert (got.zeros is None) if symmetric else torch.equal(got.zeros.cpu(), zero)
        want = bo.q4_values(codes, scale, zero, group)
        for back in TYPES:
            values = q4_dequantize(got, back)
            assert torch.equal(values.cpu(), want.float().to(back))    # one product, rounded
    assert got.shape == x.shape and torch.equal(got.dequantize(), q4_dequantize(got))


def test_ends_of_the_range(gpu):
    """Infinities and NaN, values whose scale overflows or vanishes in its type, the largest."""
    x = torch.zeros(8, 64, device=gpu)
    x[0, 3], x[1, 40], x[2, 5] = float("inf"), float("nan"), float("-inf")
    x[3], x[4] = 3e38, -3e38
    x[4, :20] = 3e38
    x[5], x[6] = 1e-44, 1e30
    x[7, 0] = -1.0
    for scales in (torch.float32, torch.float16, torch.bfloat16):
        for symmetric in (False, True):
            got = q4_quantize(x, 32, symmetric=symmetric, dtype=scales)
            codes, scale, zero = bo.q4_codes(x, 32, symmetric, scales)
            assert torch.equal(got.codes.cpu(), bo.q4_pack(codes))
            assert torch.equal(torch.isnan(got.scales.cpu()), torch.isnan(scale))
            assert torch.equal(torch.nan_to_num(got.scales.cpu()), torch.nan_to_num(scale))
            if not symmetric:
                assert torch.equal(got.zeros.cpu(), zero)
            values = q4_dequantize(got).cpu()
            assert torch.equal(torch.isnan(values), torch.isnan(bo.q4_values(codes, scale, zero, 32)))


def test_quantisation_of_views(gpu):
    draw = Draw(gpu, 1)
    x = draw(6, 5, 70)
    want = q4_quantize(x, 64)
    for other in (x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = q4_quantize(other, 64)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.zeros, want.zeros)
    assert q4_quantize(x[:0], 64).codes.shape == (0, 5, 48)
    assert q4_quantize(x[..., :0], 64).dequantize().shape == (6, 5, 0)


# ---- products ------------------------------------------------------------------------

def weight_of(draw, gpu, N, K, group, zeros, scales=torch.bfloat16):
    g = draw.g
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    groups = -(-K // group)
    scale = (torch.rand(N, groups, generator=g) + 0.1).mul(K ** -0.5).to(scales)
    zero = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None
    weight = Q4Tensor(bo.q4_pack(codes).to(gpu), scale.to(gpu),
                      zero.to(gpu) if zeros else None, K, group)
    return weight, codes, scale, zero


def check_product(x, weight, codes, scale, zero, bias=None):
    group, K = weight.group, weight.columns
    y = q4_product(x, weight, bias=bias)
    rows, values = wide(x), bo.q4_values(codes, scale, zero, group)
    want = rows @ values.t()
    # Sums go over stretches of 128 columns at most, which are the groups or parts of them.
    span = min(group, 128)
    stretches = -(-K // span)
    room = torch.zeros(*rows.shape[:-1], stretches * span, dtype=torch.float64)
    room[..., :K] = rows
    parts = room.unflatten(-1, (-1, span))
    count = torch.clamp(K - span * torch.arange(stretches), 0, span).double()
    mean = parts.sum(-1) / count.clamp(min=1)
    real = torch.arange(span) < count[:, None]
    size = parts.abs()
    spread = bo.q4_values(torch.ones_like(codes), scale, torch.zeros_like(scale, dtype=torch.uint8),
                          group)[:, ::span]                       # each stretch's scale
    if x.dtype == torch.float32:
        size = torch.where(real, (parts - mean.unsqueeze(-1)).abs(), 0.0)
        off = torch.zeros(codes.shape[0], stretches * span, dtype=torch.float64)
        off[:, :K] = (values / bo.q4_values(torch.ones_like(codes), scale,
                                            torch.zeros_like(scale, dtype=torch.uint8), group)).abs()
        around = mean.abs() @ (spread * off.unflatten(-1, (-1, span)).sum(-1)).t()
    else:
        around = torch.zeros(())
    bound = 62 * (3 * span + 6) * U * (size.sum(-1) @ spread.t()) + (span + 8) * U * around
    bound = bound + (stretches + 3) * U * (rows.abs() @ values.abs().t())
    if bias is not None:
        want = want + wide(bias)
        bound = bound + U * (want.abs() + wide(bias).abs())
    within(y, want, bound, f"y {list(x.shape)} {list(weight.shape)} {group}")
    return y


SHAPES = [  # M, N, K: one row, few, tiles' and chunks' edges, more than a tile, long sums, odd ends
    (1, 1, 1), (1, 16, 32), (1, 130, 1024), (2, 33, 97), (3, 300, 700), (4, 17, 128), (5, 50, 2100),
    (16, 70, 515), (17, 40, 300), (21, 129, 1300), (33, 260, 1000), (64, 16, 260), (70, 31, 600),
    (150, 90, 333), (1, 20, 9000), (20, 9, 4500), (2, 2100, 64),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_products(gpu, shape, dtype):
    M, N, K = shape
    draw = Draw(gpu, sum(shape))
    for group in (32, 64, 128, 256):
        weight = weight_of(draw, gpu, N, K, group, zeros=(M + group) % 3 > 0)
        bias = draw(N) if N % 2 else None
        check_product((draw(M, K) + 0.5).to(dtype), *weight, bias=bias)


# Wide weights take more strips a wavefront, by rows; scales come to a workgroup in stretches of 64
# stages of 128 columns, or of fewer where few wavefronts share a strip.
@pytest.mark.parametrize("shape", [(16, 12_301, 260), (9, 12_288, 1100), (8, 12_289, 2300), (7, 4200, 1030),
                                   (16, 4100, 8500), (12, 12_300, 130), (24, 9000, 1100)])
def test_wide_weights(gpu, shape):
    M, N, K = shape
    draw = Draw(gpu, sum(shape))
    for group, scales in ((32, torch.float32), (64, torch.float16), (128, torch.bfloat16), (384, torch.float32)):
        dtype = (torch.bfloat16, torch.float16)[group % 3 == 0]
        check_product((draw(M, K) + 0.5).to(dtype), *weight_of(draw, gpu, N, K, group, group != 64, scales))


@pytest.mark.parametrize("scales", TYPES)
def test_scale_types_and_strange_zeros(gpu, scales):
    draw = Draw(gpu, 5)
    for K, group in ((300, 32), (300, 64), (900, 128), (900, 1024)):
        weight, codes, scale, zero = weight_of(draw, gpu, 50, K, group, True, scales)
        check_product(draw(3, K), weight, codes, scale, zero)
        zero = zero + 9                          # up to 24: the bound's 62 covers 31 twice
        strange = Q4Tensor(weight.codes, weight.scales, zero.to(gpu), K, group)
        check_product(draw(3, K), strange, codes, scale, zero)


def test_quantised_weight_and_rates(gpu):
    """A read-out of rates, all positive, through quantised weights: as the values say."""
    draw = Draw(gpu, 2)
    dense, rates = draw(40, 1111), draw(2, 3, 1111).abs()
    for symmetric in (False, True):
        weight = q4_quantize(dense, 128, symmetric=symmetric)
        y = q4_product(rates, weight)
        want = wide(rates) @ wide(weight.dequantize()).t()
        assert y.shape == (2, 3, 40)
        assert (wide(y) - want).abs().max() <= 3e-6 * want.abs().max()


def test_codes_past_the_columns_count_for_nothing(gpu):
    draw = Draw(gpu, 3)
    weight, *_ = weight_of(draw, gpu, 20, 70, 32, True)
    for dtype in TYPES:
        x = draw(5, 70, dtype=dtype)
        want = q4_product(x, weight)
        filled = weight.codes.clone()
        filled[:, 35:] = 255
        other = Q4Tensor(filled, weight.scales, weight.zeros, 70, 32)
        assert torch.equal(q4_product(x, other), want)


def test_not_a_number_stays_in_its_row(gpu):
    draw = Draw(gpu, 4)
    weight, *_ = weight_of(draw, gpu, 40, 300, 64, True)
    for dtype in TYPES:
        x = draw(19, 300, dtype=dtype)
        clean = q4_product(x, weight)
        x[3, 299], x[18, 0], x[7, 100] = float("nan"), float("inf"), float("-inf")
        y = q4_product(x, weight)
        bad = torch.tensor([3, 7, 18], device=gpu)
        assert torch.isnan(y[bad]).all()
        y[bad] = clean[bad]
        assert torch.equal(y, clean)
    scales = weight.scales.clone()
    scales[5, 1] = float("nan")
    y = q4_product(draw(3, 300), Q4Tensor(weight.codes, scales, weight.zeros, 300, 64))
    assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, :5]).all() and torch.isfinite(y[:, 6:]).all()


def test_strides_alignment_and_shapes(gpu):
    draw = Draw(gpu, 6)
    weight, *_ = weight_of(draw, gpu, 30, 200, 128, True)
    for dtype in TYPES:
        x = draw(9, 200, dtype=dtype)
        want = q4_product(x, weight)
        room = torch.full((9, 211), float("nan"), dtype=dtype, device=gpu)
        room[:, 3:203] = x
        assert torch.equal(q4_product(room[:, 3:203], weight), want)
        assert torch.equal(q4_product(x.t().contiguous().t(), weight), want)
        assert torch.equal(q4_product(x.view(3, 3, 200), weight), want.view(3, 3, 30))
        assert torch.equal(q4_product(x[0], weight), q4_product(x[:1], weight)[0])
        assert torch.equal(q4_product(x[:1].expand(9, 200), weight)[8], want[0])
        assert q4_product(x[:0], weight).shape == (0, 30)
    empty = Q4Tensor(weight.codes[:, :0].contiguous(), weight.scales[:, :0].contiguous(), None, 0, 32)
    bias = draw(30)
    assert torch.equal(q4_product(draw(2, 0), empty, bias=bias), bias.expand(2, 30))
    none = Q4Tensor(weight.codes[:0], weight.scales[:0], None, 200, 128)
    assert q4_product(draw(2, 200), none).shape == (2, 0)


def test_streams_and_captures(gpu):
    draw = Draw(gpu, 7)
    for M, N, K in ((1, 900, 5000), (40, 70, 4100)):      # K shared by workgroups: two launches
        weight, *_ = weight_of(draw, gpu, N, K, 128, True)
        x = draw(M, K)
        first, others = q4_product(x, weight), []
        torch.cuda.synchronize()
        for stream in [torch.cuda.Stream() for _ in range(2)]:
            with torch.cuda.stream(stream):
                others.append(q4_product(x, weight))
        torch.cuda.synchronize()
        assert all(torch.equal(first, other) for other in others)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = q4_product(x, weight)
            back = q4_quantize(x, 64).dequantize()
        for k in range(4):
            x.copy_(draw(M, K))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, q4_product(x, weight)), k
            assert torch.equal(back, q4_quantize(x, 64).dequantize()), k


def test_refusals(gpu):
    draw = Draw(gpu, 0)
    weight, *_ = weight_of(draw, gpu, 8, 100, 32, True)
    codes, scales, zeros = weight.codes, weight.scales, weight.zeros
    for args, message in (
            ((codes, scales, zeros, 100, 48), "32, 64 or a multiple"),
            ((codes, scales, zeros, 100, 0), "32, 64 or a multiple"),
            ((codes, scales, zeros, (1 << 23) + 1, 32), "at most"),
            ((codes, scales, zeros, 130, 32), "codes must be uint8"),
            ((codes.int(), scales, zeros, 100, 32), "codes must be uint8"),
            ((codes, scales, zeros, 100, 64), "scales must be"),
            ((codes, scales.double(), zeros, 100, 32), "scales must be"),
            ((codes, scales, zeros[:, :2], 100, 32), "zeros must be"),
            ((codes, scales, zeros.int(), 100, 32), "zeros must be"),
            ((codes[:4], scales, zeros, 100, 32), "the same rows"),
            ((codes, scales.cpu(), None, 100, 32), "the same rows"),
            ((codes, scales.t().contiguous().t(), zeros, 100, 32), "contiguous"),
            ((torch.cat((codes.flatten(), codes.flatten()[:8]))[8:].view(8, 64), scales, zeros, 100, 32),
             "16-byte aligned")):
        with pytest.raises(ValueError, match=message):
            Q4Tensor(*args)
    x = draw(3, 100)
    for args, kw, message in (
            ((x, codes), {}, "Q4Tensor"), ((x.double(), weight), {}, "float32, bfloat16 or float16"),
            ((x[:, :99], weight), {}, "99 columns"), ((x.cpu(), weight), {}, "same GPU"),
            ((x, weight), {"bias": draw(7)}, "bias must be"),
            ((x, weight), {"bias": draw(8).half()}, "bias must be"),
            ((x.clone().requires_grad_(), weight), {}, "no gradients")):
        with pytest.raises(ValueError, match=message):
            q4_product(*args, **kw)
    for args, kw, message in (
            ((x, 100), {}, "32, 64 or a multiple"), ((x, 32), {"dtype": torch.float64}, "scales are"),
            ((x.cpu(), 32), {}, "on a GPU"), ((x.clone().requires_grad_(), 32), {}, "no gradients")):
        with pytest.raises(ValueError, match=message):
            q4_quantize(*args, **kw)
    with pytest.raises(ValueError, match="read back as"):
        weight.dequantize(torch.int8)
