"""Microscaled 4-bit quantisation and product against value-by-value float64 (MI355X).

Codes, scale bytes and values read back are equal to the oracle's, bit for bit.  Products:
code products and block scales are exact, so only the float32 sums round; a sum of K terms
in any order, each addition off by at most one unit in the last place (2^-23 relative,
whether it rounds or truncates), is within K 2^-23 times the sum of the terms' sizes.
"""

from __future__ import annotations

import pytest
import torch

import signal_oracle as so
from neurosim_gpu import MXTensor, microscaled, mx_dequantize, mx_product, mx_quantize

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rows(gpu, seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g))
    return x.to(dtype).to(gpu)


def check_codes(x):
    q = mx_quantize(x)
    codes, scales = so.mx_quantize(x)
    assert q.shape == x.shape
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(so.unpack(q.codes.cpu()), codes)
    return q, codes, scales


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 64), (7, 100), (2, 3, 77),
                                   (130, 515), (40,)])
def test_codes_and_values(gpu, shape, dtype):
    x = rows(gpu, sum(shape), *shape, dtype=dtype)
    q, codes, scales = check_codes(x)
    want = so.mx_values(codes, scales, shape[-1])
    for out in (torch.float32, torch.bfloat16):      # both hold every value exactly
        assert torch.equal(mx_dequantize(q, out).double().cpu(), want)
    assert torch.equal(q.dequantize(torch.float16).cpu(), want.to(torch.float16))


@pytest.mark.parametrize("width", [2048, 2046, 2044, 2040])
def test_values_of_long_rows(gpu, width):
    """Rows on and off lines of 32 bytes; the values against the oracle's of a sample of rows."""
    x = rows(gpu, 47, 700, width)
    q = mx_quantize(x)
    some = torch.tensor([0, 1, 2, 350, 698, 699])
    want = so.mx_values(so.unpack(q.codes.cpu()[some]), q.scales.cpu()[some], width)
    for dtype in TYPES:
        assert torch.equal(mx_dequantize(q, dtype).cpu()[some], want.to(dtype))
    whole = mx_dequantize(q)
    assert torch.equal(mx_dequantize(q, torch.bfloat16).float(), whole)
    assert ((whole - x).abs().amax() <= x.abs().amax() / 4)      # a step of a block's top values


def test_every_rounding(gpu):
    """Every multiple of 1/64 of a block's unit, both signs, at scales over the whole range."""
    grid = torch.arange(0, 8 * 64, dtype=torch.float64) / 64
    grid = torch.cat((grid, -grid))
    for power in (-127, -126, -60, -1, 0, 1, 77, 124, 125):
        lines = torch.zeros(grid.numel() // 16, 32, dtype=torch.float64)
        lines[:, :16] = grid.reshape(-1, 16)
        lines[:, 16] = 4.0                            # the block's peak sets the scale at 2^power
        lines = lines * 2.0 ** power
        check_codes(lines.float().to(gpu))
    small = torch.full((4, 32), 2.0 ** -149)
    small[1] = -(2.0 ** -127)
    small[2] = 2.0 ** -126 * 1.5
    small[3, 1:] = 0.0
    check_codes(small.to(gpu))


def test_blocks_without_values(gpu):
    """Zeros of both signs, infinities and NaN: a block that holds one is NaN, its
    neighbours are not."""
    x = rows(gpu, 4, 6, 96)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 40], x[3, 5], x[4, 95] = float("inf"), float("nan"), float("-inf")
    q, codes, scales = check_codes(x)
    assert (scales == 255).sum() == 3 and scales[0].tolist() == [0, 0, 0]
    back = q.dequantize().cpu()
    assert torch.isnan(back[2, 32:64]).all() and torch.isfinite(back[2, :32]).all()
    weight = mx_quantize(rows(gpu, 5, 4, 96))
    y = mx_product(q, weight).cpu()
    assert torch.isnan(y[2:5]).all() and torch.isfinite(y[[0, 1, 5]]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_row_views(gpu, dtype):
    """Rows of a wider tensor at every alignment, transposes and broadcasts."""
    base = rows(gpu, 6, 9, 200, dtype=dtype)
    for x in (base[:, 1:78], base[:, 3:100], base[2:, 64:128], base.t(), base[:1].expand(5, 200),
              base[:, ::2]):
        check_codes(x)
    assert mx_quantize(base[:0]).shape == (0, 200)
    assert mx_dequantize(mx_quantize(base[:, :0])).shape == (9, 0)


PRODUCTS = [  # M, N, K
    (1, 1, 1), (1, 5, 32), (1, 300, 33), (2, 17, 100), (3, 64, 128), (5, 31, 500), (8, 700, 1000),
    (16, 16, 4096), (17, 33, 129), (31, 100, 3000), (33, 1000, 700), (64, 64, 64), (65, 130, 257),
    (100, 40, 5000), (128, 256, 512), (130, 257, 640), (256, 256, 256), (300, 500, 1100),
    (513, 259, 96), (700, 1030, 513),
]


def check_product(x, weight, bias, dtype):
    """x and weight MXTensors."""
    y = mx_product(x, weight, bias=bias, dtype=dtype)
    a = so.mx_values(so.unpack(x.codes.cpu()), x.scales, x.columns).reshape(-1, x.columns)
    b = so.mx_values(so.unpack(weight.codes.cpu()), weight.scales, weight.columns)
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, size = want + so.wide(bias), size + so.wide(bias).abs()
    assert y.shape == (*x.shape[:-1], weight.shape[0]) and y.dtype == dtype
    bound = (x.columns + 2) * 2.0 ** -23 * size
    bound = bound + HALF_ULP[dtype] * (want.abs() + bound) + 2.0 ** -24 * (dtype == torch.float16)
    error = (y.double().cpu().reshape(want.shape) - want).abs()
    assert (error <= bound).all(), float((error / bound).max())
    return y


@pytest.mark.parametrize("shape", PRODUCTS)
def test_product(gpu, shape):
    M, N, K = shape
    x, weight = rows(gpu, M, M, K), mx_quantize(rows(gpu, N + 7, N, K) / K ** 0.5)
    bias = rows(gpu, 3, N) if M % 2 else None
    q = mx_quantize(x)
    dtype = TYPES[(M + N) % 3]
    y = check_product(q, weight, bias, dtype)
    # A float x is quantised on the way: the same bits.
    assert torch.equal(mx_product(x, weight, bias=bias, dtype=dtype), y)


@pytest.mark.parametrize("shape", [(3500, 3400, 128), (3400, 3500, 96), (3333, 3600, 384),
                                   (3400, 3700, 1000), (3500, 3500, 640), (3329, 3585, 1024),
                                   (3500, 3456, 1000), (3400, 3456, 33)])
def test_product_of_many_rows(gpu, shape):
    """The 256 x 256 tiles, K of one stage to several, whole and with a part of one, scale
    rows of whole words (K a multiple of 128) and not; a sample of rows and columns."""
    M, N, K = shape
    x, weight = mx_quantize(rows(gpu, 40, M, K)), mx_quantize(rows(gpu, 41, N, K) / K ** 0.5)
    bias, dtype = rows(gpu, 42, N), TYPES[K % 3]
    y = mx_product(x, weight, bias=bias, dtype=dtype)
    m = torch.cat((torch.arange(0, 40), torch.arange(250, 262), torch.arange(M - 40, M)))
    n = torch.cat((torch.arange(0, 70), torch.arange(500, 530), torch.arange(N - 70, N)))
    a = so.mx_values(so.unpack(x.codes.cpu()[m]), x.scales.cpu()[m], K)
    b = so.mx_values(so.unpack(weight.codes.cpu()[n]), weight.scales.cpu()[n], K)
    want = a @ b.t() + so.wide(bias)[n]
    bound = (K + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t() + so.wide(bias).abs()[n])
    bound = bound + HALF_ULP[dtype] * (want.abs() + bound) + 2.0 ** -24 * (dtype == torch.float16)
    assert ((y.cpu()[m][:, n].double() - want).abs() <= bound).all()
    # The whole result against float32, to the bound of both sums and of one rounding more.
    whole = x.dequantize() @ weight.dequantize().t() + bias
    error = (y.float() - whole).norm() / whole.norm()
    assert error <= 2 * (HALF_ULP[dtype] + K * 2.0 ** -23)


@pytest.mark.parametrize("K", [96, 128, 160, 256, 384, 500, 640, 705, 896])
def test_blocks_without_numbers_stay_in_their_row(gpu, K):
    """The 256 x 256 tiles ask for scales past a row's end; those, another row's, may be NaN."""
    x, w = rows(gpu, 43, 3500, K), rows(gpu, 44, 3400, K) / K ** 0.5
    want = mx_product(x, mx_quantize(w))
    x[1::7, 0], w[2::5, 0] = float("nan"), float("nan")
    got = mx_product(x, mx_quantize(w))
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[1::7], bad[:, 2::5] = True, True
    assert torch.equal(got.isnan(), bad)
    assert torch.equal(got[~bad], want[~bad])


def test_scales_at_any_address(gpu):
    """Rows of scales need no alignment; few rows, small tiles and large ones."""
    for M, N, K in ((2, 300, 256), (100, 300, 256), (3500, 3400, 256), (3500, 3400, 200)):
        x, w = mx_quantize(rows(gpu, 45, M, K)), mx_quantize(rows(gpu, 46, N, K))
        moved = []
        for q in (x, w):
            scales = torch.empty(q.scales.numel() + 1, dtype=torch.uint8, device=gpu)[1:]
            moved.append(MXTensor(q.codes, scales.view(q.scales.shape).copy_(q.scales), K))
        assert moved[0].scales.data_ptr() % 4 == 1
        assert torch.equal(mx_product(*moved), mx_product(x, w))


@pytest.mark.parametrize("dtype", TYPES)
def test_product_keeps_leading_dimensions(gpu, dtype):
    x = rows(gpu, 8, 3, 5, 90, dtype=dtype)
    weight = mx_quantize(rows(gpu, 9, 21, 90))
    y = mx_product(x, weight)
    assert y.shape == (3, 5, 21) and y.dtype == dtype
    assert torch.equal(y.reshape(15, 21), mx_product(x.reshape(15, 90), weight))
    assert mx_product(x[0, 0], weight).shape == (21,)
    assert mx_product(x[:0], weight).shape == (0, 5, 21)
    assert mx_product(mx_quantize(x), weight).dtype == torch.float32


def test_product_without_columns(gpu):
    empty = mx_quantize(torch.zeros(4, 0, device=gpu))
    bias = rows(gpu, 10, 4)
    assert torch.equal(mx_product(torch.zeros(3, 0, device=gpu), empty, bias=bias),
                       bias.expand(3, 4))
    nothing = mx_quantize(torch.zeros(0, 64, device=gpu))
    assert mx_product(torch.zeros(3, 64, device=gpu), nothing).shape == (3, 0)


def test_scales_far_apart(gpu):
    """Blocks whose scales lie 2^60 apart, with sums that cancel, and results that
    overflow to infinity as a float32 sum does."""
    x, w = rows(gpu, 11, 20, 256), rows(gpu, 12, 40, 256)
    x[:, :32] *= 2.0 ** 60
    w[:, :32] *= 2.0 ** -60
    check_product(mx_quantize(x), mx_quantize(w), None, torch.float32)
    huge = torch.full((3, 64), 2.0 ** 100, device=gpu)
    assert torch.isinf(mx_product(huge, mx_quantize(huge))).all()


def test_results_repeat_bit_for_bit(gpu):
    for M, N, K in ((1, 1000, 4096), (40, 100, 20_000), (300, 300, 2000)):
        x, weight = rows(gpu, 13, M, K), mx_quantize(rows(gpu, 14, N, K))
        assert torch.equal(mx_product(x, weight), mx_product(x, weight))


def test_offsets_past_32_bits(gpu):
    """A weight of more than 2^31 bytes of codes, and float rows 2^31 elements apart."""
    N, K = 70_000, 65_536
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=gpu)
    scales = torch.randint(118, 122, (N, K // 32), dtype=torch.uint8, device=gpu)
    weight = MXTensor(codes, scales, K)
    x = mx_quantize(rows(gpu, 15, 2, K))
    y = mx_product(x, weight)
    tail = MXTensor(codes[-300:].clone(), scales[-300:].clone(), K)
    check_product(x, tail, None, torch.float32)
    a = so.mx_values(so.unpack(x.codes.cpu()), x.scales, K)
    b = so.mx_values(so.unpack(tail.codes.cpu()), tail.scales, K)
    bound = (K + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t()) * 1.01
    assert ((y[:, -300:].double().cpu() - a @ b.t()).abs() <= bound).all()
    back = mx_dequantize(weight, torch.bfloat16)
    assert torch.equal(back[-1].double().cpu(), b[-1])
    del back, codes, scales, weight
    far = 2 ** 31 + 32
    base = torch.zeros(far + 64, dtype=torch.bfloat16, device=gpu)
    apart = base.as_strided((2, 64), (far, 1))
    apart.copy_(rows(gpu, 16, 2, 64, dtype=torch.bfloat16))
    near = mx_quantize(apart.contiguous())
    assert torch.equal(mx_quantize(apart).codes, near.codes)


def test_other_streams_and_graphs(gpu):
    x, weight = rows(gpu, 17, 3, 300), mx_quantize(rows(gpu, 18, 50, 300))
    want = mx_product(x, weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(mx_product(x, weight), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx_product(x, weight)
    for seed in range(4):
        x.copy_(rows(gpu, 30 + seed, 3, 300))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mx_product(x, weight))
        torch.cuda.synchronize()


def test_refusals(gpu):
    def refuses(text, fn, *args, **kw):
        with pytest.raises(ValueError, match=text):
            fn(*args, **kw)

    x = rows(gpu, 20, 4, 64)
    weight = mx_quantize(rows(gpu, 21, 5, 64))
    refuses("on a GPU", mx_quantize, x.cpu())
    refuses("float32, bfloat16 or float16", mx_quantize, x.double())
    refuses("no gradients", mx_quantize, x.clone().requires_grad_())
    refuses("MXTensor on a GPU", mx_dequantize, x)
    refuses("read back as", mx_dequantize, weight, torch.float64)
    refuses(r"\[N, K\]", mx_product, x, x)
    refuses("64", mx_product, rows(gpu, 22, 4, 65), weight)
    refuses("63", mx_product, mx_quantize(rows(gpu, 22, 4, 63)), weight)
    refuses("float tensor or", mx_product, [1.0], weight)
    refuses("bias", mx_product, x, weight, bias=rows(gpu, 23, 4))
    refuses("bias", mx_product, x, weight, bias=rows(gpu, 23, 5).half())
    refuses("no gradients", mx_product, x, weight, bias=rows(gpu, 23, 5).requires_grad_())
    refuses("a product is", mx_product, x, weight, dtype=torch.float64)
    refuses("codes must be uint8", MXTensor, weight.codes[:, :-1], weight.scales, 64)
    refuses("scales must be uint8", MXTensor, weight.codes, weight.scales.int(), 64)
    refuses("contiguous", MXTensor, weight.codes.t().contiguous().t(), weight.scales, 64)
    refuses("same rows", MXTensor, weight.codes, weight.scales[:3], 64)
    lib = microscaled._library()
    args = microscaled._PRODUCT.pack(2, 32, 0, 0, 2, 32, 0, 0, 0, 0, 2, 0, 0, 0, 0, 0)
    assert lib.ns_mx_product(args, None) == 1
    assert b"codes and scales are required" in lib.ns_last_error()
    args = microscaled._PRODUCT.pack(2, 2 ** 24, 0, 0, 2, 2 ** 24, 0, 0, 0, 0, 2, 0, 0, 0, 0, 0)
    assert lib.ns_mx_product(args, None) == 1
    assert b"at most 8388608 columns" in lib.ns_last_error()


@pytest.mark.parametrize("shape", [(17, 64, 256), (64, 64, 1792), (20, 130, 2048), (300, 500, 1024),
                                   (40, 100, 20_000), (33, 200, 50_000), (70, 90, 50_176)])
def test_small_tiles_of_whole_and_many_stages(gpu, shape):
    """The 64 x 64 tiles where K ends with a whole stage of 256 (their last requests then bring
    nothing that is read, into the LDS that the results pass through), and where it is cut into
    many parts, of whole stages and not."""
    M, N, K = shape
    x, weight = mx_quantize(rows(gpu, 50, M, K)), mx_quantize(rows(gpu, 51, N, K) / K ** 0.5)
    bias = rows(gpu, 52, N)
    for dtype in TYPES:
        y = check_product(x, weight, bias, dtype)
        for _ in range(3):
            assert torch.equal(mx_product(x, weight, bias=bias, dtype=dtype), y)


def test_forward_mode_derivatives_are_refused(gpu):
    from torch.autograd import forward_ad

    x, weight, bias = rows(gpu, 60, 4, 64), mx_quantize(rows(gpu, 61, 5, 64)), rows(gpu, 62, 5)
    with forward_ad.dual_level():
        dual, dual_bias = (forward_ad.make_dual(v, torch.ones_like(v)) for v in (x, bias))
        for call in (lambda: mx_quantize(dual), lambda: mx_product(dual, weight),
                     lambda: mx_product(x, weight, bias=dual_bias)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        mx_product(x, weight, bias=bias)


@pytest.mark.parametrize("shape", [(1, 300, 8192), (16, 17, 8000), (3, 1000, 7937), (8, 2000, 8100)])
def test_few_rows_with_the_longest_sums(gpu, shape):
    """Up to 16 rows with K near 8192, the longest that one workgroup sums by itself: no
    workspace, one launch."""
    M, N, K = shape
    assert microscaled._library().ns_mx_product_bytes(M, N, K, 0) == 0
    x, weight = mx_quantize(rows(gpu, 63, M, K)), mx_quantize(rows(gpu, 64, N, K) / K ** 0.5)
    for dtype in TYPES:
        check_product(x, weight, rows(gpu, 65, N), dtype)
