"""4-bit products through every kernel that their plan chooses between, and to the last bit (MI355X).

``test_exact_products`` takes inputs whose sums are exact in float32 in any order, so that nothing but
the result's own rounding is left.  Weights: one column of each row has a code off its zero point, scales
are powers of two.  Rows: neighbours are v and -v, or 1 + w and 1 - w, with sizes of one binade, so that
the sums over a stretch are whole multiples of one small number and stay below 2^24 of it, part by part:

* bfloat16 v has 8 bits: products with 16 + code, up to 31, are multiples of 2^-7, and 128 of them
  below 2^13: 20 bits; float16 v has 11: 23 bits;
* float32 v = 1 + a 2^-7 + b 2^-15 + c 2^-23 (a, c below 128, b in [64, 128)) has the parts 1 + a 2^-7,
  a multiple of 2^-16 below 2^-8, and one of 2^-23 of at most 2^-17: 20, 20 and 18 bits; its mean over
  a stretch is zero.  A missing part leaves an error of 2^-17 or 2^-9 of the result;
* float32 1 + w, w = b 2^-16 in [1/4, 1/2): the mean is 1, and w has the parts of 8 and 7 bits.

The three parts' sums are joined with one rounding, that of the product itself.
"""

from __future__ import annotations

import pytest
import torch

import block_oracle as bo
from signal_oracle import wide
from test_gpu_group_scaled import check_product, weight_of
from test_gpu_signal import Draw
from neurosim_gpu import Q4Tensor, q4_product

pytestmark = pytest.mark.gpu

GROUPS = (32, 64, 128, 256)
# M, N, K.  16 bits: rows straight from memory with one, two and four strips; two, three and four tiles of
# rows with one strip and with two, one chunk of columns a part of K and several; many tiles of rows;
# more than 24 parts of K.
HALF_SHAPES = [(1, 16, 32), (5, 300, 700), (8, 4200, 300), (16, 12_300, 260), (20, 129, 1300),
               (20, 17_000, 600), (33, 260, 1000), (33, 1200, 14_000), (45, 33_000, 700), (64, 16, 260),
               (64, 12_000, 1100), (700, 300, 1301), (2000, 1100, 1301), (33, 40, 30_000)]
# float32: one, two and four tiles of four rows, the same.
FLOAT_SHAPES = [(3, 33, 97), (3, 3200, 4900), (1, 70, 31_000), (7, 50, 333), (7, 16_000, 1600), (40, 70, 4100),
                (2000, 260, 1301)]
CASES = ([(torch.bfloat16, s) for s in HALF_SHAPES] + [(torch.float16, s) for s in HALF_SHAPES]
         + [(torch.float32, s) for s in FLOAT_SHAPES])


def pairs(values, K, add):
    """[M, K] of neighbours add + v, add - v."""
    both = torch.stack((add + values, add - values), -1).flatten(-2)
    return torch.nn.functional.pad(both, (0, K - both.shape[-1]), value=add)


def exact_rows(g, M, K, dtype, around_one):
    def integers(low, high):
        return torch.randint(low, high, (M, K // 2), generator=g).double()

    if dtype == torch.float32 and around_one:
        rows = pairs(integers(2 ** 14, 2 ** 15) * 2.0 ** -16, K, 1.0)
    elif dtype == torch.float32:
        rows = pairs(1 + integers(0, 128) * 2.0 ** -7 + integers(64, 128) * 2.0 ** -15
                     + integers(1, 128) * 2.0 ** -23, K, 0.0)
    else:
        bits = 7 if dtype == torch.bfloat16 else 10
        rows = pairs(1 + integers(0, 2 ** bits) * 2.0 ** -bits, K, 0.0)
    assert torch.equal(rows.to(dtype).double(), rows)
    return rows.to(dtype)


def one_column_weight(g, N, K, group, zeros):
    """(weight on the CPU, the column of each row, its value)."""
    groups = -(-K // group)
    zero = torch.randint(0, 16, (N, groups), generator=g) if zeros else torch.full((N, groups), 8)
    scale = 2.0 ** torch.randint(-3, 4, (N, groups), generator=g).double()
    codes = zero.to(torch.uint8).repeat_interleave(group, 1)[:, :K].contiguous()
    column = (torch.arange(N) * 7 + 3) % K
    row, own = torch.arange(N), column // group
    code = (zero[row, own] + torch.randint(1, 16, (N,), generator=g)) % 16
    codes[row, column] = code.to(torch.uint8)
    value = (code - zero[row, own]).double() * scale[row, own]
    return (bo.q4_pack(codes), scale, zero.to(torch.uint8) if zeros else None), column, value


@pytest.mark.parametrize("dtype,shape", CASES)
def test_exact_products(gpu, dtype, shape):
    M, N, K = shape
    for group in GROUPS:
        g = torch.Generator().manual_seed(sum(shape) + group)
        (codes, scale, zero), column, value = one_column_weight(g, N, K, group, group != 64)
        weight = Q4Tensor(codes.to(gpu), scale.to(torch.bfloat16).to(gpu),
                          None if zero is None else zero.to(gpu), K, group)
        for around_one in ((False, True) if dtype == torch.float32 else (False,)):
            x = exact_rows(g, M, K, dtype, around_one)
            want = (wide(x)[:, column] * value).to(dtype)
            got = q4_product(x.to(gpu), weight).cpu()
            assert torch.equal(got, want), (group, around_one)


@pytest.mark.parametrize("dtype,shape", CASES)
def test_products(gpu, dtype, shape):
    """Any codes and values, within the bounds of test_gpu_group_scaled.py."""
    M, N, K = shape
    draw = Draw(gpu, sum(shape))
    groups = GROUPS[:3] if N * K < 4_000_000 else ((32, 64, 128)[N % 3],)
    for group in groups:
        weight = weight_of(draw, gpu, N, K, group, zeros=(M + group) % 3 > 0)
        check_product((draw(M, K) + 0.5).to(dtype), *weight, bias=draw(N))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [2, 6, 30, 70])
def test_a_large_value_on_a_weight_of_zero(gpu, dtype, M):
    """It adds nothing to the result, but to its error: within the same bounds, which count |x| (for
    float32 its distance from the mean) whatever its weight."""
    draw = Draw(gpu, M)
    N, K = 90, 700
    x = draw(M, K).to(dtype)
    x[:, 130] = 2.0 ** 14
    for group in GROUPS[:3]:
        _, codes, scale, zero = weight_of(draw, gpu, N, K, group, zeros=True)
        codes[:, 130] = zero[:, 130 // group]
        weight = Q4Tensor(bo.q4_pack(codes).to(gpu), scale.to(gpu), zero.to(gpu), K, group)
        check_product(x, weight, codes, scale, zero)
