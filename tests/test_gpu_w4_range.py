"""Rows of x whose values differ by many orders of magnitude, through the 4-bit linear layer: a product is exact
whatever lies beside it, so a value counts in full where a larger one meets the zero point.  The bound is that of
the layer's other tests: fp32 sums of at most K/16 + K/g + 16 terms, each losing at most 4 units of the last place
of a partial sum, itself at most S = sum |w x| (a value that meets the zero point adds nothing to S), and one
rounding of the output."""

from __future__ import annotations

import pytest
import torch

from test_gpu_w4 import UNIT, check

pytestmark = pytest.mark.gpu


def weight(N, K, g, dtype, zeros, at, seed=0):
    """Codes with the zero point at the places `at` of every row, as (W4Weight, W in float64)."""
    from linatt_b200.quant import W4Weight

    gen = torch.Generator(device="cuda").manual_seed(seed)
    G, words = -(-K // g), 4 * (-(-K // 32))
    code = torch.randint(0, 16, (N, 8 * words), device="cuda", generator=gen)
    z = torch.randint(0, 16, (N, G), device="cuda", generator=gen, dtype=torch.uint8) if zeros else None
    of = torch.arange(K, device="cuda") // g
    zero = z.long()[:, of] if zeros else torch.full((N, K), 8, device="cuda")
    code[:, :K][:, at] = zero[:, at]
    packed = sum((code[:, i::8] << (4 * i)) for i in range(8))
    packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
    scales = ((0.2 + torch.rand(N, G, device="cuda", generator=gen)) * 0.05).to(dtype)
    W = (code[:, :K].double() - zero.double()) * scales.double()[:, of]
    return W4Weight(packed, scales, z, in_features=K, group_size=g), W


DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ROWS = [1, 2, 3, 4, 5, 6, 8, 10, 11, 40]


def rows_of(rows, K, seed):
    return torch.randn(rows, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("K,g,zeros", [(768, 64, False), (1000, 32, True), (515, 128, True)])
def test_small_values_beside_large_ones(rows, K, g, zeros, dtype):
    """A large value in every 128 (in some rows only) whose weight is zero."""
    from linatt_b200.quant import w4_linear

    at = torch.arange(5, K, 128, device="cuda")
    w, W = weight(200, K, g, dtype, zeros, at)
    for ratio in (2.0 ** 7, 2.0 ** 11, 2.0 ** 14, 2.0 ** 24, 2.0 ** 60):
        small = 0.05 if dtype != torch.float16 else 2.0 ** -8
        x = rows_of(rows, K, seed=rows) * small
        big = small * ratio * 1.37 if dtype != torch.float16 else min(small * ratio * 1.37, 6e4)
        x[::2, at] = big
        x[-1, at] = -big
        x = x.to(dtype)
        check(w4_linear(x, w), x, W, g, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
def test_values_of_every_size(rows, dtype):
    """Magnitudes spread over the type's range, all but the smallest at the zero point of a few rows of the weight."""
    from linatt_b200.quant import w4_linear

    K, g, N = 700, 64, 64
    lo, hi = (-20, 8) if dtype == torch.float16 else (-60, 60)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = rows_of(rows, K, seed=rows)
    x = (x * 2.0 ** (lo + (hi - lo) * torch.rand(rows, K, device="cuda", generator=gen))).to(dtype)
    sizes = x.abs().amax(0)
    for keep in (K, K // 2, 20, 1):
        w, W = weight(N, K, g, dtype, True, sizes.argsort()[keep:], seed=keep)
        check(w4_linear(x, w), x, W, g, False)


@pytest.mark.parametrize("rows", [1, 3, 6])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_smallest_and_the_largest_values(rows, dtype):
    """Down to 2^-124 and up to the largest value, alone and beside each other."""
    from linatt_b200.quant import w4_linear

    K, g = 300, 128
    at = torch.arange(3, K, 128, device="cuda")
    w, W = weight(96, K, g, dtype, False, at)
    big = torch.finfo(dtype).max
    tiny = (rows_of(rows, K, seed=4).clamp(-4, 4) * 2.0 ** -110).to(dtype)
    check(w4_linear(tiny, w), tiny, W, g, False)
    tiny[:, at] = big
    check(w4_linear(tiny, w), tiny, W, g, False)
    full = torch.full((rows, K), big / 2 ** 10, device="cuda", dtype=dtype)
    full[:, at] = big
    check(w4_linear(full, w), full, W, g, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 5, 11, 70])
def test_the_largest_values_under_the_largest_codes(rows, dtype):
    """Codes of 15 over zero points of 0, and the reverse: outputs just inside the type's range."""
    from linatt_b200.quant import W4Weight, w4_linear

    N, K, g = 48, 256, 128
    code = torch.full((N, K), 15, device="cuda")
    code[1::2] = 0
    packed = torch.where(code[:, ::8] == 15, -1, 0).to(torch.int32).contiguous()
    z = torch.where(code[:, ::g] == 15, 0, 15).to(torch.uint8).contiguous()
    scales = torch.full((N, 2), 2.0 ** -12, device="cuda", dtype=dtype)
    W = (code.double() - z.double().repeat_interleave(g, 1)) * 2.0 ** -12
    w = W4Weight(packed, scales, z, in_features=K, group_size=g)
    x = torch.full((rows, K), torch.finfo(dtype).max, device="cuda", dtype=dtype)
    y = w4_linear(x, w)
    assert torch.isfinite(y).all()
    check(y, x, W, g, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K,zeros", [(1, 40001, True), (3, 9000, False), (5, 8192, True), (6, 4100, False), (10, 2500, True)])
def test_more_small_values_than_are_kept_on_chip(rows, K, zeros, dtype):
    """A large value in every 128 of long rows, and the same bits from a second call."""
    from linatt_b200.quant import w4_linear

    at = torch.arange(77, K, 128, device="cuda")
    w, W = weight(70, K, 128, dtype, zeros, at)
    x = rows_of(rows, K, seed=K) * 2.0 ** -8
    x[:, at] = 3e4
    x = x.to(dtype)
    y = w4_linear(x, w)
    check(y, x, W, 128, False)
    assert torch.equal(y, w4_linear(x, w))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 5, 11])
def test_infinities_beside_small_values(rows, dtype):
    """Infinities and NaN give what the definition gives, and nothing to the other rows."""
    from linatt_b200.quant import w4_linear

    K, g = 384, 64
    w, W = weight(80, K, g, dtype, True, torch.tensor([130], device="cuda"))
    x = (rows_of(rows, K, seed=9) * 0.01).to(dtype)
    x[1, 130], x[1, 3] = 300.0, 2.0 ** -9
    y0 = w4_linear(x, w)
    check(y0, x, W, g, False)
    for bad in (float("inf"), -float("inf"), float("nan")):
        xb = x.clone()
        xb[0, 7] = bad
        y, ref = w4_linear(xb, w), xb.double() @ W.T
        assert torch.equal(y[1:], y0[1:])
        assert torch.equal(torch.isnan(y[0]), torch.isnan(ref[0]))
        inf = torch.isinf(ref[0])
        assert torch.equal(y[0][inf].double(), ref[0][inf]) and torch.equal(torch.isinf(y[0]), inf)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_gives_the_same_with_more_rows(dtype):
    """One row alone and among eleven: the same to the bound of the sums, at any spread."""
    from linatt_b200.quant import w4_linear

    K, g = 512, 128
    at = torch.arange(0, K, 128, device="cuda")
    w, W = weight(64, K, g, dtype, False, at)
    x = (rows_of(11, K, seed=2) * 0.02).to(dtype)
    x[:, at] = 5e4
    many = w4_linear(x, w)
    err = (K / 16 + K / g + 16) * 4 * 2.0 ** -23 * (x.double().abs() @ W.abs().T)
    for r in range(3):
        one = w4_linear(x[r:r + 1], w)
        tol = 2 * err[r] + 2.1 * UNIT[dtype] * (many[r].double().abs() + err[r]) + (2.0 ** -24 if dtype == torch.float16 else 0)
        assert ((one[0].double() - many[r].double()).abs() <= tol).all()
