"""The 4-bit linear layer where a CTA of the streaming form does not have all of x in shared memory at once (long
rows), where it has more row tiles than it keeps sums of (tall weights), and both; and the same beyond its rows.
With 1 to 4 column tiles some 60 to 150, 30 to 60, 16 to 20 and 20 steps of 128 k fit, and the sums of 16 row tiles
(1 or 2 column tiles) or 4 are kept: the cases take 2 to 8 chunks, the last one of odd lengths too, and 5 and 17
tiles a CTA."""

from __future__ import annotations

import pytest
import torch

from test_gpu_w4 import check, make

pytestmark = pytest.mark.gpu

B, F, S = torch.bfloat16, torch.float16, torch.float32
CASES = [  # rows, N, K, group, dtype, zeros, swiglu, first column of x
    (5, 40, 11008, 128, B, False, False, 0),
    (5, 41, 11009, 32, F, True, False, 0),
    (4, 100, 14336, 64, B, True, True, 0),
    (3, 33, 30001, 128, F, False, False, 0),
    (1, 48, 70001, 32, S, True, False, 0),
    (2, 130, 66000, 128, B, False, True, 1),
    (3, 50, 20500, 64, S, False, False, 3),
    (4, 40, 9000, 128, S, True, False, 0),
    (6, 34, 5001, 32, S, True, True, 0),
    (8, 70, 9007, 128, B, True, False, 0),
    (10, 200, 5001, 32, F, True, False, 0),
    (2, 40001, 256, 128, B, False, False, 0),
    (5, 40001, 100, 32, F, True, False, 0),
    (1, 2 * 20001, 300, 64, S, False, True, 0),
    (7, 10001, 250, 64, B, False, False, 0),
    (6, 10001, 129, 32, S, True, False, 0),
    (5, 38000, 8200, 128, B, False, False, 0),
    (7, 10001, 5001, 64, B, True, False, 1),
    (10, 2 * 9601, 3001, 128, F, False, True, 1),
]


@pytest.mark.parametrize("rows,N,K,g,dtype,zeros,swiglu,first", CASES)
def test_long_rows_and_tall_weights(rows, N, K, g, dtype, zeros, swiglu, first):
    from linatt_b200 import check_device_status
    from linatt_b200.quant import W4Weight, w4_linear

    packed, scales, z, W = make(N, K, g, dtype, zeros, seed=N + K)
    w = W4Weight(packed, scales, z, in_features=K, group_size=g, activation="swiglu" if swiglu else None)
    x = torch.randn(rows, K + first, device="cuda", generator=torch.Generator(device="cuda").manual_seed(K))
    x = (x * 0.25).to(dtype)[:, first:]
    y = w4_linear(x, w)
    check(y, x, W, g, swiglu)
    assert torch.equal(y, w4_linear(x, w))
    if not swiglu:  # an infinity in the last chunk of one row, where its weight is not zero
        xi = x.clone()
        xi[-1, K - 1] = float("inf")
        yi, ref = w4_linear(xi, w), xi[-1].double() @ W.T
        assert torch.equal(yi[:-1], y[:-1])
        assert torch.equal(torch.isnan(yi[-1]), torch.isnan(ref)) and torch.equal(torch.isinf(yi[-1]), torch.isinf(ref))
    check_device_status()
