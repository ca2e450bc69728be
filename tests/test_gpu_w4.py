"""GPU parity of the 4-bit linear layer against a float64 statement of it, element by element.

The bound on an output follows from the arithmetic: products are exact, sums are fp32 (at most
K/16 + K/g + 16 of them in a row, each losing at most 4 units of the last place of a partial sum,
itself at most S = sum |w x|), and the output is rounded once to its type."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def make(N, K, g, dtype, zeros, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    code = torch.randint(0, 16, (N, 8 * 4 * (-(-K // 32))), device="cuda", generator=gen)  # codes past K too
    packed = sum((code[:, i::8] << (4 * i)) for i in range(8))
    packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
    G = -(-K // g)
    scales = ((0.2 + torch.rand(N, G, device="cuda", generator=gen)) * 0.05).to(dtype)
    z = torch.randint(0, 16, (N, G), device="cuda", generator=gen, dtype=torch.uint8) if zeros else None
    of = torch.arange(K, device="cuda") // g
    W = (code[:, :K].double() - (z.double()[:, of] if zeros else 8.0)) * scales.double()[:, of]
    return packed, scales, z, W


def check(y, x, W, g, swiglu):
    K, dt = W.shape[1], y.dtype
    ref, S = x.double() @ W.T, x.double().abs() @ W.abs().T
    err = (K / 16 + K / g + 16) * 4 * 2.0 ** -23 * S
    if swiglu:
        h = W.shape[0] // 2
        a, b, ea, eb = ref[:, :h], ref[:, h:], err[:, :h], err[:, h:]
        silu = a * torch.sigmoid(a)
        ref = silu * b
        # |silu'| <= 1.1; the logistic function itself is computed to a few units
        err = 1.1 * ea * (b.abs() + eb) + silu.abs() * eb + 8 * 2.0 ** -23 * ref.abs()
    tol = err + UNIT[dt] * (ref.abs() + err) * 1.01 + TINY[dt]
    bad = ((y.double() - ref).abs() > tol).sum().item()
    assert bad == 0, f"{bad} of {y.numel()} outputs off by more than the arithmetic allows"


CASES = [  # rows, N, K, group, dtype, zeros, swiglu
    (1, 16, 128, 128, torch.bfloat16, False, False),
    (1, 1, 1, 32, torch.bfloat16, True, False),
    (1, 768, 768, 64, torch.bfloat16, False, False),
    (2, 17, 33, 32, torch.float16, True, False),
    (3, 500, 1000, 64, torch.float32, True, False),
    (2, 2304, 768, 128, torch.float32, False, False),
    (5, 333, 4100, 32, torch.float16, True, False),
    (7, 1000, 129, 128, torch.bfloat16, True, False),
    (8, 4096, 768, 64, torch.bfloat16, False, True),
    (9, 130, 640, 256, torch.bfloat16, False, False),
    (1, 2 * 37, 513, 384, torch.float16, True, True),
    (16, 2048, 2048, 128, torch.bfloat16, False, False),
    (17, 100, 16500, 128, torch.bfloat16, False, False),
    (33, 515, 1111, 32, torch.bfloat16, True, False),
    (64, 1024, 1024, 128, torch.bfloat16, False, True),
    (11, 200, 9000, 64, torch.float32, False, True),
    (100, 300, 512, 64, torch.float16, True, False),
    (257, 144, 1000, 128, torch.bfloat16, False, True),
    (300, 390, 2000, 32, torch.float32, True, False),
    (513, 1030, 640, 128, torch.float16, False, False),
]


@pytest.mark.parametrize("rows,N,K,g,dtype,zeros,swiglu", CASES)
def test_w4_linear(rows, N, K, g, dtype, zeros, swiglu):
    from linatt_b200 import check_device_status
    from linatt_b200.quant import W4Weight, w4_linear

    packed, scales, z, W = make(N, K, g, dtype, zeros, seed=N * 7 + K)
    w = W4Weight(packed, scales, z, in_features=K, group_size=g, activation="swiglu" if swiglu else None)
    x = torch.randn(rows, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows)).to(dtype)
    y = w4_linear(x, w)
    check_device_status()
    assert y.shape == (rows, N // 2 if swiglu else N) and y.dtype == dtype
    check(y, x, W, g, swiglu)
    assert torch.equal(y, w4_linear(x, w))  # and the same bits again


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_w4_linear_of_strided_and_unaligned_rows(rows):
    from linatt_b200.quant import W4Weight, w4_linear

    N, K, g = 200, 384, 128
    packed, scales, z, W = make(N, K, g, torch.bfloat16, False, seed=3)
    w = W4Weight(packed, scales, z, in_features=K, group_size=g)
    big = torch.randn(rows, 2 * K + 3, device="cuda").bfloat16()
    for x in (big[:, 1:K + 1], big[:, 8:K + 8], big[:, ::2][:, :K], big[:1, :K].expand(rows, K)):
        check(w4_linear(x, w), x, W, g, False)
    x3 = big[:, :K].reshape(rows, 1, K)
    y3 = w4_linear(x3, w)
    assert y3.shape == (rows, 1, N)
    check(y3[:, 0], x3[:, 0], W, g, False)
    assert w4_linear(x3[:0], w).shape == (0, 1, N)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_w4_linear_keeps_infinities_and_nan_in_their_rows(dtype):
    from linatt_b200.quant import W4Weight, w4_linear

    N, K = 48, 256
    packed, scales, z, W = make(N, K, 64, dtype, True, seed=5)
    w = W4Weight(packed, scales, z, in_features=K, group_size=64)
    x = torch.randn(40, K, device="cuda").to(dtype)
    x[1, 7], x[3, 9], x[30, 0] = float("inf"), float("nan"), float("inf")
    y = w4_linear(x, w)
    fine = torch.ones(40, dtype=torch.bool, device="cuda")
    fine[[1, 3, 30]] = False
    check(y[fine], x[fine], W, 64, False)
    ref = x.double() @ W.T
    for r in (1, 3, 30):
        assert torch.equal(torch.isfinite(y[r]), torch.isfinite(ref[r]))
        assert torch.equal(torch.isnan(y[r]), torch.isnan(ref[r]))


def test_w4_fp32_rows_are_used_in_full():
    """Large and tiny fp32 values: nothing of x is rounded before the product."""
    from linatt_b200.quant import W4Weight, w4_linear

    packed, scales, z, W = make(64, 300, 128, torch.float32, False, seed=6)
    w = W4Weight(packed, scales, z, in_features=300, group_size=128)
    x = torch.randn(2, 300, device="cuda") * torch.tensor([[3e36], [1e-30]], device="cuda")
    check(w4_linear(x, w), x, W, 128, False)


def test_w4_linear_on_another_stream_and_in_a_graph():
    from linatt_b200.quant import W4Weight, w4_linear

    packed, scales, z, W = make(512, 512, 64, torch.bfloat16, False, seed=8)
    w = W4Weight(packed, scales, z, in_features=512, group_size=64)
    for rows in (4, 128):
        x = torch.randn(rows, 512, device="cuda").bfloat16()
        want = w4_linear(x, w)
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            y = w4_linear(x, w)
        st.synchronize()
        assert torch.equal(y, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            yg = w4_linear(x, w)
        x.copy_(x.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        check(yg, x, W, 64, False)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("N,K,g", [(64, 256, 64), (40, 300, 128), (7, 31, 32)])
def test_quantize_w4_is_within_half_a_step(N, K, g, symmetric):
    """Every weight is within half a code step of its own value (a whole one where the clipped end
    of the asymmetric range loses up to half a step to the rounded zero point), read back through
    products with unit vectors."""
    from linatt_b200.quant import quantize_w4, w4_linear

    W = torch.randn(N, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N)) * 0.1
    w = quantize_w4(W, g, symmetric=symmetric, dtype=torch.float32)
    back = w4_linear(torch.eye(K, device="cuda"), w).T
    G = -(-K // g)
    pad = torch.nn.functional.pad(W, (0, G * g - K)).view(N, G, g)
    step = pad.abs().amax(-1) / 7 if symmetric else (pad.amax(-1).clamp(min=0) - pad.amin(-1).clamp(max=0)) / 15
    step = step.repeat_interleave(g, 1)[:, :K]
    assert ((back - W).abs() <= (0.5 if symmetric else 1.0) * step * 1.001).all()


def test_w4_refusals():
    from linatt_b200.quant import W4Weight, quantize_w4, w4_linear

    packed, scales, z, _ = make(32, 128, 64, torch.bfloat16, True, seed=1)
    with pytest.raises(ValueError):
        W4Weight(packed[:, :-1], scales, z, in_features=128, group_size=64)
    with pytest.raises(ValueError):
        W4Weight(packed, scales[:, :1], z, in_features=128, group_size=64)
    with pytest.raises(TypeError):
        W4Weight(packed.long(), scales, z, in_features=128, group_size=64)
    with pytest.raises(TypeError):
        W4Weight(packed, scales.double(), z, in_features=128, group_size=64)
    with pytest.raises(ValueError):
        W4Weight(packed, scales, z, in_features=128, group_size=64, activation="gelu")
    with pytest.raises(ValueError):
        W4Weight(packed, scales[:, :1], None, in_features=128, group_size=160)  # neither 32, 64 nor whole 128s
    with pytest.raises(ValueError):
        W4Weight(packed[:31], scales[:31], None, in_features=128, group_size=64, activation="swiglu")  # odd rows
    with pytest.raises(RuntimeError):
        W4Weight(packed.cpu(), scales.cpu(), None, in_features=128, group_size=64)
    w = W4Weight(packed, scales, z, in_features=128, group_size=64)
    with pytest.raises(TypeError):
        w4_linear(torch.zeros(1, 128, device="cuda"), w)
    with pytest.raises(ValueError):
        w4_linear(torch.zeros(1, 127, device="cuda", dtype=torch.bfloat16), w)
    with pytest.raises(RuntimeError):
        w4_linear(torch.zeros(1, 128, dtype=torch.bfloat16), w)
    with pytest.raises(ValueError):
        quantize_w4(torch.zeros(4, 4, 4, device="cuda"))
