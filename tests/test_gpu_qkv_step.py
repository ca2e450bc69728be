"""GPU parity of the one-token q/k/v step against a float64 statement of it.

Everything between the inputs and the one rounding of q, k and v is fp32: at most K + 12 roundings on
a value's way, a norm of at most 256 values, and a rotation that adds two of them.  A value may be off
by one rounding to its type and by 64 fp32 units of the size of what it was added up from (the head's
largest value; for the convolution the sum of |w x|)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
EPS_Q, EPS_K = 1e-5, 1e-6


def reference(x, pos, ring, cw, HQ, H, D, Dv, norms, ws, rope, R, cos, sin):
    x = x.double()
    B = x.shape[0]
    size = x.abs()
    K = 0 if cw is None else cw.shape[1]
    new = ring
    if K:
        a, size = x * cw[:, K - 1].double(), (x * cw[:, K - 1].double()).abs()
        new = None if ring is None else ring.clone()
        for b in range(B):
            for j in range(1, K):
                t = ring[b, (pos[b].item() - j) % (K - 1)].double() * cw[:, K - 1 - j].double()
                a[b] += t
                size[b] += t.abs()
            if new is not None:
                new[b, pos[b].item() % (K - 1)] = x[b].to(new.dtype)
        x = a * torch.sigmoid(a)
    out, at = [], 0
    for n, (heads, dim) in enumerate(((HQ, D), (H, D), (H, Dv))):
        y = x[:, at:at + heads * dim].view(B, heads, dim)
        s = size[:, at:at + heads * dim].view(B, heads, dim).amax(-1, keepdim=True).expand_as(y).clone()
        at += heads * dim
        if n < 2:
            if norms[n] != "none":
                f = y.square().sum(-1, keepdim=True) / (dim if norms[n] == "rms" else 1)
                f = torch.rsqrt(f + (EPS_Q, EPS_K)[n]) * (1.0 if ws[n] is None else ws[n].double())
                y, s = y * f, s * f.abs().amax(-1, keepdim=True)
            if rope:
                c, sn = cos[pos].double()[:, None], sin[pos].double()[:, None]
                if rope == 1:
                    p, q = y[..., 0::2], y[..., 1::2]
                    y = torch.stack((p * c - q * sn, p * sn + q * c), -1).flatten(-2)
                else:
                    g = y.view(B, heads, dim // R, 2, R // 2)
                    p, q = g[..., 0, :], g[..., 1, :]
                    c, sn = c[:, :, None], sn[:, :, None]
                    y = torch.stack((p * c - q * sn, p * sn + q * c), -2).reshape(B, heads, dim)
        out.append((y, s))
    return out, new


CASES = [  # B, HQ, H, D, Dv, K, norm_q, norm_k, weights, rope, R, dtype
    (1, 12, 12, 64, 64, 4, "none", "none", False, 0, 0, torch.bfloat16),
    (3, 8, 2, 128, 64, 4, "rms", "rms", True, 1, 128, torch.bfloat16),
    (5, 4, 4, 64, 128, 3, "l2", "l2", False, 2, 16, torch.float16),
    (2, 3, 3, 80, 40, 2, "rms", "l2", True, 2, 80, torch.float32),
    (7, 2, 1, 96, 96, 4, "none", "rms", False, 1, 96, torch.float32),
    (4, 1, 1, 8, 8, 1, "l2", "none", False, 1, 8, torch.float16),
    (300, 6, 3, 32, 256, 4, "rms", "rms", True, 2, 32, torch.bfloat16),
    (9, 5, 5, 256, 8, 0, "rms", "l2", True, 2, 64, torch.float32),
    (700, 16, 8, 128, 128, 4, "l2", "rms", True, 1, 128, torch.float16),
]


def build(B, HQ, H, D, Dv, K, nq, nk, weights, rope, R, dtype, T=50):
    from linatt_b200.qkv_step import QKVStep

    g = torch.Generator(device="cuda").manual_seed(B * 31 + D)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    C = (HQ + H) * D + H * Dv
    cw = randn(C, K) * 0.5 if K else None
    ws = [1 + 0.2 * randn(D) if weights and n == "rms" else None for n in (nq, nk)]
    ang = randn(T, R // 2) if rope else None
    cos, sin = (ang.cos(), ang.sin()) if rope else (None, None)
    step = QKVStep(num_heads=HQ, num_kv_heads=H, head_k_dim=D, head_v_dim=Dv, conv_weight=cw, norm_q=nq, norm_k=nk,
                   q_weight=ws[0], k_weight=ws[1], eps_q=EPS_Q, eps_k=EPS_K, rope=rope, rope_dim=R, cos=cos, sin=sin)
    x = randn(B, C).to(dtype)
    ring = randn(B, K - 1, C).to(dtype) if K > 1 else None
    pos = torch.randint(0, T, (B,), device="cuda", generator=g)
    return step, x, pos, ring, (cw, HQ, H, D, Dv, (nq, nk), ws, rope, R, cos, sin)


def check(got, want, dtype):
    for y, (ref, size) in zip(got, want):
        tol = UNIT[dtype] * ref.abs() * 1.01 + 64 * 2.0 ** -24 * size * (1 + UNIT[dtype]) + TINY[dtype]
        bad = ((y.double() - ref).abs() > tol).sum().item()
        assert bad == 0, f"{bad} of {y.numel()} values off by more than the arithmetic allows"


@pytest.mark.parametrize("case", CASES)
def test_qkv_step(case):
    B, dtype = case[0], case[-1]
    step, x, pos, ring, rest = build(*case)
    for _ in range(2):  # the second step reads the ring that the first one wrote
        old = None if ring is None else ring.clone()
        want, new = reference(x, pos, old, *rest)
        got = step(x, pos, ring)
        assert [tuple(t.shape) for t in got] == [(B, case[1], case[3]), (B, case[2], case[3]), (B, case[2], case[4])]
        assert all(t.dtype == dtype for t in got)
        check(got, want, dtype)
        if ring is not None:
            assert torch.equal(ring, new)
        x, pos = x.flip(0), (pos + 1) % 50


def test_qkv_step_of_strided_rows():
    case = (6, 4, 4, 64, 64, 4, "rms", "rms", True, 1, 64, torch.bfloat16)
    step, x, pos, ring, rest = build(*case)
    want, _ = reference(x, pos, ring.clone(), *rest)
    wide = torch.zeros(6, x.shape[1] + 24, device="cuda", dtype=x.dtype)
    for at in (0, 8, 3):
        wide[:, at:at + x.shape[1]] = x
        check(step(wide[:, at:at + x.shape[1]], pos, ring.clone()), want, x.dtype)
    r = ring[:1].clone()
    check(step(x[:1].expand(1, -1), pos[:1], r), [(a[:1], s[:1]) for a, s in want], x.dtype)
    assert step(x[:0], pos[:0], ring[:0])[0].shape == (0, 4, 64)


def test_qkv_step_positions_out_of_the_tables_give_nan_and_keep_the_ring():
    case = (4, 2, 2, 64, 64, 4, "rms", "rms", True, 1, 64, torch.float32)
    step, x, pos, ring, rest = build(*case)
    pos[1], pos[2] = 50, -1
    old = ring.clone()
    q, k, v = step(x, pos, ring)
    for t in (q, k, v):
        assert torch.isnan(t[1:3]).all() and torch.isfinite(t[[0, 3]]).all()
    assert torch.equal(ring[1:3], old[1:3]) and not torch.equal(ring[0], old[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_qkv_steps_continue_the_layer_of_whole_sequences(dtype):
    """A prompt through the training kernels (short convolution, norms, rotation) and its tokens one
    by one through the step give the same q, k and v: fp32 to 1e-5; bf16 to two roundings more, those
    between the separate kernels, 2^-7 of the head's largest value."""
    from linatt_b200.mixer import ShortConvQKVFunction, rope_tables, row_norm
    from linatt_b200.qkv_step import QKVStep

    B, T, H, D, K = 2, 9, 4, 64, 4
    g = torch.Generator(device="cuda").manual_seed(0)
    C = H * D
    x = torch.randn(B, T, 3 * C, device="cuda", generator=g).to(dtype)
    cw = [torch.randn(C, 1, K, device="cuda", generator=g) * 0.5 for _ in range(3)]
    qw, kw = (1 + 0.1 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
    cos, sin = rope_tables(16, D, 10000.0, x.device, torch.float32)
    q, k, v = ShortConvQKVFunction.apply(x, True, *cw)
    q, k = (row_norm(t.reshape(-1, D), w, norm="rms", eps=1e-5, cos=cos, sin=sin, rope=1, rope_dim=D, heads=H, T=T)
            for t, w in ((q, qw), (k, kw)))
    want = [t.reshape(B, T, H, D) for t in (q, k, v)]
    step = QKVStep(num_heads=H, head_k_dim=D, head_v_dim=D, conv_weight=torch.cat(cw), norm_q="rms", norm_k="rms",
                   q_weight=qw, k_weight=kw, rope=1, rope_dim=D, cos=cos, sin=sin)
    ring = step.new_ring(B, dtype, x.device)
    for t in range(T):
        if t == 5:
            assert torch.equal(ring, step.ring_of(x[:, :5]))
        got = step(x[:, t], torch.full((B,), t, device="cuda"), ring)
        for a, b in zip(got, want):
            tol = (1e-5 if dtype == torch.float32 else 2.0 ** -7) * b[:, t].float().abs().amax(-1, keepdim=True)
            assert ((a.float() - b[:, t].float()).abs() <= tol).all()


def test_qkv_step_refusals():
    from linatt_b200.qkv_step import QKVStep

    kw = dict(num_heads=4, num_kv_heads=2, head_k_dim=64, head_v_dim=64)
    C = 6 * 64 + 2 * 64
    cw = torch.randn(C, 4, device="cuda")
    tab = torch.ones(8, 32, device="cuda")
    for bad in (dict(num_kv_heads=3), dict(head_k_dim=60), dict(head_v_dim=264), dict(norm_q="layer"),
                dict(conv_weight=cw[1:]), dict(conv_weight=torch.randn(C, 5, device="cuda")),
                dict(q_weight=torch.ones(63, device="cuda")), dict(rope=3), dict(rope=1, rope_dim=64),
                dict(rope=1, rope_dim=32, cos=tab, sin=tab), dict(rope=2, rope_dim=24, cos=tab, sin=tab)):
        with pytest.raises(ValueError):
            QKVStep(**{**kw, **bad})
    with pytest.raises(RuntimeError):
        QKVStep(**kw, conv_weight=cw.cpu())
    step = QKVStep(**kw, conv_weight=cw)
    x, pos = torch.zeros(3, C, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    ring = step.new_ring(3, torch.float32, "cuda")
    for bad in ((x[:, 1:], pos, ring), (x, pos.int(), ring), (x, pos[:2], ring), (x, pos, None),
                (x, pos, ring.half()), (x, pos, ring.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            step(*bad)
    with pytest.raises(TypeError):
        step(x.double(), pos, ring)
    with pytest.raises(RuntimeError):
        step(x.cpu(), pos.cpu(), ring.cpu())


def test_silu_of_fp32_channels_to_a_few_units():
    """a / (1 + exp(-a)) with a given exactly (one tap of weight 1): an exponential of up to 2 units, a sum and a
    quotient of half a unit each, and a factor below 1 on the first two."""
    from linatt_b200.qkv_step import QKVStep

    step = QKVStep(num_heads=1, head_k_dim=256, head_v_dim=256, conv_weight=torch.ones(768, 1, device="cuda"))
    a = torch.linspace(-87, 87, 768 * 64, device="cuda").view(64, 768)
    q, k, v = step(a, torch.zeros(64, device="cuda", dtype=torch.int64))
    got = torch.cat((q.flatten(1), k.flatten(1), v.flatten(1)), 1).double()
    ref = a.double() * torch.sigmoid(a.double())
    assert ((got - ref).abs() <= 3.01 * 2.0 ** -23 * ref.abs()).all()
