"""Generation end to end: a prompt through the whole-sequence kernels and the same tokens one by one
through the recurrent step give the same logits, for every mixer variant; the 4-bit model is the LM with
its weights rounded; a captured loop draws what an uncaptured one does.

Tolerance: relative L2 3e-2 between the two ways in bf16, as for the LM's bf16 layers against fp32."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

VARIANTS = {
    "lm": dict(),
    "rope_gqa": dict(num_kv_heads=2, use_rope=True, qk_norm=True),
    "l2_group_rope": dict(use_rope=True, rope_group=True, qk_norm=True, norm_q="l2", norm_k="l2", use_short_conv=False),
    "decay": dict(use_decay=True),
    "sum": dict(feature_map="kata_quadratic_sum"),
}


def make(**kw):
    from linatt_b200.lm import KataLM, KataLMConfig

    torch.manual_seed(0)
    cfg = KataLMConfig(**{**dict(hidden_size=256, num_hidden_layers=2, num_heads=4, spd_num_groups=4, vocab_size=512,
                                 initializer_range=0.06, max_position_embeddings=128), **kw})
    return KataLM(cfg).cuda()


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("name", VARIANTS)
def test_steps_continue_a_prompt(name):
    from linatt_b200.generate import KataGenerator

    gen = KataGenerator(make(**VARIANTS[name]))
    ids = torch.randint(0, 512, (3, 24), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    whole = {n: gen.prefill(ids[:, :n]).float() for n in (18, 21, 24)}
    logits = gen.prefill(ids[:, :17])
    for t in range(17, 24):
        logits = gen.step(ids[:, t])
        if t + 1 in whole:
            assert rel(logits, whole[t + 1]) < 3e-2, (name, t)


def test_a_prompt_is_the_lm_with_rounded_weights():
    from linatt_b200.generate import KataGenerator
    from linatt_b200.quant import quantize_w4, w4_linear

    lm = make()
    gen = KataGenerator(lm, group_size=32)
    ids = torch.randint(0, 512, (2, 40), device="cuda")
    got = gen.prefill(ids)
    with torch.no_grad():
        for blk in lm.model.layers:
            for lin in (blk.attn.q_proj, blk.attn.k_proj, blk.attn.v_proj, blk.attn.o_proj, blk.mlp.gate_proj,
                        blk.mlp.up_proj, blk.mlp.down_proj):
                w = quantize_w4(lin.weight, 32, dtype=torch.bfloat16)
                lin.weight.copy_(w4_linear(torch.eye(lin.in_features, device="cuda", dtype=torch.bfloat16), w).T.float())
        with torch.autocast("cuda", torch.bfloat16):
            want = lm(ids)[:, -1]
    assert rel(got, want) < 3e-2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_converted_model_generates_as_its_own_values(dtype):
    """Parameters in 16 bits: the same as fp32 parameters of the same values."""
    from linatt_b200.generate import KataGenerator

    lm = make(use_rope=True, qk_norm=True).to(dtype)
    for p in lm.parameters():
        if p.dim() == 1:  # norm weights that differ
            torch.nn.init.uniform_(p, 0.5, 1.5)
    ids = torch.randint(0, 512, (3, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    gen = KataGenerator(lm, dtype=dtype)
    got = [gen.prefill(ids[:, :19]), gen.step(ids[:, 19])]
    gen = KataGenerator(lm.float(), dtype=dtype)
    want = [gen.prefill(ids[:, :19]), gen.step(ids[:, 19])]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("head", [False, True])
def test_generate_captured_and_not(head):
    from linatt_b200 import check_device_status
    from linatt_b200.generate import KataGenerator

    gen = KataGenerator(make(), quantize_head=head)
    ids = torch.randint(0, 512, (4, 9), device="cuda")
    u = torch.rand(12, 4, device="cuda")
    par = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    a, la = gen.generate(ids, 12, u=u, **par)
    b, lb = gen.generate(ids, 12, u=u, use_graph=False, **par)
    check_device_status()
    assert torch.equal(a, b) and torch.equal(la, lb)
    assert a.shape == (4, 12) and (0 <= a).all() and (a < 512).all() and (la <= 0).all()
    greedy, _ = gen.generate(ids, 1, temperature=0.0)
    assert torch.equal(greedy[:, 0], gen.prefill(ids).float().argmax(-1))


def test_steps_end_at_the_last_position():
    """The last position that the rotation tables have is used, the next one refused; without a rotation there is none."""
    from linatt_b200.generate import KataGenerator

    ids = torch.randint(0, 512, (2, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    gen = KataGenerator(make(use_rope=True))
    gen.prefill(ids[:, :126])
    for t in (126, 127):
        assert torch.isfinite(gen.step(ids[:, t])).all()
    with pytest.raises(ValueError, match="max_positions"):
        gen.step(ids[:, 0])
    gen.generate(ids[:, :120], 8)  # the last of eight is drawn and not passed on
    assert torch.isfinite(gen.step(ids[:, 0])).all()
    with pytest.raises(ValueError, match="max_positions"):
        gen.step(ids[:, 0])
    gen = KataGenerator(make())
    gen.prefill(ids)
    assert torch.isfinite(gen.step(ids[:, 0])).all()


def test_generate_refusals():
    from linatt_b200.generate import KataGenerator

    lm = make(use_rope=True)
    gen = KataGenerator(lm)
    ids = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        gen.step(ids[:, 0])
    with pytest.raises(ValueError):
        gen.generate(ids, 124)
    with pytest.raises(ValueError):
        gen.generate(ids, 0)
    with pytest.raises(ValueError):
        gen.generate(ids, 3, u=torch.rand(2, 2, device="cuda"))
    with pytest.raises(ValueError):
        gen.prefill(ids[:, :0])
    with pytest.raises(RuntimeError):
        gen.prefill(ids.cpu())
    with pytest.raises(TypeError):
        KataGenerator(lm, dtype=torch.float32)
    with pytest.raises(ValueError):
        KataGenerator(make(use_offset_gate=True))
