"""The C entries of the generation operators refuse bad arguments on the host (no GPU is touched), and
their Python fronts refuse CPU tensors."""

from __future__ import annotations

import pytest
import torch

from linatt_b200 import _lib


@pytest.fixture(scope="module")
def L():
    from linatt_b200 import build

    build.build()
    return _lib.lib()


def w4(**kw):
    return _lib.W4WeightArgs(**{**dict(data=16, N=32, K=128, group=64, dtype=1, gated=0, zeros=0), **kw})


def test_w4_sizes(L):
    # tiles of 16 rows (8 pairs of a gated weight), steps of 128 k: 1 KB of codes and 16 scales (zeros) a group
    assert L.kata_w4_bytes(w4()) == 2 * (1024 + 2 * 16 * 2)
    assert L.kata_w4_bytes(w4(N=33, K=129, group=32, dtype=0, zeros=1)) == 3 * 2 * (1024 + 4 * 16 * 5)
    assert L.kata_w4_bytes(w4(N=34, K=700, group=256, gated=1)) == 3 * 6 * (1024 + 16 * 2)
    assert L.kata_w4_bytes(w4(group=48)) == 0


def test_w4_refusals(L):
    ok = (16, 128, 16, 32, 1, None, 0, None, None)
    assert L.kata_w4_linear(None, *ok) == -1
    assert L.kata_w4_linear(w4(dtype=3), *ok) == -2
    for bad in (dict(group=0), dict(group=16), dict(group=96), dict(group=130), dict(N=0), dict(K=0),
                dict(N=31, gated=1), dict(N=1 << 25)):
        assert L.kata_w4_linear(w4(**bad), *ok) == -3, bad
    assert L.kata_w4_linear(w4(gated=2), *ok) == -1
    assert L.kata_w4_linear(w4(zeros=2), *ok) == -1
    assert L.kata_w4_linear(w4(data=None), *ok) == -1
    assert L.kata_w4_linear(w4(data=24), *ok) == -4
    assert L.kata_w4_linear(w4(), None, 128, 16, 32, 1, None, 0, None, None) == -1
    assert L.kata_w4_linear(w4(), 17, 128, 16, 32, 1, None, 0, None, None) == -4
    assert L.kata_w4_linear(w4(), 16, 127, 16, 32, 2, None, 0, None, None) == -3
    assert L.kata_w4_linear(w4(), 16, 128, 16, 31, 2, None, 0, None, None) == -3
    assert L.kata_w4_linear(w4(), 16, 128, 16, 32, -1, None, 0, None, None) == -3
    assert L.kata_w4_linear(w4(), None, 128, None, 32, 0, None, 0, None, None) == 0  # no rows: nothing to do
    # many rows off 16-byte boundaries, or fp32 ones, are laid out in a workspace
    assert L.kata_w4_workspace_bytes(w4(), 16, 128, 100) == 0 and L.kata_w4_workspace_bytes(w4(), 18, 128, 1) == 0
    assert L.kata_w4_workspace_bytes(w4(K=100), 18, 100, 100) == 100 * 104 * 2
    assert L.kata_w4_workspace_bytes(w4(dtype=0), 16, 128, 100) == 100 * 128 * 6
    assert L.kata_w4_linear(w4(), 18, 128, 16, 32, 100, None, 0, None, None) == -5
    assert L.kata_w4_linear(w4(), 18, 128, 16, 32, 100, 8, 25600, None, None) == -4
    assert L.kata_w4_pack(None, 16, None, w4(), None) == -1
    assert L.kata_w4_pack(16, 16, 16, w4(), None) == -1  # zeros without a place for them
    assert L.kata_w4_pack(16, 16, None, w4(data=20), None) == -4


def test_qkv_step_refusals(L):
    def step(B=1, x=16, ldx=128, pos=16, ring=16, q=16, k=16, v=16, **kw):
        a = _lib.QkvStepArgs(**{**dict(conv_w=16, dtype=1, HQ=2, H=1, D=32, Dv=32, K=4), **kw})
        return L.kata_qkv_step(a, x, ldx, pos, ring, q, k, v, B, None)

    assert L.kata_qkv_step(None, 16, 128, 16, 16, 16, 16, 16, 1, None) == -1
    assert step(dtype=5) == -2
    for bad in (dict(H=0), dict(HQ=3, H=2), dict(D=0), dict(D=12), dict(D=264), dict(Dv=4), dict(B=-1)):
        assert step(**bad) == -3, bad
    assert step(K=5) == -8
    for bad in (dict(norm_q=3), dict(rope=3), dict(rope=1, R=32), dict(conv_w=None), dict(x=None), dict(pos=None),
                dict(ring=None), dict(v=None)):
        assert step(**bad) == -1, bad
    assert step(rope=1, R=16, cos=16, sin=16, T=4) == -3
    assert step(rope=2, R=24, cos=16, sin=16, T=4) == -3
    for bad in (dict(x=8), dict(q=8), dict(ring=8), dict(ldx=132)):
        assert step(**bad) == -4, bad
    assert step(B=2, ldx=120) == -3
    assert step(B=0) == 0


def test_sample_refusals(L):
    def sample(**kw):
        a = dict(logits=16, u=16, token=16, logprob=16, ld=100, B=2, V=100, dtype=1, temperature_all=1.0, top_p_all=1.0)
        return L.kata_sample(_lib.SampleArgs(**{**a, **kw}), None)

    assert L.kata_sample(None, None) == -1
    assert sample(dtype=9) == -2
    for bad in (dict(V=0), dict(V=(1 << 22) + 1), dict(B=-1), dict(ld=99)):
        assert sample(**bad) == -3, bad
    for bad in (dict(logits=None), dict(u=None), dict(token=None), dict(logprob=None)):
        assert sample(**bad) == -1, bad
    assert sample(logits=17) == -4
    assert sample(B=0) == 0


def test_fronts_refuse_cpu_tensors():
    from linatt_b200.quant import W4Weight, quantize_w4
    from linatt_b200.qkv_step import QKVStep
    from linatt_b200.sampling import sample_tokens

    with pytest.raises(RuntimeError):
        W4Weight(torch.zeros(4, 4, dtype=torch.int32), torch.ones(4, 1), in_features=32, group_size=32)
    with pytest.raises(RuntimeError):
        quantize_w4(torch.zeros(4, 32))
    with pytest.raises(RuntimeError):
        QKVStep(num_heads=1, head_k_dim=8, head_v_dim=8, conv_weight=torch.zeros(24, 4))
    with pytest.raises(RuntimeError):
        sample_tokens(torch.zeros(2, 10), torch.zeros(2))


def test_qkv_step_refuses_inputs_on_another_device_than_its_weights(monkeypatch):
    """On the host, without a launch: the devices are stated, not looked up."""
    from linatt_b200 import qkv_step

    def on(i):
        monkeypatch.setattr(_lib, "require_cuda", lambda *ts: None if all(t is None for t in ts) else torch.device("cuda", i))

    class Never:
        def kata_qkv_step(self, *a):
            raise AssertionError("launched")

    monkeypatch.setattr(_lib, "lib", lambda: Never())
    on(0)
    step = qkv_step.QKVStep(num_heads=1, head_k_dim=8, head_v_dim=8, conv_weight=torch.zeros(24, 1))
    free = qkv_step.QKVStep(num_heads=1, head_k_dim=8, head_v_dim=8)
    on(1)
    with pytest.raises(RuntimeError, match="cuda:1.*cuda:0"):
        step(torch.zeros(2, 24), torch.zeros(2, dtype=torch.int64))
    monkeypatch.setattr(_lib, "on_device", lambda dev: _lib._STAY)
    monkeypatch.setattr(_lib, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(torch, "empty", lambda *s, dtype, device: torch.zeros(*s, dtype=dtype))
    with pytest.raises(AssertionError, match="launched"):  # without weights there is nothing to be elsewhere
        free(torch.zeros(2, 24), torch.zeros(2, dtype=torch.int64))


def test_generation_refuses_a_step_past_the_rotation_tables():
    from types import SimpleNamespace

    from linatt_b200.generate import KataGenerator

    gen = KataGenerator.__new__(KataGenerator)
    gen.layers, gen.positions, gen.max_positions, gen._length = [SimpleNamespace(cos=object())], torch.zeros(2), 5, 4
    gen._step = lambda token: "stepped"
    assert gen.step(torch.zeros(2)) == "stepped" and gen._length == 5
    with pytest.raises(ValueError, match="max_positions"):
        gen.step(torch.zeros(2))
    gen.layers[0].cos = None
    assert gen.step(torch.zeros(2)) == "stepped"


def test_counts_beyond_32_bits_keep_their_meaning():
    from linatt_b200.sampling import _setting

    t, _ = _setting(torch.tensor([5, -3, 2 ** 31, 2 ** 32 + 5, 2 ** 62, -2 ** 40]), "top_k", torch.int32, 6, torch.device("cpu"))
    assert t.dtype == torch.int32 and t[0] == 5
    assert (t[[1, 5]] <= 0).all() and (t[2:5] >= 2 ** 22).all()  # no more than 2^22 tokens: all of them
