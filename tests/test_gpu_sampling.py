"""GPU parity of token sampling: the token exactly, against the definition on whole numbers; the log
probability against float64 (fp32 output: 2^-24 of its value, and what the fp32 exponent z = (x - m) / T
and the masses' units lose: a few 2^-24 of |z| and V 2^-41 of the total)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Row by row in Python's whole numbers; weights in fp32 by torch, as the definition has them."""
    tokens, logprobs = [], []
    for b in range(logits.shape[0]):
        get = lambda v: v[b].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
        f32 = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
        x = logits[b].float()
        x = torch.where(torch.isnan(x), -math.inf, x)
        T, k, p, mp = f32(get(temperature)), int(get(top_k)), f32(get(top_p)), f32(get(min_p))
        m = x.max()
        if m == -math.inf:
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        xs, order = torch.sort(x, descending=True, stable=True)
        if T <= 0:
            tokens.append(order[0].item())
            logprobs.append(0.0)
            continue
        inv = 1.0 / T
        w = torch.where(xs == m, 1.0, torch.where((xs == -math.inf) | (m == math.inf), 0.0, torch.exp((xs - m) * inv)))
        mass = [int(v) for v in torch.round(w.double() * 2.0 ** 40).tolist()]
        order, w = order.tolist(), w.tolist()
        n = len(order) if k <= 0 else min(k, len(order))
        if p < 1:
            limit, before, keep = max(0, int(p.item() * 2 ** 24)) * sum(mass[:n]), 0, 0
            while keep < n and before * 2 ** 24 < limit:
                before += mass[keep]
                keep += 1
            n = max(keep, 1)
        n = max(1, min(n, sum(1 for v in w if v >= mp.item())))
        kept = sorted(zip(order[:n], mass[:n]))
        total = sum(q for _, q in kept)
        target, run = (min(2 ** 24 - 1, int(u[b].item() * 2 ** 24)) * total) >> 24, 0
        for i, q in kept:
            run += q
            if run > target:
                tokens.append(i)
                x64 = x.double()
                z = ((x64 - m.double()) / T.double())
                logprobs.append((z[i] if x[i] != m else torch.tensor(0.0)).item() - math.log(total / 2.0 ** 40))
                break
    return tokens, logprobs


def check(logits, u, **par):
    from linatt_b200.sampling import sample_tokens

    token, logprob = sample_tokens(logits, u, **par)
    want, lp = reference(logits, u, **par)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32
    assert token.tolist() == want
    for got, ref in zip(logprob.tolist(), lp):
        if math.isinf(ref):
            assert got == ref
        else:
            assert abs(got - ref) <= 8 * 2.0 ** -24 * (abs(ref) + 30) + logits.shape[1] * 2.0 ** -41
    again, lp2 = sample_tokens(logits, u, **par)
    assert torch.equal(again, token) and torch.equal(lp2, logprob)
    return token


def draw(B, V, dtype, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, V, device="cuda", generator=g) * scale).to(dtype), torch.rand(B, device="cuda", generator=g)


SETTINGS = [
    dict(),
    dict(temperature=0.0),
    dict(temperature=0.7, top_k=50),
    dict(temperature=0.8, top_k=50, top_p=0.95),
    dict(top_p=0.9),
    dict(temperature=1.5, top_p=0.999),
    dict(min_p=0.05),
    dict(temperature=1.2, top_k=700, top_p=0.7, min_p=0.01),
    dict(top_k=1),
    dict(top_k=10 ** 9, top_p=1.0),
    dict(top_p=1e-9),
    dict(top_p=0.0),
    dict(min_p=2.0),
    dict(min_p=1.0),
    dict(temperature=1e-6),
    dict(temperature=100.0, top_p=0.5),
    dict(temperature=math.inf, top_k=3000),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("par", SETTINGS)
def test_sampling_settings(par, dtype):
    logits, u = draw(5, 4999, dtype, seed=11)
    check(logits, u, **par)


@pytest.mark.parametrize("V", [1, 2, 31, 33, 255, 1000, 8191, 32000, 100003, 151937])
def test_sampling_vocabularies(V):
    logits, u = draw(3, V, torch.bfloat16, seed=V)
    check(logits, u, temperature=0.9, top_p=0.92)
    check(logits, u, temperature=0.9, top_k=40, top_p=0.92)
    check(logits.float(), u)


def test_sampling_rows_have_their_own_settings():
    B, V = 24, 6000
    logits, u = draw(B, V, torch.float32, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    pick = lambda v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (B,), device="cuda", generator=g)]  # noqa: E731
    check(logits, u, temperature=pick([0.0, 0.5, 1.0, 1.7]), top_k=pick([0, 1, 5, 300, 5000]),
          top_p=pick([1.0, 0.3, 0.9]), min_p=pick([0.0, 0.02]))


@pytest.mark.parametrize("par", [dict(), dict(top_k=1777), dict(top_p=0.4), dict(top_k=3000, top_p=0.77),
                                 dict(temperature=0.0), dict(top_k=4000, min_p=0.5)])
def test_sampling_equal_logits_go_by_index(par):
    """Thousands of equal logits: a cut inside them is a cut by index."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.99999994], device="cuda")
    flat = torch.full((4, 5000), 1.5, device="cuda", dtype=torch.bfloat16)
    t = check(flat, u, **par)
    assert t[0] == 0
    two = flat.clone()
    two[:, ::2] = 1.25
    check(two, u, **par)
    few = torch.randn(4, 40000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).round().half()
    check(few, u, **par)
    signed = torch.zeros(4, 5000, device="cuda")
    signed[:, ::3] = -0.0  # equal to 0
    check(signed, u, **par)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [4194295, 4194296, 4194301, 4194304])
@pytest.mark.parametrize("skew,step", [(0, 1), (3, 1), (0, 1500), (1, 2)])
def test_sampling_equal_logits_at_the_largest_vocabularies(V, dtype, skew, step):
    """A nucleus cut among millions of equal logits, or thousands that are the same number of places apart: the
    first n of them are kept, n the least with n / count >= p, and u picks one of these."""
    from linatt_b200.sampling import sample_tokens

    u = torch.tensor([0.0, 0.37, 0.99999994], device="cuda")
    buf = torch.full((3, V + skew), -40.0, device="cuda", dtype=dtype)
    x = buf[:, skew:]
    x[:, ::step] = 1.5
    count = -(-V // step)
    for top_p in (0.0001, 0.5, 0.9):
        p24 = int(torch.tensor(top_p, dtype=torch.float32).item() * 2 ** 24)
        n = -(-p24 * count // 2 ** 24)
        token, logprob = sample_tokens(x, u, top_p=top_p)
        assert token.tolist() == [(int(v * 2 ** 24) * n >> 24) * step for v in u.tolist()]
        assert (logprob.double() + math.log(n)).abs().max() <= 2.0 ** -23 * math.log(count)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9, 1001, 40003])
def test_sampling_equal_logits_in_rows_off_16_bytes(V, dtype):
    """Rows that start between 16-byte boundaries: their first and last logits tie with others."""
    u = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.99999994], device="cuda")
    x = torch.full((5, V), 2.0, device="cuda", dtype=dtype)
    for par in (dict(temperature=0.0), dict(top_k=1), dict(top_k=3), dict(top_p=0.5), dict(top_k=V - 2, top_p=0.9)):
        check(x, u, **par)
        y = x.clone()
        y[:, 1:-1] = 1.0  # only the ends
        check(y, u, **par)


def test_sampling_close_logits_share_a_histogram_bin():
    """fp32 logits that differ in their last bits only: the cut is found by their bits."""
    base = torch.tensor(5.0).view(torch.int32).item()
    g = torch.Generator(device="cuda").manual_seed(2)
    bits = base + torch.randint(0, 100, (3, 30000), device="cuda", generator=g, dtype=torch.int32)
    logits = bits.view(torch.float32)
    u = torch.rand(3, device="cuda", generator=g)
    for par in (dict(top_k=9999), dict(top_p=0.6), dict(top_k=20000, top_p=0.3)):
        check(logits, u, **par)
    far = logits - 1e5  # all but one logit far below the first, in the last bin
    far[:, 17] = 3.0
    for par in (dict(top_k=9999), dict(top_p=0.6), dict(top_k=20000, top_p=0.3)):
        check(far, u, **par)


def test_sampling_masks_and_special_values():
    logits, u = draw(8, 3000, torch.float32, seed=9)
    inf, low = math.inf, torch.finfo(torch.float32).min
    logits[0] = -inf
    logits[1], logits[1, 77] = -inf, -3.0
    logits[2, 5:2000] = -inf
    logits[3, ::7] = math.nan
    logits[4, 100], logits[4, 2000] = inf, inf
    logits[5], logits[5, 1000] = math.nan, 2.0
    logits[6] = low
    logits[7, 3:] = low
    for par in SETTINGS + [dict(temperature=math.inf), dict(top_k=2500), dict(top_k=2990, top_p=0.99)]:
        t = check(logits, u, **par)
        assert t[0] == -1 and t[1] == 77 and t[5] == 1000 and t[4] in (100, 2000)
        assert not torch.isnan(logits[3, t[3]]) and not 5 <= t[2] < 2000
    check(logits.bfloat16(), u, top_k=100, top_p=0.9)


def test_sampling_numbers_at_the_ends():
    logits, _ = draw(6, 2000, torch.bfloat16, seed=12)
    u = torch.tensor([0.0, 1.0, 1.0 - 2.0 ** -24, 2.0 ** -30, -1.0, 0.5], device="cuda")
    want_u = u.clamp(0, 1)
    from linatt_b200.sampling import sample_tokens

    for par in (dict(), dict(top_k=3), dict(top_p=0.5)):
        assert sample_tokens(logits, u, **par)[0].tolist() == reference(logits, want_u, **par)[0]


@pytest.mark.parametrize("V", [3000, 40003])
def test_sampling_settings_that_are_nan_count_as_zero(V):
    from linatt_b200.sampling import sample_tokens

    logits, u = draw(5, V, torch.float32, seed=V)
    logits[4] = logits[4].round()  # thousands of equal logits
    u[1] = math.nan
    nan, zero = torch.full((5,), math.nan, device="cuda"), torch.zeros(5, device="cuda")
    for par in (dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=2500, top_p=0.9), dict(temperature=0.0)):
        for name in ("temperature", "top_p", "min_p"):
            got = sample_tokens(logits, u, **{**par, name: nan})
            want = sample_tokens(logits, torch.nan_to_num(u, 0.0), **{**par, name: zero})
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (par, name)


def test_sampling_does_not_depend_on_the_batch_or_the_layout():
    from linatt_b200.sampling import sample_tokens

    logits, u = draw(40, 12345, torch.bfloat16, seed=21)
    par = dict(temperature=0.9, top_k=200, top_p=0.9, min_p=0.001)
    token, lp = sample_tokens(logits, u, **par)
    for b in (0, 13, 39):
        t, l = sample_tokens(logits[b:b + 1], u[b:b + 1], **par)
        assert t[0] == token[b] and l[0] == lp[b]
    wide = torch.zeros(40, 12349, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:12348] = logits
    t, l = sample_tokens(wide[:, 3:12348], u, **par)
    assert torch.equal(t, token) and torch.equal(l, lp)
    t, l = sample_tokens(logits.T.contiguous().T, u, **par)
    assert torch.equal(t, token) and torch.equal(l, lp)
    assert sample_tokens(logits[:0], u[:0])[0].shape == (0,)


def test_sampling_follows_the_distribution():
    """A grid of 4096 numbers draws each token as often as its probability says, to within one."""
    from linatt_b200.sampling import sample_tokens

    x = torch.randn(1, 50, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    n = 4096
    u = (torch.arange(n, device="cuda", dtype=torch.float32) + 0.5) / n
    t, _ = sample_tokens(x.expand(n, 50), u, temperature=0.8)
    got = torch.bincount(t, minlength=50).double()
    want = torch.softmax(x[0].double() / 0.8, 0) * n
    assert ((got - want).abs() <= 1.001).all()


def test_sampling_on_another_stream_and_in_a_graph():
    from linatt_b200.sampling import sample_tokens

    logits, u = draw(4, 32000, torch.bfloat16, seed=2)
    want = sample_tokens(logits, u, top_k=50)[0]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        t = sample_tokens(logits, u, top_k=50)[0]
    st.synchronize()
    assert torch.equal(t, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tg = sample_tokens(logits, u, top_k=50)[0]
    logits.copy_(logits.flip(0))
    graph.replay()
    assert tg.tolist() == reference(logits, u, top_k=50)[0]


def test_sampling_refusals():
    from linatt_b200.sampling import sample_tokens

    logits, u = draw(4, 100, torch.float32, seed=1)
    with pytest.raises(RuntimeError):
        sample_tokens(logits.cpu(), u.cpu())
    with pytest.raises(ValueError):
        sample_tokens(logits[0], u)
    with pytest.raises(TypeError):
        sample_tokens(logits.double(), u)
    with pytest.raises(ValueError):
        sample_tokens(logits, u[:3])
    with pytest.raises(ValueError):
        sample_tokens(logits, u.double())
    with pytest.raises(ValueError):
        sample_tokens(logits, u, top_k=torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError):
        sample_tokens(logits, u, top_p=torch.ones(4))
    with pytest.raises(ValueError):
        sample_tokens(logits[:, :0], u)
