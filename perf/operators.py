"""Cases that measure the generation operators of this library.

Three operators that a generated token (or a prompt) passes through, beside the recurrent-state attention step:

``w4``      linear layer with 4-bit weights: y = x W^T, W[n, k] = scale[n, k // g] (code[n, k] - zero[n, k // g]);
            optionally W holds gate and up rows and y = silu(gate) * up.
``step``    what stands between the fused q/k/v projection and the attention step: causal short
            convolution of width K on its ring of earlier inputs (updated), SiLU, the q / k norm of
            each head and the position rotation.
``sample``  the next token from the logits: temperature, top-k, top-p, min-p, one uniform number a row.

The plain forms compute in 32 bits with elementary torch operations.  ``sample`` is defined on whole
numbers: a token's mass is its weight exp((x - max) / T) in units of 2^-40, so sums have no order and
the drawn token is a function of the inputs alone."""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token through the attention output projection of the 768-wide LM: the smallest call
        dict(name="w4_o_proj_1", op="w4", rows=1, N=768, K=768, group=64, zeros=False, act="none", dtype="bf16"),
        # two sequences kept in fp32 through the LM's q/k/v projection: the fp32 form
        dict(name="w4_qkv_f32_2", op="w4", rows=2, N=2304, K=768, group=128, zeros=False, act="none", dtype="f32"),
        # one token, a large square layer streamed from HBM: single-stream generation
        dict(name="w4_wide_1", op="w4", rows=1, N=32768, K=8192, group=128, zeros=False, act="none", dtype="bf16"),
        # seven sequences, odd sizes, a last group that is not whole, zero points, small groups
        dict(name="w4_odd_7", op="w4", rows=7, N=5003, K=4100, group=32, zeros=True, act="none", dtype="f16"),
        # a batch of 64 sequences through a gated feed-forward's fused gate / up weight
        dict(name="w4_swiglu_64", op="w4", rows=64, N=16384, K=4096, group=128, zeros=False, act="swiglu", dtype="bf16"),
        # a prompt of 512 tokens through a square layer: the most arithmetic
        dict(name="w4_prompt_512", op="w4", rows=512, N=4096, K=4096, group=128, zeros=False, act="none", dtype="bf16"),
        # one token of the LM's layer: convolution only, as its configuration has it
        dict(name="step_lm_1", op="step", B=1, HQ=12, H=12, D=64, Dv=64, conv=4, norm="none", rope=0, dtype="bf16"),
        # a large serving batch with shared key heads, RMS norms and the interleaved rotation
        dict(name="step_gqa_1024", op="step", B=1024, HQ=32, H=8, D=128, Dv=128, conv=4, norm="rms", rope=1, dtype="bf16"),
        # one sequence of the LM (vocabulary 32000), the usual filters: the latency of one draw
        dict(name="sample_1", op="sample", B=1, V=32000, mode="top", masked=0.0, dtype="bf16"),
        # plain temperature sampling of a batch from fp32 logits, as roll-outs draw
        dict(name="sample_plain_64", op="sample", B=64, V=32000, mode="plain", masked=0.0, dtype="f32"),
        # constrained decoding: half the vocabulary masked with -inf, odd vocabulary, nucleus and floor
        dict(name="sample_masked_17", op="sample", B=17, V=100003, mode="nucleus", masked=0.5, dtype="f16"),
        # a large batch, every row with its own settings (greedy rows among them): the largest draw
        dict(name="sample_mixed_256", op="sample", B=256, V=131072, mode="mixed", masked=0.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("w4", "w4", "step", "sample"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "w4":
        while True:
            rows, N, K = _log(rng, 1, 512), _log(rng, 256, 32768), _log(rng, 256, 16384)
            act = rng.choice(("none", "none", "swiglu"))
            if act == "swiglu":
                N += N % 2
            if rng.random() < 0.5:
                K -= K % 128
            if N * K <= 2 ** 28 and rows * N * K <= 2 ** 33 and 3072 not in (N, K):
                break
        return dict(op=op, rows=rows, N=N, K=K, group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.4, act=act,
                    dtype=dtype)
    if op == "step":
        while True:
            B, H, G = _log(rng, 1, 1024), rng.randint(1, 16), rng.choice((1, 1, 2, 4))
            D, Dv = rng.choice((32, 64, 128)), rng.choice((32, 64, 128))
            conv, norm, rope = rng.choice((0, 2, 3, 4)), rng.choice(("none", "l2", "rms")), rng.choice((0, 1, 2))
            width = H * G * D + H * D + H * Dv
            if B * width <= 1024 * 6144 and width != 3072 and (conv or norm != "none" or rope):
                break
        return dict(op=op, B=B, HQ=H * G, H=H, D=D, Dv=Dv, conv=conv, norm=norm, rope=rope, dtype=dtype)
    while True:
        B, V = _log(rng, 1, 256), _log(rng, 1000, 160000)
        if B * V <= 256 * 131072:
            break
    return dict(op=op, B=B, V=V, mode=rng.choice(("top", "plain", "nucleus", "mixed")),
                masked=rng.choice((0.0, 0.0, 0.5, 0.99)), dtype=dtype)


# ----------------------------------------------------------------------------------- inputs

EPS = 1e-6
MAX_POS = 4096


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] == "w4":
        N, K, gs = case["N"], case["K"], case["group"]
        G, words = -(-K // gs), 4 * (-(-K // 32))
        # codes of normally distributed weights lie around the middle of the 16: sums of two uniform 3-bit numbers and a bit
        r = torch.randint(-2 ** 31, 2 ** 31, (N, words), device="cuda", generator=g)
        lo, hi = r & 0x77777777, torch.randint(-2 ** 31, 2 ** 31, (N, words), device="cuda", generator=g) & 0x77777777
        s["packed"] = (lo + hi + ((r >> 3) & 0x11111111)).to(torch.int32)
        s["scales"] = ((0.5 + rand(N, G)) * (0.3 / math.sqrt(K))).to(dt)
        s["zeros"] = torch.randint(5, 11, (N, G), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
        s["x"] = randn(case["rows"], K).to(dt)
        if own:
            from linatt_b200.quant import W4Weight

            s["w"] = W4Weight(s["packed"], s["scales"], s["zeros"], in_features=K, group_size=gs,
                              activation=None if case["act"] == "none" else case["act"])
    elif case["op"] == "step":
        B, HQ, H, D, Dv, K = (case[n] for n in ("B", "HQ", "H", "D", "Dv", "conv"))
        C = HQ * D + H * D + H * Dv
        s["qkv"] = randn(B, C).to(dt)
        s["pos"] = torch.randint(0, MAX_POS, (B,), device="cuda", generator=g)
        s["ring"] = randn(B, K - 1, C).to(dt) if K else None
        s["conv_w"] = randn(C, K) * 0.4 if K else None
        rms = case["norm"] == "rms"
        s["q_w"], s["k_w"] = (1 + 0.1 * randn(D) if rms else None), (1 + 0.1 * randn(D) if rms else None)
        R = {0: 0, 1: D, 2: D // 2}[case["rope"]]  # rotation 2 works in groups of half a head
        s["cos"] = s["sin"] = None
        if R:
            f = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
            a = torch.arange(MAX_POS, device="cuda", dtype=torch.float64)[:, None] * f
            s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        if own:
            from linatt_b200.qkv_step import QKVStep

            s["step"] = QKVStep(num_heads=HQ, num_kv_heads=H, head_k_dim=D, head_v_dim=Dv, conv_weight=s["conv_w"],
                                norm_q=case["norm"], norm_k=case["norm"], q_weight=s["q_w"], k_weight=s["k_w"],
                                eps_q=EPS, eps_k=EPS, rope=case["rope"], rope_dim=R, cos=s["cos"], sin=s["sin"])
    else:
        B, V, mode = case["B"], case["V"], case["mode"]
        # logits as a language model gives them: a normal bulk, and a few tens of likely tokens above it
        x = randn(B, V) * 2.0
        x.scatter_add_(1, torch.randint(0, V, (B, 40), device="cuda", generator=g), 4 + 4 * rand(B, 40))
        if case["masked"]:
            x.masked_fill_(rand(B, V) < case["masked"], -math.inf)
        s["logits"], s["u"] = x.to(dt), rand(B)
        pick = lambda v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (B,), device="cuda", generator=g)]  # noqa: E731
        s["par"] = {
            "top": dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.0),
            "plain": dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
            "nucleus": dict(temperature=1.1, top_k=0, top_p=0.9, min_p=0.001),
            "mixed": dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.4]), top_k=pick([0, 0, 1, 40, 1000]).int(),
                          top_p=pick([1.0, 0.5, 0.9, 0.99]), min_p=pick([0.0, 0.0, 0.02])),
        }[mode]
    return s


# --------------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        if op == "w4":
            from linatt_b200.quant import w4_linear

            return w4_linear(s["x"], s["w"])
        if op == "step":
            q, k, v = s["step"](s["qkv"], s["pos"], s["ring"])
            return {"q": q, "k": k, "v": v, "ring": s["ring"]}
        from linatt_b200.sampling import sample_tokens

        token, logprob = sample_tokens(s["logits"], s["u"], **s["par"])
        return {"token": token, "logprob": logprob}
    return {"w4": _plain_w4, "step": _plain_step, "sample": _plain_sample}[op](s)


def _plain_w4(s):
    case, x = s["case"], s["x"]
    K, gs = case["K"], case["group"]
    codes = ((s["packed"][:, :, None] >> torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)) & 15).flatten(1)[:, :K]
    of = torch.arange(K, device=x.device) // gs
    zero = s["zeros"].float()[:, of] if s["zeros"] is not None else 8.0
    y = x.float() @ ((codes.float() - zero) * s["scales"].float()[:, of]).T
    if case["act"] == "swiglu":
        a, b = y.chunk(2, dim=1)
        y = a / (1 + torch.exp(-a)) * b
    return y.to(x.dtype)


def _plain_norm_rope(s, x, w):
    case = s["case"]
    if case["norm"] == "l2":
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)
    elif case["norm"] == "rms":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if not case["rope"]:
        return x
    c, n = s["cos"][s["pos"]][:, None, None], s["sin"][s["pos"]][:, None, None]
    if case["rope"] == 1:  # neighbours are pairs
        p = x.unflatten(-1, (1, -1, 2))
        a, b = p[..., 0], p[..., 1]
        return torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-3)
    a, b = x.unflatten(-1, (-1, 2, 2 * c.shape[-1] // 2)).unbind(-2)  # the halves of each group are pairs
    return torch.stack((a * c - b * n, a * n + b * c), -2).flatten(-3)


def _plain_step(s):
    case, x = s["case"], s["qkv"].float()
    B, HQ, H, D, Dv, K = (case[n] for n in ("B", "HQ", "H", "D", "Dv", "conv"))
    if K:
        # position p's input is kept in slot p % (K - 1) of the ring; slot j positions back holds input p - j
        back = torch.arange(K - 1, 0, -1, device=x.device)
        at = (s["pos"][:, None] - back) % (K - 1)
        old = torch.gather(s["ring"], 1, at[:, :, None].expand(-1, -1, x.shape[1]))
        a = (torch.cat((old.float(), x[:, None]), 1) * s["conv_w"].T).sum(1)
        s["ring"].scatter_(1, (s["pos"] % (K - 1))[:, None, None].expand(-1, 1, x.shape[1]), s["qkv"][:, None])
        x = a / (1 + torch.exp(-a))
    q, k, v = x.split((HQ * D, H * D, H * Dv), 1)
    q, k = _plain_norm_rope(s, q.view(B, HQ, D), s["q_w"]), _plain_norm_rope(s, k.view(B, H, D), s["k_w"])
    dt = s["qkv"].dtype
    return {"q": q.to(dt), "k": k.to(dt), "v": v.reshape(B, H, Dv).to(dt), "ring": s["ring"]}


def _parameter(v, like, dtype):
    return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((like.shape[0], 1), v, dtype=dtype, device=like.device)


def _share(total, n24):
    """total * n24 / 2^24 as (quotient, whether something is left), without leaving 64 bits."""
    high, low = total >> 32, total & 0xFFFFFFFF
    rest = low * n24
    return ((high * n24) << 8) + (rest >> 24), (rest & 0xFFFFFF) != 0


def _plain_sample(s):
    x, u = s["logits"].float(), s["u"]
    B, V = x.shape
    T, p, m = (_parameter(s["par"][n], x, torch.float32) for n in ("temperature", "top_p", "min_p"))
    k = _parameter(s["par"]["top_k"], x, torch.int64)
    x = torch.where(torch.isnan(x), -math.inf, x)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest index first
    top = x[:, :1]
    z = torch.where(x == top, 0.0, (x - top) * (1.0 / T))
    w = torch.where(x == -math.inf, 0.0, torch.exp(z))
    mass = torch.round(w.double() * 2.0 ** 40).long()
    rank = torch.arange(V, device=x.device)
    keep = (rank < k) | (k <= 0)
    before = torch.cumsum(mass, 1) - mass
    limit, more = _share((mass * keep).sum(1, keepdim=True), (p.clamp(0, 1) * 2.0 ** 24).long())
    keep &= (before < limit + more) | (p >= 1)
    keep &= (w >= m)
    keep |= rank == 0
    keep &= (T > 0) | (rank == 0)  # temperature zero: the likeliest token
    z, kept = torch.where(T > 0, z, 0.0), mass * keep
    kept = torch.where(T > 0, kept, (rank == 0).long() << 40)
    total = kept.sum(1, keepdim=True)
    ordered = torch.zeros_like(kept).scatter_(1, order, kept)
    target, _ = _share(total, (u[:, None].clamp(0, 1) * 2.0 ** 24).long().clamp(max=2 ** 24 - 1))
    token = (torch.cumsum(ordered, 1) <= target).sum(1, keepdim=True).clamp(max=V - 1)
    z = torch.zeros_like(z).scatter_(1, order, z).gather(1, token)
    logprob = z - torch.log(total.double() * 2.0 ** -40).float()
    empty = top == -math.inf
    return {"token": torch.where(empty, -1, token)[:, 0], "logprob": torch.where(empty, -math.inf, logprob)[:, 0]}


# ------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"w4": _exact_w4, "step": _exact_step, "sample": _exact_sample}[case["op"]](s, case)


def _exact_w4(s, case):
    N, K, gs = case["N"], case["K"], case["group"]
    x = s["x"].double()
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    words = s["packed"].long() & 0xFFFFFFFF
    for first in range(0, K, gs):  # one group of the weights at a time
        n = min(gs, K - first)
        k = torch.arange(first, first + n, device=x.device)
        code = torch.bitwise_right_shift(words[:, k // 8], 4 * (k % 8)).remainder(16).double()
        zero = 8.0 if s["zeros"] is None else s["zeros"][:, first // gs, None].double()
        y += (x[:, first:first + n] @ (code - zero).T) * s["scales"][:, first // gs].double()
    if case["act"] == "swiglu":
        y = y[:, : N // 2] * torch.sigmoid(y[:, : N // 2]) * y[:, N // 2:]
    return y


def _exact_step(s, case):
    B, HQ, H, D, Dv, K = (case[n] for n in ("B", "HQ", "H", "D", "Dv", "conv"))
    x, pos = s["qkv"].double(), s["pos"]
    rows = torch.arange(B, device=x.device)
    ring = None
    if K:
        ring = s["ring"].double()
        a = x * s["conv_w"][:, K - 1].double()
        for j in range(1, K):  # the input j positions earlier has weight K - 1 - j
            a = a + ring[rows, (pos - j) % (K - 1)] * s["conv_w"][:, K - 1 - j].double()
        ring[rows, pos % (K - 1)] = x
        x = a * torch.sigmoid(a)
    out, at = {}, 0
    for name, heads, dim, w in (("q", HQ, D, s["q_w"]), ("k", H, D, s["k_w"]), ("v", H, Dv, None)):
        y = x[:, at:at + heads * dim].reshape(B, heads, dim)
        at += heads * dim
        if name != "v":
            if case["norm"] != "none":
                n = dim if case["norm"] == "rms" else 1
                y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / n + EPS) * (1 if w is None else w.double())
            if case["rope"]:
                R = 2 * s["cos"].shape[1]
                turn = torch.complex(s["cos"].double(), s["sin"].double())[pos]
                t = torch.empty_like(y)
                for first in range(0, dim, R):
                    i = torch.arange(R // 2, device=x.device)
                    a, b = (first + 2 * i, first + 2 * i + 1) if case["rope"] == 1 else (first + i, first + R // 2 + i)
                    r = torch.complex(y[..., a], y[..., b]) * turn[:, None]
                    t[..., a], t[..., b] = r.real, r.imag
                y = t
        out[name] = y
    out["ring"] = ring
    return out


def _exact_sample(s, case):
    B, V = case["B"], case["V"]
    logits, u = s["logits"].double().cpu(), s["u"].double().cpu()
    par = {n: (v.cpu().tolist() if isinstance(v, torch.Tensor) else [v] * B) for n, v in s["par"].items()}
    logprob = torch.zeros(B, dtype=torch.float64)
    for b in range(B):  # one row at a time
        T, k, p, m = par["temperature"][b], par["top_k"][b], par["top_p"][b], par["min_p"][b]
        x, order = torch.sort(logits[b], descending=True, stable=True)
        if T <= 0 or x[0] == -math.inf:
            logprob[b] = 0.0 if x[0] > -math.inf else -math.inf
            continue
        w = torch.exp((x - x[0]) / T)
        n = V if k <= 0 else min(k, V)
        if p < 1:
            c = torch.cumsum(w[:n], 0)
            n = max(1, int((c - w[:n] < p * c[-1]).sum()))
        n = min(n, max(1, int((w >= m).sum())))
        by_index, of = torch.sort(order[:n])
        w = w[:n][of]
        c = torch.cumsum(w, 0)
        i = min(int((c <= float(u[b]) * float(c[-1])).sum()), n - 1)
        logprob[b] = torch.log(w[i] / c[-1])
    return {"token": None, "logprob": logprob.to(s["u"].device)}


# ------------------------------------------------------------------------- what a pass needs

def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "w4":
        rows, N, K = case["rows"], case["N"], case["K"]
        G = -(-K // case["group"])
        out = rows * (N // 2 if case["act"] == "swiglu" else N)
        return {"bytes": N * K / 2 + N * G * (e + (1 if case["zeros"] else 0)) + (rows * K + out) * e,
                "flops": 2.0 * rows * N * K}
    if case["op"] == "step":
        B, HQ, H, D, Dv, K = (case[n] for n in ("B", "HQ", "H", "D", "Dv", "conv"))
        C = HQ * D + H * D + H * Dv
        # the row, the K - 1 earlier inputs, one input written to the ring, q, k and v; the convolution's weights
        return {"bytes": B * C * e * (2 + K) + 4 * C * K if K else 2 * B * C * e, "flops": float(B * C * (2 * K + 10))}
    return {"bytes": case["B"] * case["V"] * e + 16 * case["B"], "flops": 4.0 * case["B"] * case["V"]}
