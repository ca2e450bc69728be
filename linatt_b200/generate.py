"""Generation with a :class:`linatt_b200.lm.KataLM` on 4-bit weights and recurrent states.

The reference's flash layer keeps no cache (kata/layer.py:421-492 sets ``final_state = None``), so its
models re-run attention over the whole prefix for every token.  Here a layer carries the state of the
attention (:mod:`linatt_b200.kata_decode`) and the ring of its short convolution, and a token passes,
per layer, one launch each of

    q/k/v projection (4 bits) -> convolution, norms, rotation (:class:`QKVStep`) -> kata_decode_step
    -> output norm -> output projection (4 bits) -> residual + norm -> gate / up / SwiGLU (4 bits, one
    product) -> down projection (4 bits) -> residual + norm

and then the head and :func:`sample_tokens`.  A prompt runs the same weights through the kernels of
whole sequences.  After the first token the step is captured in a CUDA graph, since its launches are
what bounds it.  Inference only; there is no CPU path.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _lib
from .kata_decode import kata_attn_decode, kata_attn_state
from .lm import KataLM, add_rmsnorm
from .mixer import FlashKataMixer, RowNormFunction, ShortConvQKVFunction, rope_tables
from .parallel_kata_attn import parallel_kata_attn, parallel_kata_attn_decay, parallel_kata_attn_sum
from .qkv_step import QKVStep
from .quant import quantize_w4, w4_linear
from .sampling import sample_tokens

__all__ = ["KataGenerator"]


class _Layer:
    """A block's 4-bit weights and its step; the state and ring of the sequences it is generating."""

    def __init__(self, blk, dtype, group_size, symmetric, positions):
        m: FlashKataMixer = blk.attn
        if m.use_offset_gate:
            raise ValueError("generation does not support use_offset_gate")
        q4 = lambda w, act=None: quantize_w4(w.detach(), group_size, symmetric=symmetric, dtype=dtype, activation=act)  # noqa: E731
        self.blk, self.mixer, self.dtype = blk, m, dtype
        self.qkv = q4(torch.cat([m.q_proj.weight, m.k_proj.weight, m.v_proj.weight]))
        self.o_proj = q4(m.o_proj.weight)
        self.gate_up = q4(torch.cat([blk.mlp.gate_proj.weight, blk.mlp.up_proj.weight]), "swiglu")
        self.down = q4(blk.mlp.down_proj.weight)
        self.conv = [m.q_conv1d.weight, m.k_conv1d.weight, m.v_conv1d.weight] if m.use_short_conv else None
        rope = 0 if not m.use_rope else 2 if m.rope_group else 1
        R = 0 if not rope else m.head_k_dim // m.spd_num_groups if rope == 2 else m.head_k_dim
        self.cos, self.sin = rope_tables(positions, R, m.rope_theta, m.q_proj.weight.device, dtype) if rope else (None, None)
        norm = lambda kind: {False: None, "l2": "l2", "rmsnorm": "rms"}[kind if m.qk_norm else False]  # noqa: E731
        qn, kn = getattr(m, "q_norm", None), getattr(m, "k_norm", None)
        self.step = QKVStep(num_heads=m.num_heads, num_kv_heads=m.num_kv_heads, head_k_dim=m.head_k_dim,
                            head_v_dim=m.head_v_dim, conv_weight=None if self.conv is None else torch.cat(self.conv),
                            norm_q=norm(m.norm_q), norm_k=norm(m.norm_k), q_weight=None if qn is None else qn.weight,
                            k_weight=None if kn is None else kn.weight, eps_q=1e-6 if qn is None else qn.eps,
                            eps_k=1e-6 if kn is None else kn.eps, rope=rope, rope_dim=R, cos=self.cos, sin=self.sin)
        self.score = "sum" if m.feature_map_name == "kata_quadratic_sum" else "concat"
        self.state = self.ring = None

    def _log_decay(self, y):
        m = self.mixer
        if not m.use_decay:
            return None
        dt = F.softplus(F.linear(y.float(), m.dt_proj.weight.float()) + m.dt_bias)
        return -m.A_log.float().exp() * dt

    def _output(self, o):
        m = self.mixer
        Dv = m.head_v_dim
        if m.output_norm == "rmsnorm":
            o = RowNormFunction.apply(o.reshape(-1, Dv), m.norm.weight, None, None, 2, 0, Dv, m.norm.eps, m.num_heads, 1)
        return o.to(self.dtype)

    def prompt(self, y):
        """The mixer's output for y (B, T, hidden), the first T tokens; sets the state and the ring."""
        m = self.mixer
        B, T, _ = y.shape
        x = w4_linear(y, self.qkv)
        self.ring = self.step.ring_of(x)
        if self.conv is not None:
            q, k, v = ShortConvQKVFunction.apply(x, True, *self.conv)
        else:
            q, k, v = x.split([m.key_dim, m.key_dim_per_group, m.value_dim_per_group], -1)
        q = q.reshape(B, T, m.num_heads, m.head_k_dim)
        k = k.reshape(B, T, m.num_kv_heads, m.head_k_dim)
        v = v.reshape(B, T, m.num_kv_heads, m.head_v_dim).contiguous()
        q = m._qk_prologue(q, m.norm_q, getattr(m, "q_norm", None), T, self.cos, self.sin)
        k = m._qk_prologue(k, m.norm_k, getattr(m, "k_norm", None), T, self.cos, self.sin)
        M, g = m.spd_num_groups, self._log_decay(y)
        if g is not None:
            c = g.cumsum(1).contiguous()
            o = parallel_kata_attn_decay(q, k, v, c, num_groups=M)
            self.state = kata_attn_state(k, v, num_groups=M, c=c)
        else:
            o = (parallel_kata_attn_sum if self.score == "sum" else parallel_kata_attn)(q, k, v, num_groups=M)
            self.state = kata_attn_state(k, v, num_groups=M, score=self.score)
        return w4_linear(self._output(o).view(B, T, -1), self.o_proj)

    def token(self, y, pos):
        """The mixer's output for y (B, hidden), the tokens at `pos`; the state and the ring advance in place."""
        q, k, v = self.step(w4_linear(y, self.qkv), pos, self.ring)
        o = kata_attn_decode(q, k, v, self.state, num_groups=self.mixer.spd_num_groups, score=self.score,
                             g=self._log_decay(y))
        return w4_linear(self._output(o).view(y.shape[0], -1), self.o_proj)


class KataGenerator:
    """Generates with a KataLM whose projections are rounded to 4 bits (``group_size``, ``symmetric`` as
    :func:`quantize_w4`; ``quantize_head`` rounds the output head too).  Activations are ``dtype``, the residual
    stream fp32.  ``max_positions`` bounds prompt and new tokens together where the model rotates q and k."""

    def __init__(self, lm: KataLM, *, dtype: torch.dtype = torch.bfloat16, group_size: int = 64, symmetric: bool = True,
                 quantize_head: bool = False, max_positions: int | None = None):
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"activations are bf16 or f16, got {dtype}")
        _lib.require_cuda(lm.lm_head.weight)
        self.lm, self.dtype = lm, dtype
        self.max_positions = max(max_positions or 0, lm.config.max_position_embeddings)
        self.layers = [_Layer(b, dtype, group_size, symmetric, self.max_positions) for b in lm.model.layers]
        head = lm.lm_head.weight.detach()
        self.head = quantize_w4(head, group_size, symmetric=symmetric, dtype=dtype) if quantize_head else head.to(dtype)
        self.positions = None

    def _logits(self, y):
        y = y.to(self.dtype)
        return F.linear(y, self.head) if isinstance(self.head, torch.Tensor) else w4_linear(y, self.head)

    def _blocks(self, h, mix):
        """h (fp32) through the layers, `mix` being a layer's mixer for normalised hidden states."""
        layers = self.lm.model.layers
        y = layers[0].attn_norm(h).to(self.dtype)
        for i, (blk, lay) in enumerate(zip(layers, self.layers)):
            h, y = add_rmsnorm(h, mix(lay, y), blk.mlp_norm)
            nxt = layers[i + 1].attn_norm if i + 1 < len(layers) else self.lm.model.norm
            h, y = add_rmsnorm(h, w4_linear(w4_linear(y.to(self.dtype), lay.gate_up), lay.down), nxt)
            y = y.to(self.dtype)
        return y

    @torch.no_grad()
    def prefill(self, input_ids: torch.Tensor) -> torch.Tensor:
        """Logits (B, vocab) after the prompts input_ids (B, T), T >= 1; the sequences' states are set."""
        _lib.require_cuda(input_ids)
        if input_ids.dim() != 2 or input_ids.shape[1] < 1:
            raise ValueError(f"input_ids must be (B, T) with T >= 1, got {tuple(input_ids.shape)}")
        if self.layers[0].cos is not None and input_ids.shape[1] > self.max_positions:
            raise ValueError(f"the prompt has {input_ids.shape[1]} tokens, more than max_positions={self.max_positions}")
        B, T = input_ids.shape
        y = self._blocks(self.lm.model.embeddings(input_ids).float(), lambda lay, y: lay.prompt(y))
        self.positions = torch.full((B,), T, dtype=torch.int64, device=input_ids.device)
        self._length = T
        return self._logits(y[:, -1])

    @torch.no_grad()
    def step(self, token: torch.Tensor) -> torch.Tensor:
        """Logits (B, vocab) after one more token (B,) of each sequence."""
        if self.positions is None or token.shape != self.positions.shape:
            raise ValueError("step() follows prefill() of as many sequences")
        if self.layers[0].cos is not None and self._length >= self.max_positions:
            raise ValueError(f"the sequences have max_positions={self.max_positions} tokens: none more can be rotated")
        logits = self._step(token)
        self._length += 1
        return logits

    def _step(self, token):
        h = self.lm.model.embeddings(token.clamp(min=0)).float()
        y = self._blocks(h, lambda lay, y: lay.token(y, self.positions))
        self.positions.add_(1)
        return self._logits(y)

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, *, u: torch.Tensor | None = None,
                 generator: torch.Generator | None = None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 use_graph: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
        """(tokens, logprobs), each (B, max_new_tokens), after the prompts input_ids (B, T).  ``u``
        (max_new_tokens, B) fp32: the uniform numbers of the draws (default: from ``generator``); the other
        settings as :func:`sample_tokens`.  The prompts are of one length, and every sequence gets all new tokens (no
        token ends one).  From four new tokens on, every call captures its step anew."""
        B, T = input_ids.shape
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        if self.layers[0].cos is not None and T + max_new_tokens > self.max_positions:
            raise ValueError(f"{T} + {max_new_tokens} tokens are more than max_positions={self.max_positions}")
        dev = input_ids.device
        if u is None:
            u = torch.rand(max_new_tokens, B, device=dev, generator=generator)
        if u.shape != (max_new_tokens, B) or u.dtype != torch.float32:
            raise ValueError(f"u must be ({max_new_tokens}, {B}) fp32, got {tuple(u.shape)} {u.dtype}")
        par = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        tokens = torch.empty(B, max_new_tokens, dtype=torch.int64, device=dev)
        logprobs = torch.empty(B, max_new_tokens, device=dev)
        token, lp = sample_tokens(self.prefill(input_ids), u[0], **par)
        tokens[:, 0], logprobs[:, 0] = token, lp
        number = torch.empty_like(u[0])
        # the loop runs on a stream of its own: the first step there sets up what a capture must not allocate
        st, graph = torch.cuda.Stream(dev), None
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            for i in range(1, max_new_tokens):
                number.copy_(u[i])
                if graph is not None:
                    graph.replay()
                elif use_graph and i == 2 and max_new_tokens > 3:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=st):
                        t, l = sample_tokens(self._step(token), number, **par)
                        token.copy_(t)
                        lp.copy_(l)
                    graph.replay()
                else:
                    t, l = sample_tokens(self._step(token), number, **par)
                    token.copy_(t)
                    lp.copy_(l)
                self._length += 1
                tokens[:, i], logprobs[:, i] = token, lp
        torch.cuda.current_stream(dev).wait_stream(st)
        if graph is not None:
            st.synchronize()  # the graph and what it holds go with this call
        return tokens, logprobs
