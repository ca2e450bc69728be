"""One token per sequence between the fused q/k/v projection and the recurrent attention step.

For whole sequences :class:`linatt_b200.mixer.FlashKataMixer` runs the causal short convolution
(+ SiLU), the q / k norm of each head and the rotation as separate passes (kata/layer.py:296-372).  A
generated token has one row per sequence, and what bounds it is the number of passes: here all three
are one kernel (``kata_qkv_step``), with values in fp32 in between.

The convolution's K - 1 earlier inputs are a ring: input p of a sequence lies in slot p % (K - 1), so a
step overwrites one slot and moves nothing.  The reference's layer keeps no cache (kata/layer.py:421-492).
Inference only.  There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["QKVStep"]

_NORM = {None: 0, "none": 0, "l2": 1, "rms": 2, "rmsnorm": 2}


class QKVStep:
    """The settings and weights of a layer's step; call it with a row per sequence.

    ``conv_weight``: (C, K) or nn.Conv1d's (C, 1, K), C = (num_heads + num_kv_heads) head_k_dim +
    num_kv_heads head_v_dim, K <= 4, or None (no convolution, no SiLU).  ``norm_q`` / ``norm_k``: None,
    "l2" or "rms" with an optional (head_k_dim,) weight.  ``rope``: 0 none, 1 interleaved pairs over the head, 2 halves of
    groups of ``rope_dim``; ``cos`` / ``sin``: (positions, rope_dim / 2).  Weights and tables are kept as fp32."""

    def __init__(self, *, num_heads: int, num_kv_heads: int | None = None, head_k_dim: int, head_v_dim: int,
                 conv_weight: torch.Tensor | None = None, norm_q: str | None = None, norm_k: str | None = None,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps_q: float = 1e-5,
                 eps_k: float = 1e-5, rope: int = 0, rope_dim: int = 0, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None):
        self.device = _lib.require_cuda(conv_weight, q_weight, k_weight, cos, sin)  # None: nothing is kept
        H = num_heads if num_kv_heads is None else num_kv_heads
        if H < 1 or num_heads % H:
            raise ValueError(f"num_heads={num_heads} must be a multiple of num_kv_heads={H}")
        if norm_q not in _NORM or norm_k not in _NORM:
            raise ValueError(f"norms must be None, 'l2' or 'rms', got {norm_q!r} and {norm_k!r}")
        for name, d in (("head_k_dim", head_k_dim), ("head_v_dim", head_v_dim)):
            if d < 8 or d > 256 or d % 8:
                raise ValueError(f"{name} must be a multiple of 8 up to 256, got {d}")
        self.num_heads, self.num_kv_heads, self.head_k_dim, self.head_v_dim = num_heads, H, head_k_dim, head_v_dim
        self.channels = C = (num_heads + H) * head_k_dim + H * head_v_dim
        f32 = lambda t: None if t is None else t.detach().float().contiguous()  # noqa: E731
        self.conv_size = 0 if conv_weight is None else conv_weight.shape[-1]
        if conv_weight is not None:
            if conv_weight.numel() != C * self.conv_size or conv_weight.shape[0] != C:
                raise ValueError(f"conv_weight must be ({C}, K), got {tuple(conv_weight.shape)}")
            if self.conv_size > 4:
                raise ValueError(f"the convolution is at most 4 wide, got {self.conv_size}")
        for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
            if t is not None and t.shape != (head_k_dim,):
                raise ValueError(f"{name} must be ({head_k_dim},), got {tuple(t.shape)}")
        if rope not in (0, 1, 2):
            raise ValueError(f"rope must be 0, 1 or 2, got {rope}")
        T = 0
        if rope:
            if rope == 1 and rope_dim != head_k_dim or rope == 2 and (rope_dim < 16 or rope_dim % 16 or
                                                                      head_k_dim % rope_dim):
                raise ValueError(f"rope={rope} does not go with rope_dim={rope_dim} and head_k_dim={head_k_dim}")
            if cos is None or sin is None or cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != rope_dim // 2 \
                    or cos.shape[0] < 1:
                raise ValueError(f"cos and sin must be (positions, {rope_dim // 2})")
            T = cos.shape[0]
        if conv_weight is not None:
            conv_weight = conv_weight.detach().reshape(C, self.conv_size).T  # taps first, as the kernel reads them
        self._keep = [f32(t) for t in (conv_weight, q_weight, k_weight, cos, sin)]
        self._args = {dt: _lib.QkvStepArgs(*[_lib.ptr(t) for t in self._keep], code, num_heads, H, head_k_dim, head_v_dim,
                                           self.conv_size, _NORM[norm_q], _NORM[norm_k], rope, rope_dim, T, eps_q, eps_k)
                      for dt, code in _lib.DTYPE.items()}

    def new_ring(self, batch: int, dtype: torch.dtype, device) -> torch.Tensor | None:
        """The ring (batch, K - 1, C) of sequences without a token yet, or None without a convolution of several taps."""
        if self.conv_size < 2:
            return None
        return torch.zeros(batch, self.conv_size - 1, self.channels, dtype=dtype, device=device)

    def ring_of(self, x: torch.Tensor) -> torch.Tensor | None:
        """The ring after the tokens of x (B, T, C), the projections of a prompt that starts at position 0."""
        ring = self.new_ring(x.shape[0], x.dtype, x.device)
        if ring is not None:
            for p in range(max(0, x.shape[1] - ring.shape[1]), x.shape[1]):
                ring[:, p % ring.shape[1]] = x[:, p]
        return ring

    def __call__(self, qkv: torch.Tensor, positions: torch.Tensor, ring: torch.Tensor | None = None):
        """q (B, num_heads, head_k_dim), k (B, num_kv_heads, head_k_dim), v (B, num_kv_heads, head_v_dim) of the
        projections qkv (B, C) of the tokens at ``positions`` (B,) int64.  ``ring`` (B, K - 1, C) is updated in place.
        A position that is negative or past the rotation tables gives NaN."""
        dev = _lib.require_cuda(qkv, positions, ring)
        if self.device is not None and dev != self.device:
            raise RuntimeError(f"qkv is on {dev}, the weights and tables on {self.device}")
        dt, shape = qkv.dtype, qkv.shape
        if len(shape) != 2 or shape[1] != self.channels:
            raise ValueError(f"qkv must be (B, {self.channels}), got {tuple(shape)}")
        args = self._args.get(dt)
        if args is None:
            raise TypeError(f"unsupported dtype {dt}")
        B = shape[0]
        if positions.shape != (B,) or positions.dtype != torch.int64:
            raise ValueError(f"positions must be ({B},) int64, got {tuple(positions.shape)} {positions.dtype}")
        if self.conv_size > 1 and (ring is None or ring.shape != (B, self.conv_size - 1, self.channels) or
                                   ring.dtype != dt or not ring.is_contiguous()):
            raise ValueError(f"ring must be a contiguous ({B}, {self.conv_size - 1}, {self.channels}) {dt} tensor")
        ld, one = qkv.stride()
        if one != 1 or ld % 8 or ld < self.channels or qkv.data_ptr() % 16:
            qkv = qkv.clone(memory_format=torch.contiguous_format)
            ld = self.channels
        if positions.stride(0) != 1:
            positions = positions.contiguous()
        q = torch.empty(B, self.num_heads, self.head_k_dim, dtype=dt, device=dev)
        k = torch.empty(B, self.num_kv_heads, self.head_k_dim, dtype=dt, device=dev)
        v = torch.empty(B, self.num_kv_heads, self.head_v_dim, dtype=dt, device=dev)
        with _lib.on_device(dev):
            rc = _lib.lib().kata_qkv_step(args, qkv.data_ptr(), ld, positions.data_ptr(), _lib.ptr(ring), q.data_ptr(),
                                          k.data_ptr(), v.data_ptr(), B, _lib.stream_handle(dev))
        if rc:
            _lib.check(rc, "kata_qkv_step")
        return q, k, v
