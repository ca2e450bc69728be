"""Linear layers with 4-bit weights, for generation.

A weight W (N, K) is kept as codes 0..15 with a scale (and optionally a zero point) for every group
of ``group_size`` values of a row:

    W[n, k] = scale[n, k // g] (code[n, k] - zero[n, k // g])          zero = 8 when not given

:class:`W4Weight` lays such a weight out for the kernels once; :func:`w4_linear` is y = x W^T (or the
SwiGLU of a weight that holds gate and up rows); :func:`quantize_w4` makes one from a 16- or 32-bit
weight by rounding to the nearest code.  The reference keeps its weights in 16 or 32 bits and has no
counterpart.  Inference only (no autograd).  There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["W4Weight", "w4_linear", "quantize_w4"]


class W4Weight:
    """A 4-bit weight in the kernels' layout.

    ``packed``: (N, 4 ceil(K/32)) int32, code k of a row in bits 4 (k % 8) .. +3 of word k // 8 (codes
    past K are ignored).  ``scales``: (N, ceil(K/group_size)) bf16, f16 or fp32; activations are of the
    same type.  ``zeros``: (N, ceil(K/group_size)) uint8 in 0..15, or None for 8 throughout.
    ``group_size``: 32, 64 or a multiple of 128.  ``activation="swiglu"``: the rows are N/2 gate rows
    and then N/2 up rows, and the layer's output is silu(gate) * up, N/2 wide.  The three tensors are
    copied into the layout; none is kept."""

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
                 in_features: int, group_size: int = 128, activation: str | None = None):
        dev = _lib.require_cuda(packed, scales, zeros)
        if activation not in (None, "swiglu"):
            raise ValueError(f"activation must be None or 'swiglu', got {activation!r}")
        if scales.dtype not in _lib.DTYPE:
            raise TypeError(f"unsupported scale dtype {scales.dtype}")
        if packed.dtype != torch.int32 or (zeros is not None and zeros.dtype != torch.uint8):
            raise TypeError("packed must be int32 and zeros uint8")
        K = int(in_features)
        if K < 1 or group_size < 1:
            raise ValueError(f"in_features and group_size must be positive, got {K} and {group_size}")
        if packed.dim() != 2 or packed.shape[1] != 4 * (-(-K // 32)):
            raise ValueError(f"packed must be (N, {4 * (-(-K // 32))}) for in_features={K}, got {tuple(packed.shape)}")
        N, G = packed.shape[0], -(-K // group_size)
        for name, t in (("scales", scales), ("zeros", zeros)):
            if t is not None and tuple(t.shape) != (N, G):
                raise ValueError(f"{name} must be (N, ceil(in_features / group_size)) = ({N}, {G}), got {tuple(t.shape)}")
        self.out_features = N // 2 if activation else N
        self.in_features, self.group_size, self.activation = K, int(group_size), activation
        self.dtype, self.device = scales.dtype, dev
        L = _lib.lib()
        a = _lib.W4WeightArgs(None, N, K, int(group_size), _lib.DTYPE[scales.dtype], int(activation == "swiglu"),
                              int(zeros is not None))
        n = L.kata_w4_bytes(a)
        if n == 0:
            raise ValueError(f"unsupported 4-bit weight: N={N}, K={K}, group_size={group_size} (32, 64 or a multiple of "
                             f"128), activation={activation!r} (an even N)")
        with _lib.on_device(dev):
            data = torch.empty(n, dtype=torch.uint8, device=dev)
            a.data = data.data_ptr()
            pc, sc, zc = packed.contiguous(), scales.contiguous(), None if zeros is None else zeros.contiguous()
            _lib.check(L.kata_w4_pack(pc.data_ptr(), sc.data_ptr(), _lib.ptr(zc), a, _lib.stream_handle(dev)),
                       "kata_w4_pack")
        self._data, self._args = data, a

    @property
    def nbytes(self) -> int:
        """Device bytes of the laid-out codes, scales and zero points."""
        return self._data.numel()


def w4_linear(x: torch.Tensor, w: W4Weight) -> torch.Tensor:
    """y = x W^T of x (..., in_features) in the weight's dtype, or silu(gate) * up for a gated weight:
    (..., out_features).  Products are exact and summed in fp32; y is rounded once.  Up to 2^21 rows."""
    if x.device != w.device:
        _lib.require_cuda(x)
        raise RuntimeError(f"x is on {x.device}, the weight on {w.device}")
    if x.dtype != w.dtype:
        raise TypeError(f"x is {x.dtype}, the weight's scales are {w.dtype}")
    K, shape = w.in_features, x.shape
    if not shape or shape[-1] != K:
        raise ValueError(f"x must be (..., {K}), got {tuple(shape)}")
    x2 = x if len(shape) == 2 else x.reshape(-1, K)
    ldx, one = x2.stride()
    rows = x2.shape[0]
    if one != 1 or (ldx < K and rows > 1):
        x2 = x2.contiguous()
        ldx = K
    dev = w.device
    y = torch.empty(*shape[:-1], w.out_features, dtype=w.dtype, device=dev)
    if rows:
        with _lib.on_device(dev):
            L, xp, ws, n = _lib.lib(), x2.data_ptr(), None, 0
            # three rows, and 16-bit ones that lie on 16-byte boundaries, never need any
            if rows > 3 and (w.dtype is torch.float32 or ldx % 8 or xp % 16):
                n = L.kata_w4_workspace_bytes(w._args, xp, ldx, rows)
                if n:
                    ws = torch.empty(n, dtype=torch.uint8, device=dev)
            rc = L.kata_w4_linear(w._args, xp, ldx, y.data_ptr(), w.out_features, rows, _lib.ptr(ws), n,
                                  _lib.status_word(dev).data_ptr(), _lib.stream_handle(dev))
        if rc:
            _lib.check(rc, "kata_w4_linear")
    return y


@torch.no_grad()
def quantize_w4(weight: torch.Tensor, group_size: int = 128, *, symmetric: bool = True, dtype: torch.dtype | None = None,
                activation: str | None = None) -> W4Weight:
    """Round a (N, K) weight to 4 bits.  ``symmetric``: zero point 8, scale max|w| / 7 of the group; otherwise the
    group's [min(w, 0), max(w, 0)] is spread over the 16 codes with a zero point of its own.  ``dtype``: of the
    scales and of the activations it will meet (default: the weight's)."""
    _lib.require_cuda(weight)
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"weight must be a floating (N, K) matrix, got {tuple(weight.shape)} {weight.dtype}")
    dtype = weight.dtype if dtype is None else dtype
    N, K = weight.shape
    G = -(-K // group_size)
    w = torch.nn.functional.pad(weight.float(), (0, G * group_size - K)).view(N, G, group_size)
    if symmetric:
        scale = (w.abs().amax(-1) / 7).to(dtype)
        zero = None
        z = 8.0
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scale = ((hi - lo) / 15).to(dtype)
        s = scale.float()
        zero = torch.where(s > 0, (-lo / s).round().clamp(0, 15), 8.0).to(torch.uint8)
        z = zero.float()[..., None]
    s = scale.float()[..., None]
    code = torch.where(s > 0, (w / s).round() + z, 8.0).clamp(0, 15).to(torch.int32).view(N, -1)
    words = 4 * (-(-K // 32))
    code = torch.nn.functional.pad(code, (0, max(0, 8 * words - code.shape[1])))[:, : 8 * words].reshape(N, words, 8)
    # the eight nibbles do not overlap: their sum is their union (modulo 2^32)
    packed = (code << torch.arange(0, 32, 4, device=code.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)
    return W4Weight(packed, scale, zero, in_features=K, group_size=group_size, activation=activation)
