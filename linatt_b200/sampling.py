"""Drawing the next token: temperature, top-k, top-p and min-p from given random numbers.

A token's weight is w = exp((x - max x) / T), its mass the whole number rint(w 2^40).  Sums of masses
have no order: the drawn token depends on the row of logits, its settings and its uniform number
alone, not on the batch around it.  Tokens are ordered by logit, equal ones by index, and the filters
keep beginnings of that order: the first ``top_k`` tokens, of these the ones with less than ``top_p``
of their mass before them, of these the ones with w >= ``min_p`` (the first token always).  Drawn is
the first token, in vocabulary order, whose inclusive kept mass exceeds u times the whole.
The reference does not generate and has no counterpart.  There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["sample_tokens"]


def _setting(v, name, dtype, B, dev):
    """(tensor or None, scalar) of a setting given as a number or as a (B,) tensor."""
    if type(v) in (int, float):
        return None, v
    if not isinstance(v, torch.Tensor):
        return None, float(v)
    if v.shape != (B,):
        raise ValueError(f"{name} must be a number or a ({B},) tensor, got {tuple(v.shape)}")
    if v.device != dev:
        raise RuntimeError(f"{name} is on {v.device}, the logits on {dev}")
    if dtype == torch.int32 and v.dtype != dtype:
        v = v.clamp(0, 1 << 30)  # beyond 32 bits too (the vocabulary is smaller)
    return v.to(dtype).contiguous(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(token (B,) int64, logprob (B,) fp32) drawn from logits (B, V) bf16 / f16 / fp32 with the uniform
    numbers u (B,) in [0, 1).  Each setting is a number or a (B,) tensor.  ``temperature`` <= 0: the
    likeliest token (the lowest index of equal ones).  ``top_k`` <= 0, ``top_p`` >= 1 and ``min_p`` <= 0
    keep everything.  Logits of -inf (a mask) and NaN are never drawn; a row with nothing else gives token
    -1 and logprob -inf.  ``logprob`` is the token's log probability among the kept ones."""
    dev = _lib.require_cuda(logits, u)
    if logits.dim() != 2:
        raise ValueError(f"logits must be (B, V), got {tuple(logits.shape)}")
    if logits.dtype not in _lib.DTYPE:
        raise TypeError(f"unsupported logits dtype {logits.dtype}")
    B, V = logits.shape
    ld, one = logits.stride()
    if u.shape != (B,) or u.dtype != torch.float32:
        raise ValueError(f"u must be ({B},) fp32, got {tuple(u.shape)} {u.dtype}")
    if V < 1:
        raise ValueError("the vocabulary is empty")
    if one != 1 or (ld < V and B > 1):
        logits = logits.contiguous()
        ld = V
    tt, ts = _setting(temperature, "temperature", torch.float32, B, dev)
    kt, ks = _setting(top_k, "top_k", torch.int32, B, dev)
    pt, ps = _setting(top_p, "top_p", torch.float32, B, dev)
    mt, ms = _setting(min_p, "min_p", torch.float32, B, dev)
    if u.stride(0) != 1:
        u = u.contiguous()
    token = torch.empty(B, dtype=torch.int64, device=dev)
    logprob = torch.empty(B, dtype=torch.float32, device=dev)
    a = _lib.SampleArgs(logits.data_ptr(), u.data_ptr(), _lib.ptr(tt), _lib.ptr(kt), _lib.ptr(pt), _lib.ptr(mt),
                        token.data_ptr(), logprob.data_ptr(), ld, B, V, _lib.DTYPE[logits.dtype], ts,
                        min(max(int(ks), 0), 2 ** 31 - 1), ps, ms)
    with _lib.on_device(dev):
        rc = _lib.lib().kata_sample(a, _lib.stream_handle(dev))
    if rc:
        _lib.check(rc, "kata_sample")
    return token, logprob
