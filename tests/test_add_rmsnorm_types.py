"""The fused residual add and RMSNorm hands its kernels fp32 weights and takes an fp32 weight gradient,
whatever the type of the parameter: the entries are replaced by ones that look at what they are given, so
nothing is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from linatt_b200 import _lib, lm


def floats(address, n):
    return torch.tensor((ctypes.c_float * n).from_address(address)[:])


class Entries:
    """The first half of the weights (and of their gradient), read and written as fp32: within a 16-bit buffer too."""

    def kata_add_rmsnorm_fwd(self, a, stream):
        self.fwd = floats(a.w, a.N // 2)
        return 0

    def kata_add_rmsnorm_bwd_workspace_bytes(self, a):
        return 0

    def kata_add_rmsnorm_bwd(self, a, stream):
        self.bwd = floats(a.w, a.N // 2)
        (ctypes.c_float * (a.N // 2)).from_address(a.dw)[:] = [1.5] * (a.N // 2)
        return 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_weights_reach_the_kernels_as_fp32(monkeypatch, dtype):
    entries, N = Entries(), 256
    monkeypatch.setattr(_lib, "require_cuda", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(_lib, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(_lib, "lib", lambda: entries)
    norm = lm.RMSNorm(N, 1e-6).to(dtype)
    with torch.no_grad():
        norm.weight.copy_(torch.randn(N, generator=torch.Generator().manual_seed(1)))
    h = torch.zeros(3, N, requires_grad=True)
    h_out, y = lm.add_rmsnorm(h, torch.zeros(3, N, dtype=torch.bfloat16), norm)
    assert torch.equal(entries.fwd, norm.weight.detach().float()[: N // 2])
    torch.autograd.backward([h_out, y], [torch.zeros_like(h_out), torch.zeros_like(y)])
    assert torch.equal(entries.bwd, entries.fwd)
    assert norm.weight.grad.dtype == dtype and (norm.weight.grad[: N // 2] == 1.5).all()
