"""The SwiGLU backward's third output: h = silu(g^) u^ at the values g^, u^ of the 8-bit copies."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import fsi

pytestmark = pytest.mark.gpu
kernels = fsi.kernels
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 7, 31, 33, 1001, 4096, 5003])
def test_swiglu_backward_h(n, dtype):
    """h against the 64-bit formula; the gradients are the bits they are without it; bytes behind each output's n
    elements stay as they were.  Roundings: sigmoid 8 u (exponential two steps, sum, division: 4 steps), the two
    products one each, the output's half step; the bf16 kernel's fast exponential (2 + 1.16 |g| steps) adds
    (4 + 3 |g|) u."""
    gen = torch.Generator(device="cuda").manual_seed(400 + n)
    g = (torch.randn(n, generator=gen, device="cuda") * 4).to(dtype)
    u, d = (torch.randn(n, generator=gen, device="cuda").to(dtype) for _ in range(2))
    _, buf = kernels.swiglu_fwd_mxfp8(g, u)
    dg, du, h = kernels.swiglu_bwd_mxfp8(d, buf, want_h=True)
    rg, ru, none = kernels.swiglu_bwd_mxfp8(d, buf)
    assert none is None and torch.equal(dg, rg) and torch.equal(du, ru)
    gq, uq = (fsi.checkpoint_mxfp8(t).restore().double() for t in (g, u))
    ref = gq * torch.sigmoid(gq) * uq
    tol = (torch.finfo(dtype).eps / 2 + (16 + 3 * gq.abs()) * U) * ref.abs() + 1e-37
    assert bool(((h.double() - ref).abs() <= tol).all())
    out = [torch.full((n + 64,), 7.0, dtype=dtype, device="cuda") for _ in range(3)]
    half = kernels._swiglu_half(n)
    P = ctypes.c_void_p
    at = [P(a) for a in (*kernels._mx_addrs(buf, n), *kernels._mx_addrs(buf, n, half))]
    rc = fsi.load_library().fp_swiglu_bwd_mxfp8(P(d.data_ptr()), *at, 0 if dtype == torch.float32 else 1, n,
                                                *(P(t.data_ptr()) for t in out),
                                                P(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    for o, r in zip(out, (dg, du, h)):
        assert torch.equal(o[:n], r) and bool((o[n:] == 7.0).all())
