"""The training step of FovealPattentionMLP with its options: precision of the kept form, second derivatives, bytes
held between the passes.  u = 2^-24 is half a step of fp32."""

from __future__ import annotations

import pytest
import torch

from conftest import fsi
from test_router_gradient import EPS, U, budget

kernels = fsi.kernels


def make_mlp(dtype, checkpoint, device="cuda", D=256, Np=1024, out_scale=3000.0):
    """``out_scale`` makes the additive stream's gradients as large as the contraction's (twice at 3000)."""
    torch.manual_seed(0)
    m = fsi.FovealPattentionMLP(D, Np, base_blocks=2, remote_blocks=4, dtype=dtype, checkpoint=checkpoint,
                                min_remote_blocks=1, max_remote_blocks=5)
    with torch.no_grad():
        m.out_proj_16d.weight.mul_(out_scale)
        m.block_keys_16d.mul_(3)
    return m.to(device).train()


def randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def additive_gradients(m, x, dy):
    """(the router's part of dx, block_keys' gradient) of the additive stream in 64 bits."""
    wq, k16, wo = (t.detach().double() for t in (m.q_proj_16d.weight, m.block_keys_16d, m.out_proj_16d.weight))
    q = x.double() @ wq.t()
    r = ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    n = q * r
    soft = torch.softmax(n @ k16.t() / 4 / m.temperature, dim=1)
    dctx = dy.double() @ wo
    dsoft = dctx @ k16.t()
    dS = soft * (dsoft - (dsoft * soft).sum(dim=1, keepdim=True)) / m.temperature
    a = dS @ k16 / 4
    dq = r * (a - n * (a * n).mean(dim=1, keepdim=True))
    return dq @ wq, soft.t() @ dctx + dS.t() @ n / 4


def check_rounded_once(got, ref, e):
    """``got`` is ``ref`` rounded to bf16, but for elements that a relative error e of the sum in front of the rounding
    moves over a border: sqrt(2^-7 e) of the norm (as in test_router_gradient.py)."""
    d = (got.double() - ref.to(torch.bfloat16).double()).norm()
    tol = ((2.0 ** -7 * e) ** 0.5 + e) * float(ref.norm()) + 3 * 2.0 ** -7 * float(ref.abs().max())
    assert float(d) <= tol, (float(d / ref.norm()), tol / float(ref.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_module_sums_round_once(checkpoint):
    """dx and block_keys' gradient are sums of the contraction's or the stream's part and the router's, which reach
    the module's type in one rounding: the parts are added in 32 bits.  e: the router gradient's budget, and as
    much again for each of the products in front of it (dy out_proj over 256 terms, the softmax, soft^T dctx)."""
    m = make_mlp(torch.bfloat16, checkpoint)
    x, dy = randn(300, 256, seed=300, dtype=torch.bfloat16), randn(300, 256, seed=301, dtype=torch.bfloat16)
    xin = x.clone().requires_grad_()
    m(xin).backward(dy)
    without = make_mlp(torch.bfloat16, checkpoint, out_scale=0.0)  # no additive stream: dx is the contraction's part
    x0 = x.clone().requires_grad_()
    without(x0).backward(dy)
    dx_r, dk = additive_gradients(m, x, dy)
    e = 4 * budget(256)
    assert 0.5 < float(dx_r.norm() / x0.grad.double().norm()) < 5
    check_rounded_once(xin.grad, x0.grad.double() + dx_r, e)
    check_rounded_once(m.block_keys_16d.grad, dk, e)


# ------------------------------------------------------------------ second derivatives
class Square(torch.autograd.Function):
    """x^2 whose backward pass saves x and is declared first order."""

    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return x * x

    @staticmethod
    @fsi.training.once
    def backward(ctx, d):
        x, = ctx.saved_tensors
        return 2 * x.detach() * d


def check_first_order(f, leaves, up=None):
    """The gradients of ``f(*leaves)`` under create_graph are the plain ones, and a penalty on one of them raises
    instead of losing its own gradient, whether or not the upstream gradient requires one."""
    plain = torch.autograd.grad(f(*leaves).sum(), leaves)
    for y_of in (lambda y: y.sum(), lambda y: (y * y).sum()):
        y = f(*leaves)
        grads = torch.autograd.grad(y_of(y), leaves, create_graph=True)
        if y_of(torch.full((2,), 3.0)) == 6.0:
            assert all(torch.equal(a.detach(), b) for a, b in zip(grads, plain))
        for g in grads:
            with pytest.raises(RuntimeError):
                (y.float().sum() + g.float().pow(2).sum()).backward(retain_graph=True)


def test_once_refuses_a_second_derivative():
    check_first_order(Square.apply, [torch.randn(5, requires_grad=True)])
    x = torch.randn(5, requires_grad=True)
    Square.apply(x).sum().backward()
    assert torch.equal(x.grad, 2 * x.detach()) and not x.grad.requires_grad
    x.grad = None
    Square.apply(x).sum().backward(create_graph=True)  # and an in-place update of what it left
    x.grad.detach_().add_(1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_second_derivatives_raise(checkpoint):
    x, wq, k16 = (randn(*s, seed=310 + i).requires_grad_() for i, s in enumerate(((40, 64), (16, 64), (8, 16))))
    check_first_order(lambda *t: fsi.router_scores(*t, checkpoint=checkpoint), [x, wq, k16])
    g, u = (randn(33, 65, seed=320 + i).requires_grad_() for i in range(2))
    check_first_order(lambda *t: fsi.triton_fused_swiglu(*t, checkpoint=checkpoint), [g, u])
    m = make_mlp(torch.float32, checkpoint)
    xm = randn(20, 256, seed=330).requires_grad_()
    check_first_order(lambda t, *_: m(t), [xm, m.q_proj_16d.weight, m.block_keys_16d, m.out_proj_16d.weight, m.v])
    check_first_order(lambda t, *_: m.balance_loss(t)[0], [xm, m.q_proj_16d.weight, m.block_keys_16d])
    s = randn(50, 8, seed=340).requires_grad_()
    idx = torch.full((50, 1), 5, dtype=torch.int32, device="cuda")
    cnt = torch.ones(50, dtype=torch.int32, device="cuda")
    check_first_order(lambda t: fsi.balance_loss(t, idx, cnt, base_blocks=1)[0], [s])
