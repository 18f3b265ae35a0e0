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


# ------------------------------------------------------------------ the balance loss of a module with a checkpoint
def balance_gradients(m, x, valid):
    """(loss, dx, dwq, dk) of the module's balance loss in 64 bits, on the routes that token routing takes."""
    base, T = m.base_blocks, m.temperature
    s, idx, cnt = None, None, None
    with torch.no_grad():
        s = m.compute_router_scores(x)
        idx, cnt, _, _ = kernels.select(s, base_blocks=base, top_p=m.top_p, min_remote=m.min_remote_blocks,
                                        max_remote=m.max_remote_blocks, capacity=m.max_remote_blocks, temperature=T)
    live = (torch.arange(idx.shape[1], device=x.device) < cnt[:, None]) & valid[:, None]
    counts = torch.bincount(idx[live].long(), minlength=m.num_blocks)
    leaves = [t.detach().double().requires_grad_() for t in (x, m.q_proj_16d.weight, m.block_keys_16d)]
    xx, wq, k16 = leaves
    q = xx @ wq.t()
    n = q * ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    p = torch.softmax((n @ k16.t() / 4)[:, base:] / T, dim=1)[valid]
    f = counts[base:].double() / int(counts.sum())
    loss = (m.num_blocks - base) * (f * p.mean(dim=0)).sum()
    return (loss.detach(), counts, *torch.autograd.grad(loss, leaves))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead,D", [((3, 70), 256), ((401,), 1000)])
def test_balance_loss_of_a_checkpointed_module(lead, D, dtype):
    """The loss and counts are those without a checkpoint; the gradients, under an upstream gradient of 0.3 and for each
    subset of what requires one, are the 64-bit formula's, rounded once (e: the router gradient's budget, and as
    much for the softmax and its projection)."""
    m, plain = make_mlp(dtype, "mxfp8", D=D), make_mlp(dtype, None, D=D)
    x = randn(*lead, D, seed=350, dtype=dtype)
    valid = torch.rand(lead, generator=torch.Generator(device="cuda").manual_seed(351), device="cuda") < 0.8
    loss, counts, *ref = balance_gradients(m, x.reshape(-1, D), valid.reshape(-1))
    e = 2 * budget(D)
    full = None
    for mask in (7, 1, 2, 4, 6):
        xin = x.clone().requires_grad_(bool(mask & 1))
        leaves = [xin, m.q_proj_16d.weight.requires_grad_(bool(mask & 2)), m.block_keys_16d.requires_grad_(bool(mask & 4))]
        got, c = m.balance_loss(xin, valid)
        pl, pc = plain.balance_loss(x, valid)
        assert torch.equal(got.detach(), pl.detach()) and torch.equal(c, pc) and torch.equal(c, counts)
        assert abs(float(got.detach()) - float(loss)) <= e * float(loss)
        want = [i for i in range(3) if mask >> i & 1]
        grads = torch.autograd.grad(got, [leaves[i] for i in want], torch.full((), 0.3, device="cuda"))
        if mask == 7:
            full = grads
            for g, r in zip(grads, ref):
                g, r = g.reshape(r.shape), 0.3 * r
                if dtype == torch.bfloat16:
                    check_rounded_once(g, r, e)
                else:
                    assert float((g.double() - r).norm()) <= e * float(r.norm())
            assert not bool(grads[0][~valid].any())
        assert all(torch.equal(g, full[i]) for g, i in zip(grads, want))
    with torch.no_grad():
        assert m.balance_loss(x, valid)[0].grad_fn is None
    with pytest.raises(ValueError):
        m.balance_loss(x[..., :D - 8])
    y = torch.zeros(0, D, dtype=dtype, device="cuda", requires_grad=True)
    g = torch.autograd.grad(m.requires_grad_().balance_loss(y)[0], [y, m.q_proj_16d.weight, m.block_keys_16d])
    assert g[0].shape == (0, D) and not bool(g[1].any()) and not bool(g[2].any())


def held_bytes(checkpoint, M, D):
    """Bytes that a step's graph holds between the passes, with x itself an activation that only the graph keeps."""
    m = make_mlp(torch.bfloat16, checkpoint, D=D)
    leaf = randn(M, D, seed=360, dtype=torch.bfloat16).requires_grad_()
    for _ in range(2):  # the first step leaves packed weights and workspaces
        m.zero_grad(set_to_none=True)
        leaf.grad = None
        before = torch.cuda.memory_allocated()
        x = leaf * 1.0
        y, (loss, counts) = m(x), m.balance_loss(x)
        del x
        held = torch.cuda.memory_allocated() - before - y.numel() * 2
        torch.autograd.backward([y, loss], [torch.ones_like(y), torch.ones_like(loss)])
        del y, loss, counts
    return held


@pytest.mark.gpu
def test_step_with_a_checkpoint_holds_fewer_bytes():
    """Output and balance loss of one step: without a checkpoint both keep x (2 bytes an element, once), with it one
    8-bit copy (1 + 1/32) is left.  Queries (68 bytes a token), q_proj's gradient (64 D bytes) and rounded
    allocations are the rest: 0.88 bytes an element fewer at 1024 wide."""
    M, D = 8192, 1024
    plain, kept = held_bytes(None, M, D), held_bytes("mxfp8", M, D)
    assert 2 * M * D <= plain and kept <= plain - 0.88 * M * D, (plain / M / D, kept / M / D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_router_scores_keep_the_tokens_for_q_proj_only(checkpoint, dtype):
    """Where q_proj takes no gradient (a frozen projection), nothing of x's size is kept, and the other gradients are the
    same bits."""
    x, wq, k16 = randn(120, 256, seed=370, dtype=dtype), randn(16, 256, seed=371, dtype=dtype), randn(9, 16, seed=372, dtype=dtype)
    ds = randn(120, 9, seed=373)
    leaves = [t.clone().requires_grad_() for t in (x, wq, k16)]
    full = torch.autograd.grad(fsi.router_scores(*leaves, checkpoint=checkpoint), leaves, ds)
    for frozen, kept in ((True, 0), (False, 256 + 8 if checkpoint else 256 * x.element_size())):
        xin, k = x.clone().requires_grad_(), k16.clone().requires_grad_()
        w = wq.clone().requires_grad_(not frozen)
        s = fsi.router_scores(xin, w, k, checkpoint=checkpoint)
        sizes = sorted(t.numel() * t.element_size() for t in s.grad_fn.saved_tensors if t is not None)
        rest = [w.numel() * w.element_size(), k.numel() * k.element_size(), 17 * 120 * 4]
        assert sizes == sorted(rest + ([120 * kept] if kept else [])), (frozen, sizes)
        dx, dk = torch.autograd.grad(s, (xin, k), ds)
        assert torch.equal(dx, full[0]) and torch.equal(dk, full[2])


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_balance_loss_of_a_module_captured_and_replayed(checkpoint):
    """The module's balance loss with its gradients in a CUDA graph, replayed on other inputs and weights."""
    m = make_mlp(torch.bfloat16, checkpoint)
    x = randn(90, 256, seed=380, dtype=torch.bfloat16).requires_grad_()
    valid = torch.ones(90, dtype=torch.bool, device="cuda")
    leaves = [x, m.q_proj_16d.weight, m.block_keys_16d]

    def step():
        loss, counts = m.balance_loss(x, valid)
        return [loss.detach(), counts, *torch.autograd.grad(loss, leaves, torch.full((), 0.5, device="cuda"))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(randn(90, 256, seed=381, dtype=torch.bfloat16))
        m.q_proj_16d.weight.mul_(1.5)
        valid[40:60] = False
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_balance_loss_of_a_module_with_a_temperature_of_another_type(checkpoint):
    """A temperature that is a tensor or a numpy number counts as its value; one token alone has its gradients."""
    import numpy as np

    m = make_mlp(torch.float32, checkpoint)
    x = randn(256, seed=390).requires_grad_()
    out = []
    for T in (0.5, torch.tensor(0.5), np.float32(0.5)):
        m.temperature = T
        loss, counts = m.balance_loss(x)
        out.append([loss.detach(), counts, *torch.autograd.grad(loss, [x, m.q_proj_16d.weight, m.block_keys_16d])])
    assert out[0][2].shape == (256,) and bool(out[0][2].any())
    assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(o, out[0]))
