"""Precision of the router scores' gradient, by norms against a 64-bit restatement.

Elementwise bounds from sums of magnitudes grow faster than the gradients themselves; what the kernels' roundings
do to a gradient as a whole is far smaller, and its norm shows a wrong or imprecise term that such bounds let
pass.  u = 2^-24 is half a step of fp32.  A gradient's relative error in norm is taken to be at most
``budget(D)`` = (24 + D / 256) u, the sum of

* 4 u: dS as two tf32 pieces (the rest is below 2^-22 of each term);
* 8 u: a = dS K / 4 in chains of 8 steps of the tensor cores, which round towards zero, u on average a step;
* 8 u: the normalisation, its dot product and the projection (a rounding each of a few fp32 operations);
* 4 u: the last product (three steps of the tensor cores, or one chain of 16 fused multiply-adds);
* D / 256 u: the forward's projections, D / 64 truncated steps in a quarter of the width (on partial sums, which
  grow like a square root, and of which the part common to all of a query drops out in the normalisation).

dx in bf16 is compared with the reference rounded to bf16.  An error d of an element moves its rounding over a
border with probability |d| / s, s <= 2^-7 |v| the step there, and changes it by s; the squares add up to
sum |d| s <= 2^-7 |d| |v| in norms (Cauchy-Schwarz), so the norm of the change is sqrt(2^-7 e) |v|; three steps at
the largest element are left for the chance in it.
"""

from __future__ import annotations

import pytest
import torch

from conftest import fsi

kernels = fsi.kernels
U = 2.0 ** -24
EPS = 1.1920928955078125e-07
SIZES = [(1, 8, 1), (1, 64, 16), (3, 72, 5), (16, 256, 16), (17, 264, 33), (64, 256, 224), (130, 1000, 65),
         (33, 512, 1024), (257, 1024, 130), (1000, 128, 12), (700, 512, 448)]
LARGE = [(2111, 4096, 224), (5000, 2056, 64), (9001, 1536, 1000)]  # many CTAs along both sides, odd ends


def budget(D):
    return (24 + D / 256) * U


def inputs(M, D, NB, dtype, device, seed=200):
    """x in ``dtype``, weights of fp32 that hold values of ``dtype`` (their gradients leave in fp32), dS."""
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)
    x, wq, k16, ds = r(M, D), r(16, D) * D ** -0.5, r(NB, 16) * 0.25, r(M, NB)
    return x.to(dtype), wq.to(dtype).float(), k16.to(dtype).float(), ds


def gradient(x, xq, wq, k16, ds):
    """(dx, dwq, dk) in 64 bits; ``xq``: the tokens that q_proj's gradient reads."""
    x, xq, wq, k16, ds = (t.detach().double() for t in (x, xq, wq, k16, ds))
    q = x @ wq.t()
    r = ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    n = q * r
    a = ds @ k16 / 4
    dq = r * (a - n * (a * n).mean(dim=1, keepdim=True))
    return dq @ wq, dq.t() @ xq, ds.t() @ n / 4


def check_norms(got, ref, dtype, e):
    """dx, dwq and dk as wholes, and dwq by router dimension, dx by token and dk by block: none may have less
    than the average of the allowance."""
    for name, g, r in zip(("dx", "dwq", "dk")[-len(got):], got, ref):
        assert bool(torch.isfinite(g).all()), name
        one = r.double()
        tol = e
        slack = 0.0
        if name == "dx" and dtype == torch.bfloat16:
            one = one.to(dtype).double()
            tol = (2.0 ** -7 * e) ** 0.5 + e
            slack = 3 * 2.0 ** -7
        d = g.double() - one
        assert float(d.norm()) <= tol * float(r.norm()) + slack * float(r.abs().max()), \
            (name, float(d.norm() / r.norm()), tol)
        rows = r.norm(dim=1).clamp_min(float(r.norm()) / r.shape[0] ** 0.5)
        over = d.norm(dim=1) - (4 * tol * rows + slack * r.abs().amax(dim=1))
        assert float(over.max()) <= 0, (name, int(over.argmax()), float(over.max()))


def run(x, wq, k16, ds, checkpoint):
    leaves = [t.clone().requires_grad_() for t in (x, wq, k16)]
    return torch.autograd.grad(fsi.router_scores(*leaves, checkpoint=checkpoint), leaves, ds)


def kept(x, checkpoint):
    return fsi.checkpoint_mxfp8(x).restore() if checkpoint else x


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D,NB", SIZES + LARGE)
def test_gradient_norms(M, D, NB, dtype, checkpoint):
    x, wq, k16, ds = inputs(M, D, NB, dtype, "cuda")
    got = run(x, wq, k16, ds, checkpoint)
    assert [g.dtype for g in got] == [dtype, torch.float32, torch.float32]
    check_norms(got, gradient(x, kept(x, checkpoint), wq, k16, ds), dtype, budget(D))



def pieces(v, k):
    """``v`` as the sum of its k leading bf16 pieces."""
    out = torch.zeros_like(v)
    for _ in range(k):
        out = out + (v - out).to(torch.bfloat16).double()
    return out


def mutants(x, wq, k16, ds):
    """(name, gradients) of calculations that are wrong or too coarse."""
    x, wq, k16, ds = (t.double() for t in (x, wq, k16, ds))
    q = x @ wq.t()
    r = ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    n = q * r
    a = ds @ k16 / 4
    dq = r * (a - n * (a * n).mean(dim=1, keepdim=True))
    dk = ds.t() @ n / 4
    right = (dq @ wq, dq.t() @ x, dk)
    for i, name in enumerate(("dx", "dwq", "dk")):
        yield name + " zero", tuple(torch.zeros_like(t) if i == j else t for j, t in enumerate(right))
        yield name + " of one token less", tuple(
            (torch.cat([t[:-1], 0 * t[-1:]]) if i == 0 else t - (dq[-1:].t() @ x[-1:] if i == 1 else ds[-1:].t() @ n[-1:] / 4))
            if i == j else t for j, t in enumerate(right))
    for name, d in (("no projection", r * a), ("no factor", dq / r), ("dq in one bf16 piece", pieces(dq, 1))):
        yield name + " in dx", (d @ wq, right[1], dk)
        yield name + " in dwq", (right[0], d.t() @ x, dk)
    yield "a transposed sign", (right[0], right[1], -dk)
    if x.shape[0] >= 16:  # (a few elements alone may be rounded well by chance)
        yield "dq in two bf16 pieces", (right[0], pieces(dq, 2).t() @ x, dk)
        yield "dk off by 2^-12", (right[0], right[1], dk * (1 + 2.0 ** -12))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D,NB", SIZES)
def test_the_norms_reject_what_is_wrong(M, D, NB, dtype):
    """On the CPU, at every size: the right gradients pass, rounded to the outputs' types, and every wrong one fails."""
    x, wq, k16, ds = inputs(M, D, NB, dtype, "cpu")
    ref = gradient(x, x, wq, k16, ds)
    out = lambda t: (t[0].to(dtype), t[1].float(), t[2].float())
    check_norms(out(ref), ref, dtype, budget(D))
    for name, t in mutants(x, wq, k16, ds):
        if dtype == torch.bfloat16 and name == "dq in one bf16 piece in dx" and M * D < 4096:
            continue  # bf16 outputs of few elements: the allowance for the chance in their rounding is as large
        with pytest.raises(AssertionError):
            check_norms(out(t), ref, dtype, budget(D))
            raise ValueError(f"not rejected: {name}")

@pytest.mark.gpu
def test_input_gradient_has_no_part_along_the_query():
    """A token that is the d-th unit vector has the d-th column of q_proj as its query q, and dx_d = dq q, which the
    normalisation makes 0 but for eps.  What is left are the roundings: of the factor r (twice, on the quarter
    of a that a direction among 16 has), of the dot product and of each dq, together some u of |dq| |q|; 4 u
    are allowed.  dq in fewer than 24 bits shows: two bf16 pieces leave 2^-18.7 / 4 = 10 u."""
    D, NB = 64, 40
    g = torch.Generator(device="cuda").manual_seed(210)
    wq = torch.randint(-60, 61, (16, D), generator=g, device="cuda").to(torch.bfloat16)
    k16 = torch.randn(NB, 16, generator=g, device="cuda").to(torch.bfloat16)
    ds = torch.randn(8 * D, NB, generator=g, device="cuda")
    x = torch.eye(D, device="cuda").repeat(8, 1).to(torch.bfloat16).requires_grad_()
    dx, = torch.autograd.grad(fsi.router_scores(x, wq, k16), x, ds)
    at = torch.arange(8 * D, device="cuda")
    ref = gradient(x, x, wq, k16, ds)[0]
    q = wq.double().t().repeat(8, 1)
    n = q * ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    a = ds.double() @ k16.double() / 4
    dq = (a - n * (a * n).mean(dim=1, keepdim=True)) * (n.norm(dim=1) / q.norm(dim=1))[:, None]
    err = (dx.double() - ref)[at, at % D].norm()
    assert float(err) <= 4 * U * float((dq.norm(dim=1) * q.norm(dim=1)).norm()), \
        float(err / (dq.norm(dim=1) * q.norm(dim=1)).norm() / U)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_key_gradient_over_many_tokens(dtype):
    """dk's error does not grow with the tokens: its sums leave the tensor cores, which round towards zero, every 8
    steps (one chain over a CTA's tokens left 100 u here)."""
    M, D, NB = 1 << 18, 256, 32
    x, wq, k16, ds = inputs(M, D, NB, dtype, "cuda", seed=220)
    k16 = k16.requires_grad_()
    got, = torch.autograd.grad(fsi.router_scores(x, wq, k16), k16, ds)
    ref = gradient(x, x, wq, k16, ds)[2]
    assert float((got.double() - ref).norm()) <= budget(D) * float(ref.norm()), float((got.double() - ref).norm() / ref.norm() / U)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_projection_gradient_over_many_tokens(checkpoint):
    """dwq's error does not grow with the tokens: a tile of 16 leaves the tensor cores before the next (a chain over
    a warp's 228 tiles, which round towards zero, left 150 u here)."""
    M, D, NB = 1 << 17, 4096, 8
    x, wq, k16, ds = inputs(M, D, NB, torch.bfloat16, "cuda", seed=230)
    wq = wq.requires_grad_()
    got, = torch.autograd.grad(fsi.router_scores(x, wq, k16, checkpoint=checkpoint), wq, ds)
    xk = kept(x, checkpoint)
    ref = sum(gradient(*(t[a:a + 16384] for t in (x, xk)), wq, k16, ds[a:a + 16384])[1] for a in range(0, M, 16384))
    assert float((got.double() - ref).norm()) <= budget(D) * float(ref.norm()), float((got.double() - ref).norm() / ref.norm() / U)


# Widths whose rows of codes TMA cannot address: they go through the workspace as bf16, in pieces.
PIECES = [(40000, 1000, 24), (33568, 1000, 5), (33569, 1000, 5), (4200000, 8, 3)]


def test_workspace_of_unaligned_codes_stays_small():
    """A piece is at most 64 MB or an eighth of the codes (a sixteenth of the rows in bf16), not all of x in bf16."""
    __import__("importlib").import_module("foveal-sparse-indexer_b200.build").build()
    size = fsi.load_library().fp_router_scores_bwd_workspace_size
    for M, D in [(4096, 1000), (131072, 1000), (1 << 20, 1000), (1 << 20, 4104), (1 << 22, 8), (1 << 27, 8)]:
        codes, extra = M * D, size(1, M, D, 64, 1) - size(1, M, D, 64, 0)
        # and a set of partial sums of dwq a piece: 296 CTAs, 256 columns each, 16 sums of 4 bytes a column
        pieces = min(16, -(-codes // (32 << 20))) + 1
        assert 0 < extra <= max((64 << 20) + 512 * D, codes // 8 + 512 * D) + pieces * 296 * 256 * 64, (M, D, extra)
        assert size(1, M, D + 8, 64, 1) - size(1, M, D + 8, 64, 0) == 0  # addressable rows need none


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,NB", PIECES)
def test_gradient_from_unaligned_codes_in_pieces(M, D, NB):
    """More than one piece, and last pieces of one row, of a part of a tile and of all rows: dx is that of the uncopied
    input bit by bit, dwq and dk are the 64-bit formula's at the copy."""
    x, wq, k16, ds = inputs(M, D, NB, torch.bfloat16, "cuda", seed=240)
    got, plain = run(x, wq, k16, ds, "mxfp8"), run(x, wq, k16, ds, None)
    assert torch.equal(got[0], plain[0])
    check_norms(got[1:], gradient(x, kept(x, True), wq, k16, ds)[1:], torch.float32, budget(D))
    part = [t.clone().requires_grad_(i != 1) for i, t in enumerate((x, wq, k16))]  # no gradient for q_proj: one launch
    dx, = torch.autograd.grad(fsi.router_scores(*part, checkpoint="mxfp8"), part[0], ds)
    assert torch.equal(dx, got[0])
