"""Training operators on the GPU: MXFP8 activation copies, SwiGLU and router scores whose backward passes
read them, the balance loss with the blocks' counts, and the module's training step with all of them.

Every operator is compared with a plain 64-bit restatement on the same inputs.  Tolerances count roundings:
u = 2^-24 is half a step of fp32, ``half(t)`` half a step of an output type relative to its value, and the
bounds multiply u by the number of fp32 operations on the longest path and by the sum of the magnitudes that
go into a result (the standard linear bound of a sum in any order).
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from conftest import fsi, golden, rel_err  # noqa: F401

pytestmark = pytest.mark.gpu
kernels = fsi.kernels
DEV = "cuda"
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float32]


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def check(got, ref, tol, what=""):
    """|got - ref| <= tol elementwise; NaN where the reference has NaN."""
    g, r = got.double(), ref.double()
    nan = torch.isnan(r)
    assert torch.equal(torch.isnan(g), nan), what
    bad = ((g - r).abs() > tol) & ~nan & ~(g == r)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((g - r).abs() - tol)[bad].max()))


# ------------------------------------------------------------------ MXFP8 copies
def mx_ref(x):
    """(values, scale bytes) of the format, in 64 bits and from its definition."""
    v = x.detach().double().reshape(-1)
    n = v.numel()
    b = torch.zeros((n + 31) // 32 * 32, dtype=torch.float64, device=v.device)
    b[:n] = v
    b = b.view(-1, 32)
    fin = torch.isfinite(b)
    top = torch.where(fin, b, 0.0).abs().amax(dim=1)
    grid = torch.arange(-118, 121, device=v.device, dtype=torch.float64)
    fits = top[:, None] <= 448.0 * torch.exp2(grid)[None, :]
    k = torch.where(fits.any(dim=1), grid[fits.to(torch.uint8).argmax(dim=1)], 120.0)
    y = b / torch.exp2(k)[:, None]
    _, e = torch.frexp(torch.where(fin, y, 0.0))
    step = torch.exp2((e - 4).clamp_min(-9).double())  # 3 stored bits; subnormals below 2^-6
    q = torch.round(y / step) * step * torch.exp2(k)[:, None]
    q = q.clamp(-240.0 * 2.0 ** 120, 240.0 * 2.0 ** 120)  # 2^128 is past fp32's range
    q[~fin] = math.nan
    return q.reshape(-1)[:n].view(x.shape), (k + 127).to(torch.uint8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (31,), (32,), (33,), (0, 5), (3, 1001), (64, 320), (2, 3, 4097), (257, 64),
                                   (1, 8), (5, 17)])
def test_checkpoint_values(shape, dtype):
    x = randn(*shape, seed=3, dtype=dtype, scale=3.0)
    if x.numel() > 64:  # magnitudes over the whole range, wide channels next to small ones
        x = (x.float() * torch.exp2(torch.randint(-40, 40, shape, generator=gen(4), device=DEV).float())).to(dtype)
    c = fsi.checkpoint_mxfp8(x)
    y = c.restore()
    ref, byte = mx_ref(x)
    assert y.shape == x.shape and y.dtype == dtype
    assert torch.equal(y.double(), ref)
    assert torch.equal(c.scales, byte)
    assert c.codes.shape == x.shape and c.codes.dtype == torch.float8_e4m3fn
    assert c.nbytes == kernels.mxfp8_nbytes(x.numel())


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_borders(dtype):
    """Block maxima at and next to 448 * 2^k for every k, values half way between codes, and the clamps."""
    rows = []
    for k in range(-126, 119):
        for top in (448.0, 449.9, 446.0, 256.0, 255.0):
            r = torch.linspace(-1, 1, 32, dtype=torch.float64) * top * 2.0 ** k
            r[0] = top * 2.0 ** k
            rows.append(r)
    ties = torch.arange(32, dtype=torch.float64) * 0.5 + 16.5  # half steps of [16, 32): ties to even
    rows += [ties, -ties, torch.zeros(32, dtype=torch.float64), torch.full((32,), -0.0, dtype=torch.float64)]
    big = torch.finfo(dtype).max
    rows += [torch.full((32,), float(big), dtype=torch.float64), torch.full((32,), -float(big), dtype=torch.float64)]
    tiny = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    rows += [torch.full((32,), tiny, dtype=torch.float64), torch.linspace(0, 1, 32, dtype=torch.float64) * 2.0 ** -126]
    x = torch.stack(rows).to(DEV).to(dtype)
    c = fsi.checkpoint_mxfp8(x)
    ref, byte = mx_ref(x)
    assert torch.equal(c.scales, byte)
    assert torch.equal(c.restore().double(), ref)
    # every value within half a step of e4m3, or of its smallest step 2^-9 of the scale
    unit = torch.exp2(byte.double() - 127)[:, None]
    assert bool(((ref - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, unit * 2.0 ** -10)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_nonfinite(dtype):
    """NaN and infinities become NaN, and leave the block's other elements as they would be without them."""
    x = randn(40, 32, seed=5, dtype=dtype)
    y = x.clone()
    y[0, 3], y[1, 0], y[2, 31], y[3, :16], y[4] = math.inf, -math.inf, math.nan, math.inf, math.nan
    got = fsi.checkpoint_mxfp8(y).restore()
    hit = ~torch.isfinite(y)
    z = torch.where(hit, 0.0, x.float()).to(dtype)
    assert bool(torch.isnan(got[hit]).all())
    assert torch.equal(got[~hit].double(), mx_ref(z)[0][~hit])


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_strides_and_offsets(dtype):
    """Transposed, sliced and unaligned inputs are taken in row-major order of their values."""
    base = randn(70, 90, seed=6, dtype=dtype)
    flat = randn(1000, seed=7, dtype=dtype)
    for x in (base.t(), base[::2, 3:77], flat[1:], flat[3:131], base[:, :1], base[0].expand(5, 90)):
        assert torch.equal(fsi.checkpoint_mxfp8(x).restore().double(), mx_ref(x)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 15, 16, 33, 100, 1024, 4095, 5000])
def test_checkpoint_writes_nothing_else(n, dtype):
    """Bytes around the codes, the scales and the restored values stay as they were."""
    lib, dt = fsi.load_library(), 0 if dtype == torch.float32 else 1
    P = ctypes.c_void_p
    st = P(torch.cuda.current_stream().cuda_stream)
    x = randn(n, seed=8, dtype=dtype)
    codes = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full(((n + 31) // 32 + 64,), 0xAB, dtype=torch.uint8, device=DEV)
    y = torch.full((n + 64,), 7.0, dtype=dtype, device=DEV)
    assert lib.fp_mxfp8_quantize(P(x.data_ptr()), dt, n, P(codes.data_ptr() + 32), P(scales.data_ptr() + 31), st) == 0
    es = x.element_size()
    assert lib.fp_mxfp8_dequantize(P(codes.data_ptr() + 32), P(scales.data_ptr() + 31), dt, n,
                                   P(y.data_ptr() + 32 * es), st) == 0
    ref, byte = mx_ref(x)
    assert torch.equal(y[32:32 + n].double(), ref)
    assert torch.equal(scales[31:31 + byte.numel()], byte)
    for t, a, m, v in ((codes, 32, n, 0xAB), (scales, 31, byte.numel(), 0xAB), (y, 32, n, 7.0)):
        assert bool((t[:a] == v).all()) and bool((t[a + m:] == v).all())


# ------------------------------------------------------------------ SwiGLU on 8-bit copies
def swiglu_grads(g, u, dh):
    s = torch.sigmoid(g)
    return dh * u * s * (1 + g * (1 - s)), dh * g * s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 33), (64, 320), (17, 1001), (300, 512), (0, 64)])
def test_swiglu_checkpoint(shape, dtype):
    g = randn(*shape, seed=10, dtype=dtype, scale=4.0).requires_grad_()
    u = randn(*shape, seed=11, dtype=dtype).requires_grad_()
    dh = randn(*shape, seed=12, dtype=dtype, scale=1e-2)
    h = fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8")
    assert torch.equal(h, fsi.triton_fused_swiglu(g.detach(), u.detach()))  # the forward is the same
    dg, du = torch.autograd.grad(h, (g, u), dh)
    gq, uq = mx_ref(g)[0], mx_ref(u)[0]
    rg, ru = swiglu_grads(gq, uq, dh.double())
    # sigmoid: exp within 2 steps, a sum and a division -> 4 steps = 8 u of its value; 1 - s and the product
    # with g carry that times |g| s; seven more products and sums: below 32 u of the magnitudes' product
    s, d = torch.sigmoid(gq), dh.double().abs()
    check(dg, rg, half(dtype) * rg.abs() + 32 * U * d * uq.abs() * s * (1 + gq.abs()) + 1e-37)
    check(du, ru, half(dtype) * ru.abs() + 32 * U * d * gq.abs() * s + 1e-37)


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_checkpoint_extremes(dtype):
    """Saturated gates, zeros, and NaN or infinity in g or u, which the gradients show as NaN."""
    g = torch.tensor([-200.0, -88.0, -30.0, -1.278, 0.0, 1.0, 30.0, 88.0, 200.0] + [0.5] * 23, device=DEV).to(dtype)
    u = torch.linspace(-2, 2, 32, device=DEV).to(dtype)
    g, u = g.repeat(3, 1), u.repeat(3, 1)
    g[1, 2], g[1, 5], u[2, 7], u[2, 8] = math.nan, math.inf, math.nan, -math.inf
    dh = torch.ones_like(g)
    g.requires_grad_(), u.requires_grad_()
    dg, du = torch.autograd.grad(fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8"), (g, u), dh)
    gq, uq = mx_ref(g)[0], mx_ref(u)[0]
    rg, ru = swiglu_grads(gq, uq, dh.double())
    s = torch.sigmoid(gq)
    check(dg, rg, torch.nan_to_num(half(dtype) * rg.abs() + 32 * U * uq.abs() * s * (1 + gq.abs())) + 1e-36)
    check(du, ru, torch.nan_to_num(half(dtype) * ru.abs() + 32 * U * gq.abs() * s) + 1e-36)
    assert bool(torch.isnan(dg[1, 2]) and torch.isnan(du[1, 5]) and torch.isnan(dg[2, 8]) and not torch.isnan(du[2, 7]))


def test_swiglu_checkpoint_against_differences():
    """The gradient along a direction against central differences of the 64-bit formula at the copies' values."""
    g, u = randn(64, 96, seed=13).requires_grad_(), randn(64, 96, seed=14).requires_grad_()
    dh, vg, vu = (randn(64, 96, seed=s).double() for s in (15, 16, 17))
    dg, du = torch.autograd.grad(fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8"), (g, u), dh.float())
    gq, uq, d = mx_ref(g)[0], mx_ref(u)[0], dh.float().double()
    f = lambda e: float((d * torch.nn.functional.silu(gq + e * vg) * (uq + e * vu)).sum())
    e = 1e-4
    num = (f(e) - f(-e)) / (2 * e)
    got = float((dg.double() * vg + du.double() * vu).sum())
    # third derivative term e^2 / 6 * O(1) per element, fp32 roundings of the gradient
    mag = float((d.abs() * (vg.abs() * (1 + uq.abs()) + vu.abs() * (1 + gq.abs()))).sum())
    assert abs(num - got) <= (e * e + 64 * U) * mag


def test_swiglu_checkpoint_holds_half_the_bytes():
    g, u = (randn(1024, 1024, seed=s, dtype=torch.bfloat16).requires_grad_() for s in (18, 19))
    h = fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8")
    saved, = h.grad_fn.saved_tensors
    assert saved.numel() == 2 * (1024 * 1024 + 1024 * 1024 // 32)
    with torch.no_grad():
        assert fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8").grad_fn is None


def test_swiglu_checkpoint_mixed_inputs():
    """Strided inputs, u in another type, a gradient for one input only, an upstream gradient that is a view."""
    g = randn(96, 80, seed=20, dtype=torch.bfloat16).t().requires_grad_()
    u = randn(80, 96, seed=21)
    h = fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8")
    h.sum().backward()  # the upstream gradient is one expanded element
    gq, uq = mx_ref(g)[0], mx_ref(u.to(torch.bfloat16))[0]
    rg, _ = swiglu_grads(gq, uq, torch.ones((), dtype=torch.float64, device=DEV))
    s = torch.sigmoid(gq)
    check(g.grad, rg, half(torch.bfloat16) * rg.abs() + 32 * U * uq.abs() * s * (1 + gq.abs()))
    u.requires_grad_()
    du, = torch.autograd.grad(fsi.triton_fused_swiglu(g.detach(), u, checkpoint="mxfp8"), u, torch.ones_like(h))
    assert du.dtype == torch.float32
    with pytest.raises(ValueError):
        fsi.triton_fused_swiglu(g, u[:1], checkpoint="mxfp8")


# ------------------------------------------------------------------ router scores
EPS = 1.1920928955078125e-07


def router_ref(x, xq, wq, k16, ds):
    """(scores, dx, dwq, dk, and the magnitudes that bound each one's roundings)."""
    x, xq, wq, k16, ds = (t.detach().double() for t in (x, xq, wq, k16, ds))
    q = x @ wq.t()
    r = ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    n = q * r
    s = n @ k16.t() / 4
    a = ds @ k16 / 4
    dk = ds.t() @ n / 4
    dq = r * (a - n * (a * n).mean(dim=1, keepdim=True))
    N = r * (x.abs() @ wq.abs().t())          # magnitude behind a normalised query
    kap = 1 + (n.abs() * N).mean(dim=1, keepdim=True)  # r's relative error is D u times this
    A = ds.abs() @ k16.abs() / 4
    DQ = r * (A + N * (A * N).mean(dim=1, keepdim=True)) * kap * 3
    mag = ((N * kap) @ k16.abs().t() / 4, DQ @ wq.abs(), DQ.t() @ xq.abs(), ds.abs().t() @ (N * kap) / 4)
    # dq itself is held in two bf16 pieces for the tensor cores: 2^-16 of it
    mag2 = (0, dq.abs() @ wq.abs(), dq.abs().t() @ xq.abs(), 0)
    return (s, dq @ wq, dq.t() @ xq, dk), mag, mag2


def router_case(M, D, NB, dtype, seed=30, wdtype=None):
    x = randn(M, D, seed=seed, dtype=dtype)
    wq = randn(16, D, seed=seed + 1, dtype=wdtype or dtype, scale=D ** -0.5)
    k16 = randn(NB, 16, seed=seed + 2, dtype=wdtype or dtype, scale=0.25)
    ds = randn(M, NB, seed=seed + 3)
    return x, wq, k16, ds


def check_router(x, wq, k16, ds, checkpoint, got):
    dtype = x.dtype
    w, k = wq.to(dtype), k16.to(dtype)  # the kernels read the weights in x's type
    xq = mx_ref(x)[0] if checkpoint else x
    ref, mag, mag2 = router_ref(x, xq, w, k, ds)
    (M, D), NB = x.shape, k16.shape[0]
    split = 2.0 ** -16 if dtype == torch.bfloat16 else 0.0
    ops = (D + 64, D + NB + 64, D + NB + M + 64, D + M + 64)
    for name, o, r, m, m2, n in zip(("scores", "dx", "dwq", "dk"), got, ref, mag, mag2, ops):
        check(o, r, half(o.dtype) * r.abs() + n * U * m + split * m2 + 1e-37, name)


@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,NB", [(1, 8, 1), (1, 64, 16), (3, 72, 5), (16, 256, 16), (17, 264, 33), (64, 256, 224),
                                    (130, 1000, 65), (33, 512, 1024), (257, 1024, 130), (1000, 128, 12)])
def test_router_scores(M, D, NB, dtype, checkpoint):
    x, wq, k16, ds = router_case(M, D, NB, dtype)
    for t in (x, wq, k16):
        t.requires_grad_()
    s = fsi.router_scores(x, wq, k16, checkpoint=checkpoint)
    assert torch.equal(s, kernels.router_scores(x.detach(), wq.detach(), k16.detach())[0])
    grads = torch.autograd.grad(s, (x, wq, k16), ds)
    assert [g.dtype for g in grads] == [dtype] * 3
    check_router(x, wq, k16, ds, checkpoint, (s, *grads))


@pytest.mark.parametrize("D", [768, 2304, 4096, 8192])
def test_router_scores_are_the_inference_scores(D):
    """The training forward gives the same bits as fp_router_scores at wide inputs, and its 8-bit copy is
    checkpoint_mxfp8's, NaN and infinities included."""
    x, wq, k16, _ = router_case(75, D, 224, torch.bfloat16)
    x[3, 5], x[4, D - 1], x[60, 33] = math.nan, math.inf, -3e38
    ref = kernels.router_scores(x, wq, k16)[0]
    for keep in (False, True):
        s, _, buf = kernels.router_scores_train(x, wq, k16, keep_mxfp8=keep)
        assert torch.equal(torch.nan_to_num(s, nan=7.0), torch.nan_to_num(ref, nan=7.0))
        assert torch.equal(torch.isnan(s), torch.isnan(ref))
    c = fsi.checkpoint_mxfp8(x)
    n = x.numel()
    assert torch.equal(buf[:n], c.buffer[:n]) and torch.equal(buf[-n // 32:], c.scales)


def test_router_scores_partial_gradients():
    """Each subset of the inputs' gradients is that of all of them, bit by bit; leading dimensions, strides and
    weights of another type are taken."""
    x, wq, k16, ds = router_case(66, 192, 20, torch.bfloat16, wdtype=torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, wq, k16)]
    full = torch.autograd.grad(fsi.router_scores(*leaves), leaves, ds)
    assert [g.dtype for g in full] == [torch.bfloat16, torch.float32, torch.float32]
    check_router(x, wq, k16, ds, None, (fsi.router_scores(x, wq, k16), *full))
    for mask in range(1, 7):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, wq, k16))]
        want = [i for i in range(3) if mask >> i & 1]
        got = torch.autograd.grad(fsi.router_scores(*ts), [ts[i] for i in want], ds)
        assert all(torch.equal(g, full[i]) for g, i in zip(got, want))
    xt = x.view(3, 22, 192).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()  # strided [3, 22, 192]
    s = fsi.router_scores(xt, wq, k16)
    assert s.shape == (3, 22, 20)
    g, = torch.autograd.grad(s, xt, ds.view(3, 22, 20).transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(g.reshape(66, 192), full[0])
    mixed = (x.clone().requires_grad_(), wq.clone().requires_grad_(), k16.to(torch.bfloat16).requires_grad_())
    g = torch.autograd.grad(fsi.router_scores(*mixed), mixed, ds)
    assert [t.dtype for t in g] == [torch.bfloat16, torch.float32, torch.bfloat16]


@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_router_scores_no_tokens_and_zero_token(checkpoint):
    x, wq, k16, _ = router_case(0, 64, 8, torch.bfloat16)
    for t in (x, wq, k16):
        t.requires_grad_()
    s = fsi.router_scores(x, wq, k16, checkpoint=checkpoint)
    assert s.shape == (0, 8)
    g = torch.autograd.grad(s, (x, wq, k16), torch.zeros(0, 8, device=DEV))
    assert g[0].shape == (0, 64) and not bool(g[1].any()) and not bool(g[2].any())
    # a token of zeros has a zero query: eps keeps its factor finite
    x, wq, k16, ds = router_case(5, 64, 8, torch.float32)
    x[2] = 0
    x.requires_grad_()
    s = fsi.router_scores(x, wq, k16, checkpoint=checkpoint)
    dx, = torch.autograd.grad(s, x, ds)
    assert not bool(s[2].any())
    check(dx, router_ref(x, x, wq, k16, ds)[0][1], 1e-3 * router_ref(x, x, wq, k16, ds)[1][1])


def test_router_scores_nan_stays_in_its_token():
    x, wq, k16, ds = router_case(40, 256, 16, torch.bfloat16)
    x[7, 3] = math.nan
    x.requires_grad_()
    s = fsi.router_scores(x, wq, k16)
    dx, = torch.autograd.grad(s, x, ds)
    rows = torch.arange(40, device=DEV) == 7
    assert bool(torch.isnan(s[7]).all()) and bool(torch.isfinite(s[~rows]).all())
    assert bool(torch.isnan(dx[7]).all()) and bool(torch.isfinite(dx[~rows]).all())


def test_router_scores_against_differences():
    x, wq, k16, ds = router_case(48, 128, 20, torch.float32)
    for t in (x, wq, k16):
        t.requires_grad_()
    grads = torch.autograd.grad(fsi.router_scores(x, wq, k16), (x, wq, k16), ds)
    dirs = [randn(*t.shape, seed=40 + i).double() * t.detach().abs().mean().double() for i, t in enumerate((x, wq, k16))]
    base = [t.detach().double() for t in (x, wq, k16)]

    def f(e):
        a, b, c = (t + e * v for t, v in zip(base, dirs))
        q = a @ b.t()
        return float((ds.double() * (q * ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt() @ c.t() / 4)).sum())

    e = 1e-4
    num = (f(e) - f(-e)) / (2 * e)
    got = sum(float((g.double() * v).sum()) for g, v in zip(grads, dirs))
    mag = sum(float((g.double() * v).abs().sum()) for g, v in zip(grads, dirs))
    assert abs(num - got) <= (100 * e * e + 256 * U) * mag


# ------------------------------------------------------------------ balance loss
def balance_case(M, NB, base, cap, seed=50, spread=1.0):
    g = gen(seed)
    s = torch.randn(M, NB, generator=g, device=DEV) * spread + 0.5 * torch.randn(NB, generator=g, device=DEV)
    cap = min(cap, NB - base)
    idx = (torch.rand(M, NB - base, generator=g, device=DEV).topk(cap, dim=-1).indices + base).to(torch.int32)
    cnt = torch.randint(0, cap + 1, (M,), generator=g, device=DEV, dtype=torch.int32)
    return s, idx, cnt


def balance_ref(s, idx, cnt, base, T=1.0, valid=None, counts=None):
    M, NB = s.shape
    s = s.detach().double()
    ok = torch.ones(M, dtype=torch.bool, device=s.device) if valid is None else valid
    if counts is None:
        live = (torch.arange(idx.shape[1], device=s.device) < cnt[:, None]) & ok[:, None] & (idx >= 0) & (idx < NB)
        counts = torch.bincount(idx[live].long(), minlength=NB)
    z = s[:, base:] / T
    rows = ok & ~(z == -math.inf).all(dim=1)
    p = torch.where(rows[:, None], torch.softmax(z, dim=1), 0.0)
    n, R = max(1, int(rows.sum())), NB - base
    f = counts[base:].double() / max(1, int(counts.sum()))
    loss = R * (f * p.sum(dim=0)).sum() / n
    ds = torch.zeros_like(s)
    ds[:, base:] = p * (f - (p * f).sum(dim=1, keepdim=True)) * R / (T * n)
    if int(counts.sum()) == 0:
        ds.zero_()
    # magnitudes: exp's argument carries |z| u twice (division, difference), exp 2 steps, sums over NB
    # (scores of a mask's lowest value have p = 0 next to others and difference 0 among themselves)
    zmax = torch.where(z.abs() < 1e30, z.abs(), 0.0).amax(dim=1, keepdim=True)
    c = (4 * zmax + NB + 32) * U
    g = (f - 1.0 / R).abs() if int(counts.sum()) else torch.zeros_like(f)
    tol = torch.zeros_like(s)
    tol[:, base:] = p * (g + (p * g).sum(dim=1, keepdim=True)) * R / (T * n) * (c + 8 * U)
    tol_loss = float((R * (p * f) * (c + (M / 8 + 16) * U)).sum() / n) + U * float(loss)
    return loss, counts, ds, tol, tol_loss


def run_balance(s, idx, cnt, base, up=1.0, **kw):
    leaf = s.detach().clone().requires_grad_()
    loss, counts = fsi.balance_loss(leaf, idx, cnt, base_blocks=base, **kw)
    ds, = torch.autograd.grad(loss, leaf, torch.full((), up, device=DEV))
    return loss.detach(), counts, ds


def check_balance(s, idx, cnt, base, T=1.0, valid=None, up=1.0, **kw):
    loss, counts, ds = run_balance(s, idx, cnt, base, up=up, temperature=T, valid=valid, **kw)
    ref, rc, rds, tol, tl = balance_ref(s, idx, cnt, base, T, valid, kw.get("counts"))
    assert counts.dtype == torch.int64 and torch.equal(counts, rc)
    if not math.isnan(float(ref)):
        assert abs(float(loss) - float(ref)) <= tl, (float(loss), float(ref), tl)
    else:
        assert math.isnan(float(loss))
    check(ds, rds * up, torch.nan_to_num(tol) * abs(up) + U * torch.nan_to_num(rds).abs() * abs(up) + 1e-37)
    return loss, counts, ds


@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("M,NB,base,cap", [(1, 2, 0, 1), (1, 1, 0, 1), (5, 3, 2, 1), (7, 32, 1, 8), (64, 33, 4, 5), (129, 64, 0, 64),
                                           (512, 224, 4, 56), (300, 448, 8, 112), (100, 1000, 7, 20), (33, 1024, 0, 8),
                                           (9000, 20, 3, 4)])
def test_balance_loss(M, NB, base, cap, T):
    s, idx, cnt = balance_case(M, NB, base, cap)
    check_balance(s, idx, cnt, base, T, up=0.37)
    assert torch.equal(fsi.block_counts(idx, cnt, NB), balance_ref(s, idx, cnt, base)[1])


def test_balance_loss_masks():
    """Padding, rows with no score above -inf, partly masked rows, the type's lowest value as a mask, NaN in
    left-out rows, no valid row at all."""
    s, idx, cnt = balance_case(200, 40, 3, 6)
    valid = torch.rand(200, generator=gen(51), device=DEV) < 0.7
    check_balance(s, idx, cnt, 3, valid=valid)
    t = s.clone()
    t[5] = -math.inf                      # nothing left
    t[6, 3:] = -math.inf                  # only base blocks left
    t[7, 3:39] = -math.inf                # one block left
    t[8, 10:20] = torch.finfo(torch.float32).min
    t[9, 3:] = torch.finfo(torch.float32).min  # all alike: a distribution
    _, _, ds = check_balance(t, idx, cnt, 3)
    assert not bool(ds[5].any()) and not bool(ds[6].any())
    bad = torch.where(valid[:, None], t, math.nan)
    loss, _, ds = check_balance(bad, idx, cnt, 3, valid=valid)
    assert math.isfinite(float(loss)) and not bool(ds[~valid].any()) and bool(torch.isfinite(ds).all())
    bad = s.clone()
    bad[11, 0] = math.nan                 # a base block's score is not read
    check_balance(bad, idx, cnt, 3)
    none = torch.zeros(200, dtype=torch.bool, device=DEV)
    loss, counts, ds = check_balance(s, idx, cnt, 3, valid=none)
    assert float(loss) == 0.0 and not bool(counts.any()) and not bool(ds.any())


def test_balance_loss_nan_and_inf_show():
    s, idx, cnt = balance_case(50, 40, 3, 6)
    for v in (math.nan, math.inf):
        t = s.clone()
        t[4, 9] = v
        loss, _, ds = run_balance(t, idx, cnt, 3)
        assert math.isnan(float(loss)) and bool(torch.isnan(ds[4, 3:]).all()) and not bool(ds[4, :3].any())
    t = s.clone()
    t[4] = math.nan
    assert math.isnan(float(run_balance(t, idx, cnt, 3)[0]))


def test_balance_loss_route_lists():
    """Empty lists, counts past the capacity or below zero, ids out of range (skipped), an id named twice, int64."""
    s, idx, cnt = balance_case(64, 40, 3, 6)
    loss, counts, ds = check_balance(s, idx, torch.zeros_like(cnt), 3)
    assert float(loss) == 0.0 and not bool(counts.any()) and not bool(ds.any())
    empty = torch.zeros(64, 0, dtype=torch.int32, device=DEV)
    assert not bool(fsi.block_counts(empty, cnt, 40).any())
    check_balance(s, empty, cnt, 3)
    wild = cnt.clone()
    wild[0], wild[1], wild[2] = 1000000, -5, 6
    check_balance(s, idx, wild, 3)
    ids = idx.clone()
    ids[3, 0], ids[4, 1], ids[5, 2], ids[6, 0] = -1, 40, 2 ** 31 - 1, -2 ** 31
    check_balance(s, ids, torch.full_like(cnt, 6), 3)
    ids = idx.clone()
    ids[:, 1] = ids[:, 0]
    ids[7] = 1                              # a base block named by the lists
    check_balance(s, ids, cnt, 3)
    a, b = run_balance(s, idx, cnt, 3), run_balance(s, idx.long(), cnt.long(), 3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    far, n = idx.long(), cnt.long()  # 64-bit values that would wrap into range
    far[0, 0], far[1, 0], n[2] = 2 ** 32 + 5, -2 ** 32 + 5, 2 ** 32
    check_balance(s, far, n, 3)


def test_balance_loss_even_load_and_collapse():
    """Uniform scores and an even load give 1 and no gradient; one block with all slots and all mass gives R."""
    M, R = 64, 16
    s = torch.zeros(M, R, device=DEV)
    idx = torch.arange(M, device=DEV, dtype=torch.int32)[:, None] % R
    one = torch.ones(M, dtype=torch.int32, device=DEV)
    loss, _, ds = run_balance(s, idx, one, 0)
    assert float(loss) == 1.0 and not bool(ds.any())
    s[:, 3] = 200.0
    loss, counts, _ = run_balance(s, torch.full_like(idx, 3), one, 0)
    assert float(loss) == R and int(counts[3]) == M


def test_balance_loss_given_counts():
    """Counts summed over shards replace the lists'; the lists may be left out."""
    s, idx, cnt = balance_case(100, 40, 3, 6)
    parts = [fsi.block_counts(idx[a:b], cnt[a:b], 40) for a, b in ((0, 37), (37, 100))]
    total = parts[0] + parts[1]
    a = run_balance(s, idx, cnt, 3)
    b = run_balance(s, None, None, 3, counts=total)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    big = total * 10_000_000_000  # 64-bit counts
    loss, counts, ds = run_balance(s, None, None, 3, counts=big)
    assert torch.equal(counts, big) and abs(float(loss) - float(a[0])) <= 4 * U * float(a[0])
    huge = total * 10 ** 15  # their products with the number of blocks pass 64 bits
    check(run_balance(s, None, None, 3, counts=huge)[2], a[2], 8 * U * a[2].abs())
    check(ds, a[2], 8 * U * a[2].abs())


def test_balance_loss_shapes_types_strides():
    s, idx, cnt = balance_case(60, 24, 2, 5)
    flat = run_balance(s, idx, cnt, 2)
    loss, counts, ds = run_balance(s.view(3, 20, 24), idx.view(3, 20, 5), cnt.view(3, 20), 2)
    assert ds.shape == (3, 20, 24)
    assert torch.equal(loss, flat[0]) and torch.equal(counts, flat[1]) and torch.equal(ds.view(60, 24), flat[2])
    leaf = s.t().contiguous().requires_grad_()
    loss, _ = fsi.balance_loss(leaf.t(), idx.t().contiguous().t(), cnt, base_blocks=2)
    g, = torch.autograd.grad(loss, leaf)
    assert torch.equal(g.t(), flat[2])
    pad = torch.zeros(61 * 24 + 1, device=DEV)
    pad[1:1 + 60 * 24] = s.reshape(-1)
    leaf = pad[1:1 + 60 * 24].view(60, 24).requires_grad_()  # not 16-byte aligned
    loss, _ = fsi.balance_loss(leaf, idx, cnt, base_blocks=2)
    assert torch.equal(loss.detach(), flat[0]) and torch.equal(torch.autograd.grad(loss, leaf)[0], flat[2])
    leaf = s.to(torch.bfloat16).requires_grad_()
    loss, _ = fsi.balance_loss(leaf, idx, cnt, base_blocks=2)
    g, = torch.autograd.grad(loss, leaf)
    ref = run_balance(leaf.detach().float(), idx, cnt, 2)
    assert torch.equal(loss.detach(), ref[0]) and torch.equal(g, ref[2].to(torch.bfloat16))
    empty = run_balance(s[:0], idx[:0], cnt[:0], 2)
    assert float(empty[0]) == 0.0 and not bool(empty[1].any()) and empty[2].shape == (0, 24)


def test_balance_loss_against_differences():
    s, idx, cnt = balance_case(40, 30, 2, 6)
    _, _, ds = run_balance(s, idx, cnt, 2, temperature=0.7)
    v, e = randn(40, 30, seed=55).double(), 1e-4
    f = lambda x: float(balance_ref(x, idx, cnt, 2, 0.7)[0])
    num = (f(s.double() + e * v) - f(s.double() - e * v)) / (2 * e)
    mag = float((ds.double() * v).abs().sum())
    assert abs(num - float((ds.double() * v).sum())) <= (100 * e * e + 256 * U) * mag


# ------------------------------------------------------------------ offsets past 32 bits
def test_checkpoint_past_32_bits():
    n = 2 ** 31 + 4096 + 37
    x = torch.empty(n, dtype=torch.bfloat16, device=DEV)
    x[:1000] = 1.5
    x[1000:-5000] = 0
    tail = randn(5000 - 5000 % 32 + 37, seed=120, dtype=torch.bfloat16)  # from a block's border to the end
    x[-tail.numel():] = tail
    c = fsi.checkpoint_mxfp8(x)
    y = c.restore()
    assert torch.equal(y[-tail.numel():].double(), mx_ref(tail)[0])
    assert bool((y[:1000] == 1.5).all()) and not bool(y[1000:-tail.numel()].any())
    del x, y, c
    torch.cuda.empty_cache()


def test_swiglu_past_32_bits():
    n = 2 ** 31 + 64
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    u = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    tg, tu, td = (randn(96, seed=s, dtype=torch.bfloat16) for s in (121, 122, 123))
    g[-96:], u[-96:] = tg, tu
    h, buf = kernels.swiglu_fwd_mxfp8(g, u)
    ht, bt = kernels.swiglu_fwd_mxfp8(tg, tu)
    assert torch.equal(h[-96:], ht) and not bool(h[:-96].any())
    del h
    g.zero_()
    g[-96:] = td
    dg, du, _ = kernels.swiglu_bwd_mxfp8(g, buf)
    rg, ru, _ = kernels.swiglu_bwd_mxfp8(td, bt)
    assert torch.equal(dg[-96:], rg) and torch.equal(du[-96:], ru) and not bool(dg[:-96].any())
    del g, u, dg, du, buf
    torch.cuda.empty_cache()


@pytest.mark.parametrize("checkpoint", [None, "mxfp8"])
def test_router_past_32_bits(checkpoint):
    """A row's scores and input gradient do not depend on the rows before it, and zero rows add nothing to the
    weights' gradients."""
    M, D, NB, last = 2 ** 19 + 70, 4096, 8, 70
    x = torch.zeros(M, D, dtype=torch.bfloat16, device=DEV)
    t, wq, k16, dt = router_case(last, D, NB, torch.bfloat16, seed=124)
    x[-last:] = t
    ds = torch.zeros(M, NB, device=DEV)
    ds[-last:] = dt
    s, saved, buf = kernels.router_scores_train(x, wq, k16, keep_mxfp8=checkpoint is not None)
    st, saved_t, buf_t = kernels.router_scores_train(t, wq, k16, keep_mxfp8=checkpoint is not None)
    assert torch.equal(s[-last:], st) and not bool(s[:-last].any())
    a = kernels.router_scores_bwd(ds, None if buf is not None else x, buf, wq, k16, saved, torch.bfloat16)
    b = kernels.router_scores_bwd(dt, None if buf is not None else t, buf_t, wq, k16, saved_t, torch.bfloat16)
    assert torch.equal(a[0][-last:], b[0]) and not bool(a[0][:-last].any())
    ref, mag, mag2 = router_ref(t, mx_ref(t)[0] if checkpoint else t, wq, k16, dt)
    for i in (1, 2):
        r = ref[i + 1]
        check(a[i], r, half(torch.bfloat16) * r.abs() + (D + NB + last + 64) * U * mag[i + 1] + 2.0 ** -16 * mag2[i + 1])
    del x, ds, s, saved, buf, a
    torch.cuda.empty_cache()


def test_balance_past_32_bits():
    M, NB, last = 2 ** 21 + 21, 1024, 37
    s = torch.zeros(M, NB, device=DEV)
    t, idx, cnt = balance_case(last, NB, 4, 8, seed=125)
    s[-last:] = t
    ids = torch.zeros(M, 8, dtype=torch.int32, device=DEV)
    ids[-last:] = idx
    n = torch.zeros(M, dtype=torch.int32, device=DEV)
    n[-last:] = cnt
    valid = torch.zeros(M, dtype=torch.bool, device=DEV)
    valid[-last:] = True
    loss, counts, state = kernels.balance_loss_fwd(s, ids, n, NB, 4, 1.0, valid)
    ref, rc, rds, tol, tl = balance_ref(t, idx, cnt, 4)
    assert torch.equal(counts, rc) and abs(float(loss) - float(ref)) <= tl
    ds = kernels.balance_loss_bwd(s, 4, 1.0, valid, state, torch.ones((), device=DEV))
    check(ds[-last:], rds, tol + U * rds.abs() + 1e-37)
    assert not bool(ds[:-last].any())
    del s, ds, ids
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ streams, graphs, determinism
def step(x, wq, k16, idx, cnt, g, u, dh):
    """One pass through all operators: loss, counts and gradients."""
    s = fsi.router_scores(x, wq, k16, checkpoint="mxfp8")
    loss, counts = fsi.balance_loss(s, idx, cnt, base_blocks=2)
    h = fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8")
    c = fsi.checkpoint_mxfp8(x.detach()).restore()
    grads = torch.autograd.grad([loss, h], [x, wq, k16, g, u], [torch.ones_like(loss), dh])
    return [loss.detach(), counts, h.detach(), c, *grads]


def step_inputs(seed, M=500, D=768, NB=70):
    x, wq, k16, _ = router_case(M, D, NB, torch.bfloat16, seed=seed)
    _, idx, cnt = balance_case(M, NB, 2, 9, seed=seed)
    g, u, dh = (randn(M, 192, seed=seed + i, dtype=torch.bfloat16) for i in (5, 6, 7))
    for t in (x, wq, k16, g, u):
        t.requires_grad_()
    return [x, wq, k16, idx, cnt, g, u, dh]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_repeatable_and_on_two_streams():
    """Bitwise the same every time, also when two passes run at once on streams of their own."""
    ins = [step_inputs(60), step_inputs(70)]
    ref = [step(*i) for i in ins]
    torch.cuda.synchronize()
    assert same(step(*ins[0]), ref[0])
    streams = [torch.cuda.Stream() for _ in ins]
    for _ in range(4):
        outs = []
        for st, i in zip(streams, ins):
            with torch.cuda.stream(st):
                outs.append(step(*i))
        torch.cuda.synchronize()
        assert same(outs[0], ref[0]) and same(outs[1], ref[1])


def test_captured_and_replayed():
    """Two graphs hold passes of their own; replays follow the inputs' new values, in either order."""
    a, b = step_inputs(80), step_inputs(90, M=300, D=512, NB=40)
    ref = {id(i): step(*i) for i in (a, b)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*a), step(*b)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in (a, b):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(*i))
        graphs.append(gr)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        assert same(outs[0], ref[id(a)]) and same(outs[1], ref[id(b)])
    new = step_inputs(100)
    with torch.no_grad():
        for dst, src in zip(a, new):
            dst.copy_(src)
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert same(outs[0], step(*new)) and same(outs[1], ref[id(b)])


def test_captured_while_an_eager_graph_lives():
    """A pass captured on leaves of its own (the same memory) while an eager graph of the originals is alive; both
    give what they give alone.  (On the originals themselves PyTorch's accumulation nodes, which keep the eager
    graph's stream, end the capture with an error, whatever the operator.)"""
    ins = step_inputs(130)
    ref = step(*ins)
    x, wq, k16, idx, cnt, g, u, dh = ins
    loss, _ = fsi.balance_loss(fsi.router_scores(x, wq, k16), idx, cnt, base_blocks=2)
    h = fsi.triton_fused_swiglu(g, u, checkpoint="mxfp8")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*[t.detach().requires_grad_(t.requires_grad) for t in ins])
    graph.replay()
    torch.cuda.synchronize()
    assert same(out, ref)
    torch.autograd.backward([loss, h], [torch.ones_like(loss), dh])
    assert torch.equal(g.grad, ref[7]) and torch.equal(u.grad, ref[8]) and torch.equal(x.grad, ref[4])
    graph.replay()
    torch.cuda.synchronize()
    assert same(out, ref)


def test_two_host_threads():
    """Two threads with streams of their own give what each gives alone."""
    import threading

    ins = [step_inputs(60), step_inputs(70, M=333, D=520, NB=65)]
    ref = [step(*i) for i in ins]
    torch.cuda.synchronize()
    ok = [True, True]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                out = step(*ins[k])
                torch.cuda.current_stream().synchronize()
                ok[k] = ok[k] and same(out, ref[k])

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(ok)


def test_another_current_device(monkeypatch):
    """Where another device is current, a call makes its tensors' device current first (each wrapper's own branch;
    one GPU here, so the question is answered yes once per call)."""
    ins = step_inputs(60)
    ref = step(*ins)
    seen = []

    def once_elsewhere(device):
        seen.append(device)
        return len(seen) % 2 == 1

    monkeypatch.setattr(fsi._lib, "elsewhere", once_elsewhere)
    assert same(step(*ins), ref)
    assert len(seen) == 2 * 8  # forward and backward of three operators, copy and restore


def test_double_backward_refused():
    x, wq, k16, ds = router_case(4, 64, 8, torch.float32)
    x.requires_grad_()
    g, = torch.autograd.grad(fsi.router_scores(x, wq, k16), x, ds, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ------------------------------------------------------------------ the module
def make_mlp(dtype, checkpoint, D=256, Np=1024, base=2, remote=4):
    torch.manual_seed(0)
    m = fsi.FovealPattentionMLP(D, Np, base_blocks=base, remote_blocks=remote, dtype=dtype, checkpoint=checkpoint,
                                top_p=0.9, min_remote_blocks=1, max_remote_blocks=5)
    with torch.no_grad():
        m.out_proj_16d.weight.mul_(30)
        m.block_keys_16d.mul_(3)
    return m.to(DEV).train()


def pooled_grads_ref(m, x, xq, dy, active):
    """The training forward's gradients in 64 bits: products that read the kept input at ``xq``."""
    P = {n: p.detach().double() for n, p in m.named_parameters()}
    x, xq, dy = x.double(), xq.double(), dy.double()
    rows = (active.long()[:, None] * 64 + torch.arange(64, device=x.device)).flatten()
    kg, ku, v = (P[n][rows] for n in ("k_gate", "k_up", "v"))
    G, U_ = xq @ kg.t(), xq @ ku.t()
    s = torch.sigmoid(G)
    dH = dy @ v.t()
    dG, dU = dH * U_ * s * (1 + G * (1 - s)), dH * G * s
    wq, k16, wo = P["q_proj_16d.weight"], P["block_keys_16d"], P["out_proj_16d.weight"]
    q = x @ wq.t()
    r = ((q * q).mean(dim=1, keepdim=True) + EPS).rsqrt()
    n = q * r
    soft = torch.softmax(n @ k16.t() / 4 / m.temperature, dim=1)
    dctx = dy @ wo
    dsoft = dctx @ k16.t()
    dS = soft * (dsoft - (dsoft * soft).sum(dim=1, keepdim=True)) / m.temperature
    a = dS @ k16 / 4
    dq = r * (a - n * (a * n).mean(dim=1, keepdim=True))
    out = {"x": dG @ kg + dU @ ku + dq @ wq, "q_proj_16d.weight": dq.t() @ xq,
           "block_keys_16d": soft.t() @ dctx + dS.t() @ n / 4, "out_proj_16d.weight": dy.t() @ (soft @ k16)}
    for name, d in (("k_gate", dG.t() @ xq), ("k_up", dU.t() @ xq), ("v", (G * s * U_).t() @ dy)):
        out[name] = torch.zeros_like(P[name]).index_copy_(0, rows, d)
    return out


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
def test_module_checkpoint_gradients(dtype, tol):
    """checkpoint="mxfp8": the forward is unchanged, the gradients are those at the kept copy (to the module's
    own parity bounds, relative to each gradient's norm)."""
    plain, m = make_mlp(dtype, None), make_mlp(dtype, "mxfp8")
    x = randn(3, 37, 256, seed=110, dtype=dtype).requires_grad_()
    dy = randn(3, 37, 256, seed=111, dtype=dtype)
    y, info = m(x, return_router_info=True)
    with torch.no_grad():
        assert torch.equal(y, plain.train()(x.detach()))
    y.backward(dy)
    ref = pooled_grads_ref(m, x.detach().reshape(-1, 256), mx_ref(x.detach().reshape(-1, 256))[0],
                           dy.reshape(-1, 256), info["active_blocks"])
    got = {n: p.grad for n, p in m.named_parameters()}
    got["x"] = x.grad.reshape(-1, 256)
    for name, r in ref.items():
        assert rel_err(got[name], r) <= tol, (name, rel_err(got[name], r))


def test_module_balance_loss():
    """The module's loss is the operators' composition, and reaches the router only."""
    m = make_mlp(torch.float32, None)
    x = randn(2, 50, 256, seed=112).requires_grad_()
    valid = torch.ones(2, 50, dtype=torch.bool, device=DEV)
    valid[1, 31:] = False
    loss, counts = m.balance_loss(x, valid)
    tok = fsi.FovealPattentionMLP(256, 1024, base_blocks=2, remote_blocks=4, dtype=torch.float32, routing="token",
                                  top_p=0.9, min_remote_blocks=1, max_remote_blocks=5).to(DEV).eval()
    tok.load_state_dict(m.state_dict())
    with torch.no_grad():
        _, info = tok(x.detach(), return_router_info=True)
    scores = m.compute_router_scores(x.detach()).reshape(100, 16)
    ref, rc, rds, tol, tl = balance_ref(scores, info["remote_indices"], info["remote_counts"], 2,
                                        valid=valid.reshape(-1))
    assert torch.equal(counts, rc) and abs(float(loss.detach()) - float(ref)) <= tl
    loss.backward()
    assert m.k_gate.grad is None and m.out_proj_16d.weight.grad is None
    r, mag, _ = router_ref(x.reshape(-1, 256), x.reshape(-1, 256), m.q_proj_16d.weight, m.block_keys_16d, rds)
    assert rel_err(x.grad.reshape(-1, 256), r[1]) <= 1e-4
    assert rel_err(m.q_proj_16d.weight.grad, r[2]) <= 1e-4
    assert rel_err(m.block_keys_16d.grad, r[3]) <= 1e-4
    assert not bool(x.grad[1, 31:].any())


def test_module_balance_loss_edges():
    m = make_mlp(torch.bfloat16, "mxfp8")
    loss, counts = m.balance_loss(torch.zeros(0, 256, dtype=torch.bfloat16, device=DEV))
    assert float(loss.detach()) == 0.0 and not bool(counts.any())
    loss, counts = m.balance_loss(randn(256, seed=115))  # one token, another type
    assert loss.shape == () and int(counts.sum()) >= 1
    m.checkpoint = "fp4"
    with pytest.raises(ValueError):
        m(randn(4, 256, seed=116, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        m.balance_loss(randn(4, 256, seed=116, dtype=torch.bfloat16))
    del m.__dict__["checkpoint"]  # as in a module saved whole before the attribute existed
    m(randn(4, 256, seed=116, dtype=torch.bfloat16)).sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
def test_training_step_of_all(dtype):
    """A training step as a program makes it: output loss plus balance loss on kept 8-bit inputs, gradients that
    are the sum of the two losses' own, and weights that move by them; a second step runs on the new weights."""
    m = make_mlp(dtype, "mxfp8")
    x = randn(4, 33, 256, seed=113, dtype=dtype)
    target = randn(4, 33, 256, seed=114, dtype=dtype)
    out_loss = lambda: (m(x).float() - target.float()).pow(2).mean()
    m.zero_grad()
    out_loss().backward()
    a = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    loss, counts = m.balance_loss(x)
    (0.01 * loss).backward()
    b = {n: p.grad.clone() if p.grad is not None else torch.zeros_like(p) for n, p in m.named_parameters()}
    assert bool(b["q_proj_16d.weight"].any()) and bool(b["block_keys_16d"].any())
    m.zero_grad()
    loss, _ = m.balance_loss(x)
    (out_loss() + 0.01 * loss).backward()
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    for n, p in m.named_parameters():
        s = a[n].double() + b[n].double()
        check(p.grad, s, half(dtype) * s.abs() + 1e-37, n)
    opt.step()
    if dtype == torch.float32:  # a bf16 weight may round a small step away
        assert all(not torch.equal(p, before[n]) for n, p in m.named_parameters())
    opt.zero_grad()
    (out_loss() + 0.01 * m.balance_loss(x)[0]).backward()
    assert all(bool(torch.isfinite(p.grad).all()) for p in m.parameters())
    assert int(counts.sum()) >= 4 * 33


def check_balance_by_differences(s, idx, cnt, base, T):
    """Against the reference with the tolerance of scores whose largest is 0: p depends on differences only."""
    loss, counts, ds = run_balance(s, idx, cnt, base, temperature=T)
    top = s[:, base:].amax(dim=1, keepdim=True)
    shifted = s.double() - torch.where(top.isfinite(), top, 0.0).double()
    ref, rc, rds, _, _ = balance_ref(s, idx, cnt, base, T)
    z = shifted[:, base:] / T
    # exp2's argument: |z| steps of c, of the difference and of the product; beyond 150 p is below 2^-200
    zmax = torch.where(z.abs() < 150, z.abs(), 0.0).amax(dim=1, keepdim=True)
    rows = ~(s[:, base:] == -math.inf).all(dim=1)
    p = torch.where(rows[:, None], torch.softmax(z, dim=1), 0.0)
    R, n, M = s.shape[1] - base, int(rows.sum()), s.shape[0]
    f = counts[base:].double() / int(counts.sum())
    g, c = (f - 1.0 / R).abs(), 4 * zmax + s.shape[1] + 40
    tol = torch.zeros_like(rds)
    tol[:, base:] = p * (g + (p * g).sum(dim=1, keepdim=True)) * R / (T * n) * c * U
    assert torch.equal(counts, rc)
    assert abs(float(loss) - float(ref)) <= float((R * p * f * (c + M / 8 + 16)).sum() / n) * U + U * float(ref)
    check(ds, rds, tol + U * rds.abs() + 1e-37)


@pytest.mark.parametrize("at", [0.0, 2.0 ** 18, -2.0 ** 20, 2.0 ** 22, -2.0 ** 40, 1e12, -1e30, 2.0 ** 105, -2.0 ** 120])
@pytest.mark.parametrize("unit", [False, True])
def test_balance_loss_large_scores(at, unit):
    """Rows whose scores are all large, a few steps of fp32 apart: temperature 1, and the temperature of one step."""
    M, NB, base = 90, 100, 3
    s, idx, cnt = balance_case(M, NB, base, 6)
    k = torch.randint(0, 5, (M, NB), generator=gen(61), device=DEV).double()
    step = max(torch.finfo(torch.float32).eps * 2 * abs(at), 2.0 ** -23)
    s = (at + k * step).float()
    s[:, :base] = 7.0
    s[5, 10:60] = -math.inf
    s[6, base:] = -math.inf
    s[7, 20] += 8 * step
    T = 1.0 if unit else step
    check_balance_by_differences(s, idx, cnt, base, T)


@pytest.mark.parametrize("T", [1e-30, 1e-6, 1e8, 1e30])
def test_balance_loss_extreme_temperatures(T):
    """Smallest: one block takes each row.  Largest: all alike, and finfo.min still a mask."""
    s, idx, cnt = balance_case(70, 100, 2, 6)
    s[3, 5:90] = -math.inf
    s[4] = -math.inf
    s[5, 40:] = torch.finfo(torch.float32).min
    check_balance_by_differences(s, idx, cnt, 2, T)
