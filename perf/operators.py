"""Measured cases of the training operators of a routed parameter-block layer.

Four operators: a tensor kept in 8 bits from the forward to the backward pass and read back (``checkpoint``),
SwiGLU whose backward reads such copies (``swiglu``), the 16-D router's scores with their gradient
(``router``) and the load-balance loss over the routed blocks with the blocks' counts (``balance``).  A pass
of the last three is a forward and its backward.

8-bit copies are MXFP8: blocks of 32 consecutive elements in row-major order share a power of two 2^k, the
smallest with max|x| <= 448 * 2^k over the block's finite elements (k in [-118, 120]); elements are e4m3,
rounded to nearest even, infinities held as NaN.
"""

import math

import torch

own = False

EPS = 1.1920928955078125e-07  # of the router's RMS norm
DEVICE = "cuda"


def _case(name, op, **kw):
    return dict(name=name, op=op, **kw)


def listed():
    return [
        # the layer input of the small fp32 configuration (4 x 128 tokens, width 512)
        _case("checkpoint-512x512-fp32", "checkpoint", rows=512, cols=512, dtype="fp32"),
        # the layer input of the 8B training step: 8 x 2048 tokens, width 4096
        _case("checkpoint-16384x4096", "checkpoint", rows=16384, cols=4096, dtype="bf16"),
        # packed sequences of odd total length through a layer of odd width
        _case("checkpoint-20011x1001", "checkpoint", rows=20011, cols=1001, dtype="bf16"),
        # the gradient test's step: 64 tokens, 5 active blocks of 64 channels
        _case("swiglu-64x320", "swiglu", rows=64, cols=320, dtype="bf16"),
        # pooled training at the 8B batch: 4 + 20 active blocks of 64 channels
        _case("swiglu-16384x1536", "swiglu", rows=16384, cols=1536, dtype="bf16"),
        # the dense MLP of the 8B configuration: every channel of 16384 tokens
        _case("swiglu-16384x14336", "swiglu", rows=16384, cols=14336, dtype="bf16"),
        # the gradient test's router in fp32
        _case("router-64x256x16-fp32", "router", rows=64, cols=256, blocks=16, dtype="fp32", mxfp8=False),
        # the 8B configuration's router over one training batch
        _case("router-16384x4096x224", "router", rows=16384, cols=4096, blocks=224, dtype="bf16", mxfp8=False),
        # the 70B configuration's router, its input kept in 8 bits for the backward pass
        _case("router-16384x8192x448-mxfp8", "router", rows=16384, cols=8192, blocks=448, dtype="bf16", mxfp8=True),
        # the small configuration: 512 tokens, 32 blocks of which one is always on, at most 8 routed
        _case("balance-512x32", "balance", rows=512, blocks=32, base=1, kmin=2, kmax=8, temperature=1.0, padded=False),
        # the 8B configuration's routes with padded sequences
        _case("balance-16384x224", "balance", rows=16384, blocks=224, base=4, kmin=8, kmax=56, temperature=1.0,
              padded=True),
        # the 70B configuration's routes over four batches at once, odd token count, sharper softmax
        _case("balance-65521x448", "balance", rows=65521, blocks=448, base=8, kmin=16, kmax=112, temperature=0.7,
              padded=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["checkpoint", "swiglu", "router", "balance"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("checkpoint", "swiglu"):
        cols = _log(rng, 8, 16384)
        if rng.random() < 0.4:
            cols = max(1, cols // 64) * 64
        rows = _log(rng, 1, min(65536, (1 << 26) // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype)
    if op == "router":
        cols = 8 * _log(rng, 8, 1024)
        if rng.random() < 0.4:
            cols = max(1, cols // 256) * 256
        rows = _log(rng, 1, min(65536, (1 << 26) // cols))
        return dict(op=op, rows=rows, cols=cols, blocks=_log(rng, 2, 1024), dtype=dtype, mxfp8=rng.random() < 0.5)
    blocks = _log(rng, 4, 1024)
    base = rng.randint(0, min(8, blocks - 2))
    kmax = rng.randint(1, min(128, blocks - base))
    rows = _log(rng, 1, min(131072, (1 << 25) // blocks))
    return dict(op=op, rows=rows, blocks=blocks, base=base, kmin=rng.randint(0, kmax), kmax=kmax,
                temperature=rng.choice([1.0, 0.7, 2.0]), padded=rng.random() < 0.5)


def _dtype(case):
    return torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16


def _activations(gen, rows, cols, dtype):
    """Normal values with a few wide channels, as hidden states have them."""
    wide = torch.exp(1.2 * torch.randn(cols, generator=gen, device=DEVICE)).clamp_(0.3, 20.0)
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    return x.mul_(wide).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op, dt = case["op"], _dtype(case)
    st = {"case": case}
    if op == "checkpoint":
        st["x"] = _activations(gen, case["rows"], case["cols"], dt)
    elif op == "swiglu":
        shape = (case["rows"], case["cols"])
        st["g"] = torch.randn(shape, generator=gen, device=DEVICE).mul_(2.0).to(dt).requires_grad_()
        st["u"] = torch.randn(shape, generator=gen, device=DEVICE).to(dt).requires_grad_()
        st["dh"] = torch.randn(shape, generator=gen, device=DEVICE).mul_(1e-2).to(dt)
    elif op == "router":
        M, D, NB = case["rows"], case["cols"], case["blocks"]
        st["x"] = _activations(gen, M, D, dt).requires_grad_()
        st["wq"] = (torch.randn(16, D, generator=gen, device=DEVICE) * D ** -0.5).to(dt).requires_grad_()
        st["k16"] = (torch.randn(NB, 16, generator=gen, device=DEVICE) * 0.25).to(dt).requires_grad_()
        st["ds"] = torch.randn(M, NB, generator=gen, device=DEVICE) * 1e-2
    else:
        M, NB, base, kmax = case["rows"], case["blocks"], case["base"], case["kmax"]
        s = torch.randn(M, NB, generator=gen, device=DEVICE)
        s += 0.5 * torch.randn(NB, generator=gen, device=DEVICE)  # blocks the router prefers
        st["s"] = s.requires_grad_()
        noise = s.detach()[:, base:] + torch.rand(M, NB - base, generator=gen, device=DEVICE)
        st["idx"] = (noise.topk(kmax, dim=-1).indices + base).to(torch.int32)
        st["cnt"] = torch.randint(case["kmin"], kmax + 1, (M,), generator=gen, device=DEVICE, dtype=torch.int32)
        st["valid"] = None
        if case["padded"]:  # sequences of up to 256 tokens, padded behind their last one
            last = torch.randint(64, 257, ((M + 255) // 256,), generator=gen, device=DEVICE)
            pos = torch.arange(M, device=DEVICE)
            st["valid"] = (pos % 256) < last[pos // 256]
        st["dloss"] = torch.full((), 0.01, device=DEVICE)
    return st


# ------------------------------------------------------------------ plain forms
def _mxfp8(x):
    """The values that x's 8-bit copy stands for, in 32 bits."""
    flat = x.detach().reshape(-1).float()
    n = flat.numel()
    pad = (-n) % 32
    b = torch.nn.functional.pad(flat, (0, pad)).view(-1, 32)
    finite = torch.isfinite(b)
    amax = torch.where(finite, b, 0.0).abs().amax(dim=1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    k = torch.where(m <= 0.875, e - 9, e - 8)
    k = torch.where(amax > 0, k, -118).clamp(-118, 120)
    code = torch.where(finite, torch.ldexp(b, -k), float("nan")).to(torch.float8_e4m3fn)
    return torch.ldexp(code.float(), k).reshape(-1)[:n].view(x.shape)


def _plain_checkpoint(st):
    return [_mxfp8(st["x"]).to(st["x"].dtype)]


def _plain_swiglu(st):
    g, u, dh = st["g"].detach(), st["u"].detach(), st["dh"].float()
    gf = g.float()
    h = (gf * torch.sigmoid(gf) * u.float()).to(g.dtype)
    gq, uq = _mxfp8(g), _mxfp8(u)
    sig = torch.sigmoid(gq)
    du = (dh * gq * sig).to(u.dtype)
    dg = (dh * uq * sig * (1.0 + gq * (1.0 - sig))).to(g.dtype)
    return [h, dg, du]


def _plain_router(st):
    x, wq, k16, ds = st["x"].detach(), st["wq"].detach(), st["k16"].detach(), st["ds"]
    xf, wf, kf = x.float(), wq.float(), k16.float()
    q = xf @ wf.t()
    r = torch.rsqrt((q * q).mean(dim=-1, keepdim=True) + EPS)
    qn = q * r
    s = (qn @ kf.t()) * 0.25
    dqn = (ds @ kf) * 0.25
    dk = (ds.t() @ qn) * 0.25
    dq = r * (dqn - qn * (dqn * qn).mean(dim=-1, keepdim=True))
    dx = (dq @ wf).to(x.dtype)
    dw = dq.t() @ (_mxfp8(x) if st["case"]["mxfp8"] else xf)
    return [s, dx, dw.to(wq.dtype), dk.to(k16.dtype)]


def _plain_balance(st):
    case, s = st["case"], st["s"].detach()
    NB, base, T = case["blocks"], case["base"], case["temperature"]
    R = NB - base
    valid = st["valid"] if st["valid"] is not None else torch.ones(s.shape[0], dtype=torch.bool, device=s.device)
    idx, cnt = st["idx"].long(), st["cnt"].long()
    live = (torch.arange(idx.shape[1], device=s.device) < cnt[:, None]) & valid[:, None]
    counts = torch.zeros(NB, dtype=torch.int64, device=s.device).index_add_(0, idx.reshape(-1), live.reshape(-1).long())
    z = s[:, base:] / T
    top = z.amax(dim=-1, keepdim=True)
    rows = valid & (top[:, 0] > -math.inf)
    e = torch.where(rows[:, None], torch.exp(z - top), 0.0)
    p = e / e.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    n = rows.sum().clamp_min(1)
    f = counts[base:].double() / counts.sum().clamp_min(1)
    loss = (R * (f * p.sum(dim=0, dtype=torch.float64)).sum() / n).float()
    ff = f - 1.0 / R
    ff = ff.float()
    inner = (p * ff).sum(dim=-1, keepdim=True)
    ds = torch.zeros_like(s)
    ds[:, base:] = p * (ff - inner) * (st["dloss"] * R / (T * n))
    return [loss, counts, ds]


# ------------------------------------------------------------------ the framework's operators
def _own(st):
    import foveal_sparse_indexer_b200 as fsi

    case, op = st["case"], st["case"]["op"]
    if op == "checkpoint":
        return [fsi.checkpoint_mxfp8(st["x"]).restore()]
    if op == "swiglu":
        h = fsi.triton_fused_swiglu(st["g"], st["u"], checkpoint="mxfp8")
        return [h.detach(), *torch.autograd.grad(h, (st["g"], st["u"]), st["dh"])]
    if op == "router":
        s = fsi.router_scores(st["x"], st["wq"], st["k16"], checkpoint="mxfp8" if case["mxfp8"] else None)
        return [s.detach(), *torch.autograd.grad(s, (st["x"], st["wq"], st["k16"]), st["ds"])]
    loss, counts = fsi.balance_loss(st["s"], st["idx"], st["cnt"], base_blocks=case["base"],
                                    temperature=case["temperature"], valid=st["valid"])
    return [loss.detach(), counts, *torch.autograd.grad(loss, (st["s"],), st["dloss"])]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "checkpoint":
        return _plain_checkpoint(state)
    if op == "swiglu":
        return _plain_swiglu(state)
    if op == "router":
        return _plain_router(state)
    return _plain_balance(state)


def work(case):
    op = case["op"]
    s = 4 if case.get("dtype") == "fp32" else 2
    if op == "balance":
        M, NB, k = case["rows"], case["blocks"], (case["kmin"] + case["kmax"]) / 2
        # scores in both passes' one reading, their gradient, the lists' live part and their lengths
        return {"bytes": int(8 * M * NB + 4 * M * k + 4 * M + 8 * NB), "flops": 14 * M * (NB - case["base"])}
    n = case["rows"] * case["cols"]
    if op == "checkpoint":
        return {"bytes": 2 * s * n, "flops": 4 * n}
    if op == "swiglu":
        return {"bytes": 6 * s * n, "flops": 24 * n}
    M, D, NB = case["rows"], case["cols"], case["blocks"]
    return {"bytes": 2 * s * n + 8 * M * NB + 2 * s * 16 * (D + NB), "flops": 96 * n + 96 * M * NB}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_mxfp8(x):
    """Value by value: the grid step of e4m3 at each magnitude, and rounding to the nearest even multiple."""
    v = x.detach().reshape(-1).double()
    n = v.numel()
    blocks = torch.zeros((n + 31) // 32 * 32, dtype=torch.float64, device=v.device)
    blocks[:n] = v
    blocks = blocks.view(-1, 32)
    top = torch.nan_to_num(blocks.abs(), nan=0.0, posinf=0.0).max(dim=1).values
    k = torch.full_like(top, -118.0)
    some = top > 0
    k[some] = torch.ceil(torch.log2(top[some] / 448.0))
    k = torch.where(some & (top > 448.0 * torch.exp2(k)), k + 1, k)  # log2 may be one step off at the border
    k = torch.where(some & (top <= 448.0 * torch.exp2(k - 1)), k - 1, k)
    unit = torch.exp2(k.clamp(-118, 120))[:, None]
    y = blocks / unit
    _, e = torch.frexp(y)  # |y| in [2^(e-1), 2^e)
    step = torch.exp2((e - 4).clamp_min(-9).double())
    q = torch.round(y / step) * step * unit
    q[~torch.isfinite(blocks)] = math.nan
    return q.reshape(-1)[:n].view(x.shape)


def _exact_swiglu(g, u, dh, gq, uq):
    t = torch.exp(-g)
    h = g * u / (1.0 + t)
    t = torch.exp(-gq)
    w = 1.0 / (1.0 + t)
    return h, dh * uq * w * (1.0 + gq * t * w), dh * gq * w


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        return [_exact_mxfp8(st["x"])]
    if op == "swiglu":
        g, u, dh = st["g"].detach(), st["u"].detach(), st["dh"]
        parts = []
        flat = [t.reshape(-1) for t in (g, u, dh)]
        step = 1 << 25  # a multiple of the blocks of 32
        for a in range(0, max(1, flat[0].numel()), step):
            ga, ua, da = (t[a:a + step] for t in flat)
            parts.append(_exact_swiglu(ga.double(), ua.double(), da.double(), _exact_mxfp8(ga), _exact_mxfp8(ua)))
        return [torch.cat(p).view(g.shape) for p in zip(*parts)]
    if op == "router":
        x, wq, k16 = (st[n].detach().double() for n in ("x", "wq", "k16"))
        ds = st["ds"].double()
        q = x @ wq.t()
        m = (q * q).sum(dim=1, keepdim=True) / 16.0 + EPS
        s = q @ k16.t() / (4.0 * m.sqrt())
        a = ds @ k16 / 4.0
        dk = (ds / m.sqrt()).t() @ q / 4.0
        dq = a / m.sqrt() - q * (a * q).sum(dim=1, keepdim=True) / (16.0 * m * m.sqrt())
        dw = dq.t() @ (_exact_mxfp8(st["x"]) if case["mxfp8"] else x)
        return [s, dq @ wq, dw, dk]
    s = st["s"].detach().double()
    NB, base, T = case["blocks"], case["base"], case["temperature"]
    M = s.shape[0]
    ok = torch.ones(M, dtype=torch.bool, device=s.device) if st["valid"] is None else st["valid"]
    slots = torch.arange(st["idx"].shape[1], device=s.device)[None, :].expand(M, -1)
    named = st["idx"][(slots < st["cnt"][:, None]) & ok[:, None]].long()
    counts = torch.bincount(named, minlength=NB)
    p = torch.softmax(s[:, base:] / T, dim=1)
    p = torch.where(ok[:, None], p, 0.0)
    n = max(1, int(ok.sum()))
    c = counts[base:].double()
    weight = (NB - base) * c / max(1.0, float(c.sum())) / n
    loss = (p.sum(dim=0) * weight).sum()
    ds = torch.zeros_like(s)
    ds[:, base:] = p * (weight - (p @ weight)[:, None]) / T * float(st["dloss"])
    return [loss, counts, ds]
