"""Refusals of the training operators, on the CPU: the Python layer's argument checks and the C ABI's, which
come before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import fsi

P = ctypes.c_void_p
A = P(4096)      # an aligned address that no check dereferences
ODD = P(4100)    # not 16-byte aligned
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    __import__("importlib").import_module("foveal-sparse-indexer_b200.build").build()
    return fsi.load_library()


def test_cpu_tensors_raise():
    x = torch.randn(4, 64)
    with pytest.raises(RuntimeError):
        fsi.checkpoint_mxfp8(x)
    with pytest.raises(RuntimeError):
        fsi.triton_fused_swiglu(x.requires_grad_(), x, checkpoint="mxfp8")
    with pytest.raises(RuntimeError):
        fsi.router_scores(x, torch.randn(16, 64), torch.randn(8, 16))
    idx, cnt = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        fsi.block_counts(idx, cnt, 8)
    with pytest.raises(RuntimeError):
        fsi.balance_loss(torch.randn(4, 8), idx, cnt, base_blocks=1)


def test_unknown_checkpoint():
    x = torch.randn(4, 64)
    for call in (lambda: fsi.triton_fused_swiglu(x, x, checkpoint="int8"),
                 lambda: fsi.router_scores(x, torch.randn(16, 64), torch.randn(8, 16), checkpoint="e4m3"),
                 lambda: fsi.FovealPattentionMLP(64, 128, base_blocks=1, remote_blocks=1, checkpoint="fp8")):
        with pytest.raises(ValueError, match="unknown checkpoint"):
            call()


def test_checkpoint_argument_reaches_the_module():
    dense = torch.nn.Module()
    for name, a, b in (("gate_proj", 64, 256), ("up_proj", 64, 256), ("down_proj", 256, 64)):
        setattr(dense, name, torch.nn.Linear(a, b, bias=False))
    layer = torch.nn.Module()
    layer.mlp = dense
    model = torch.nn.Module()
    model.layers = torch.nn.ModuleList([layer])
    fsi.sparsify_model_with_foveal_pattention(model, base_blocks=1, remote_blocks=2, checkpoint="mxfp8")
    assert model.layers[0].mlp.checkpoint == "mxfp8"
    assert fsi.FovealPattentionMLP(64, 128, base_blocks=1, remote_blocks=1).checkpoint is None


@pytest.mark.parametrize("x,wq,k", [((4, 60), (16, 60), (8, 16)), ((4, 64), (8, 64), (8, 16)), ((4, 64), (16, 32), (8, 16)),
                                    ((4, 64), (16, 64), (8, 8)), ((4, 64), (16, 64), (1025, 16)),
                                    ((4, 64), (16, 64), (0, 16)), ((4, 0), (16, 0), (8, 16)), ((), (16, 1), (8, 16))])
def test_router_scores_shapes(x, wq, k):
    with pytest.raises(ValueError):
        fsi.router_scores(torch.zeros(x), torch.zeros(wq), torch.zeros(k))


def test_router_scores_dtypes():
    with pytest.raises(TypeError):
        fsi.router_scores(torch.zeros(4, 64, dtype=torch.float16), torch.zeros(16, 64), torch.zeros(8, 16))


def _routes(M=4, cap=2):
    return torch.zeros(M, cap, dtype=torch.int32), torch.zeros(M, dtype=torch.int32)


@pytest.mark.parametrize("kw", [dict(base_blocks=8), dict(base_blocks=-1), dict(base_blocks=0, temperature=0.0),
                                dict(base_blocks=0, temperature=float("nan")),
                                dict(base_blocks=0, temperature=float("inf")),
                                dict(base_blocks=0, valid=torch.ones(3, dtype=torch.bool)),
                                dict(base_blocks=0, valid=torch.ones(4, dtype=torch.uint8)),
                                dict(base_blocks=0, counts=torch.zeros(7, dtype=torch.int64)),
                                dict(base_blocks=0, counts=torch.zeros(8, dtype=torch.int32))])
def test_balance_loss_values(kw):
    idx, cnt = _routes()
    with pytest.raises(ValueError):
        fsi.balance_loss(torch.zeros(4, 8), idx, cnt, **kw)


@pytest.mark.parametrize("temperature", [1e300, 3.5e38, 1e31, 1e-31, 1e-60])
def test_balance_loss_temperature_range(temperature):
    idx, cnt = _routes()
    with pytest.raises(ValueError, match="temperature"):
        fsi.balance_loss(torch.zeros(4, 8), idx, cnt, base_blocks=0, temperature=temperature)


def test_route_list_too_long():
    idx, cnt = torch.zeros(1, 1, dtype=torch.int32).expand(4, 2 ** 20 + 1), _routes()[1]
    with pytest.raises(ValueError, match="slots"):
        fsi.block_counts(idx, cnt, 8)
    with pytest.raises(ValueError, match="slots"):
        fsi.balance_loss(torch.zeros(4, 8), idx, cnt, base_blocks=0)


def test_balance_loss_shapes_and_dtypes():
    idx, cnt = _routes()
    s = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        fsi.balance_loss(torch.zeros(5, 8), idx, cnt, base_blocks=0)
    with pytest.raises(ValueError):
        fsi.balance_loss(s, idx, cnt[:3], base_blocks=0)
    with pytest.raises(ValueError):
        fsi.balance_loss(s, None, cnt, base_blocks=0)
    with pytest.raises(ValueError):
        fsi.balance_loss(torch.zeros(4, 1025), idx, cnt, base_blocks=0)
    with pytest.raises(ValueError):
        fsi.balance_loss(torch.tensor(1.0), idx, cnt, base_blocks=0)
    with pytest.raises(TypeError):
        fsi.balance_loss(torch.zeros(4, 8, dtype=torch.int64), idx, cnt, base_blocks=0)
    with pytest.raises(TypeError):
        fsi.balance_loss(s, idx.float(), cnt, base_blocks=0)
    with pytest.raises(ValueError):
        fsi.block_counts(idx, cnt, 0)
    with pytest.raises(ValueError):
        fsi.block_counts(idx, cnt, 2000)
    with pytest.raises(TypeError):
        fsi.block_counts(idx, cnt.short(), 8)


def test_c_mxfp8(lib):
    q, d = lib.fp_mxfp8_quantize, lib.fp_mxfp8_dequantize
    assert q(None, 1, 0, None, None, None) == OK
    assert q(A, 1, -1, A, A, None) == INVALID
    assert q(A, 2, 64, A, A, None) == UNSUPPORTED
    for bad in ((None, A, A), (A, None, A), (A, A, None), (ODD, A, A), (A, ODD, A)):
        assert q(bad[0], 1, 64, bad[1], bad[2], None) == INVALID
    assert d(None, None, 0, 0, None, None) == OK
    assert d(A, A, 0, -5, A, None) == INVALID
    assert d(A, A, 7, 64, A, None) == UNSUPPORTED
    for bad in ((None, A, A), (A, None, A), (A, A, None), (ODD, A, A), (A, A, ODD)):
        assert d(bad[0], bad[1], 0, 64, bad[2], None) == INVALID


def test_c_swiglu_mxfp8(lib):
    f, b = lib.fp_swiglu_fwd_mxfp8, lib.fp_swiglu_bwd_mxfp8
    assert f(None, None, 1, 0, None, None, None, None, None, None) == OK
    assert f(A, A, 1, -1, A, A, A, A, A, None) == INVALID
    assert f(A, A, 3, 64, A, A, A, A, A, None) == UNSUPPORTED
    assert b(A, A, A, A, A, 1, -1, A, A, None, None) == INVALID
    assert b(A, A, A, A, A, 3, 64, A, A, None, None) == UNSUPPORTED
    for k in (0, 1, 4, 5, 6, 7, 8):
        args = [A, A, 1, 64, A, A, A, A, A, None]
        args[k] = None
        assert f(*args) == INVALID, k
        if k not in (6, 8):  # scale bytes have no alignment
            args[k] = ODD
            assert f(*args) == INVALID, k
    for k in (0, 1, 2, 3, 4, 7, 8):
        args = [A, A, A, A, A, 1, 64, A, A, None, None]
        args[k] = None
        assert b(*args) == INVALID, k
    assert b(A, A, A, A, A, 1, 64, A, A, ODD, None) == INVALID


def test_c_router(lib):
    f, b, w = lib.fp_router_scores_train, lib.fp_router_scores_bwd, lib.fp_router_scores_bwd_workspace_size
    assert f(None, None, None, 1, 0, 64, 8, None, None, None, None, None, None) == OK
    assert f(A, A, A, 1, -1, 64, 8, A, A, A, None, None, None) == INVALID
    assert f(A, A, A, 1, 4, 60, 8, A, A, A, None, None, None) == UNSUPPORTED
    assert f(A, A, A, 1, 4, 64, 1025, A, A, A, None, None, None) == UNSUPPORTED
    assert f(A, A, A, 1, 4, 2 ** 24 + 8, 8, A, A, A, None, None, None) == UNSUPPORTED
    assert f(A, A, A, 5, 4, 64, 8, A, A, A, None, None, None) == UNSUPPORTED
    assert f(A, A, A, 1, 4, 64, 8, A, A, A, A, None, None) == INVALID
    assert f(A, A, A, 1, 4, 64, 8, A, A, A, ODD, A, None) == INVALID
    n = w(1, 4, 64, 8, 0)
    assert n > 0 and w(1, 0, 0, 0, 0) > 0
    assert w(1, 4096, 1000, 8, 1) >= w(1, 4096, 1000, 8, 0) + 4096 * 1000 * 2  # rows of codes that need a copy

    def go(ds=A, x=A, c=None, s=None, wq=A, k=A, q=A, r=A, dt=1, M=4, D=64, NB=8, dx=A, dw=A, dk=A, gd=0, ws=A, nb=n):
        return b(ds, x, c, s, wq, k, q, r, dt, M, D, NB, dx, dw, dk, gd, ws, nb, None)

    assert go(M=0) == INVALID
    assert go(D=12) == UNSUPPORTED
    assert go(D=2 ** 24 + 8) == UNSUPPORTED
    assert go(NB=2000) == UNSUPPORTED
    assert go(dt=4) == UNSUPPORTED
    assert go(gd=4) == UNSUPPORTED
    assert go(nb=n - 1) == WORKSPACE
    assert go(x=None) == INVALID          # dq_proj needs the tokens
    assert go(c=A) == INVALID             # codes without scales
    for name in ("ds", "wq", "k", "q", "r", "ws"):
        assert go(**{name: None}) == INVALID, name
    for name in ("ds", "x", "wq", "k", "q", "dx", "ws"):
        assert go(**{name: ODD}) == INVALID, name


def test_c_balance(lib):
    f, b, w = lib.fp_balance_loss_fwd, lib.fp_balance_loss_bwd, lib.fp_balance_workspace_size
    n = w(4, 8)

    def go(s=A, M=4, NB=8, base=1, T=1.0, valid=None, idx=A, cnt=A, cap=2, ci=None, co=A, loss=A, state=A, ws=A, nb=n):
        return f(s, M, NB, base, T, valid, idx, cnt, cap, ci, co, loss, state, ws, nb, None)

    assert go(M=-1) == INVALID
    assert go(NB=1025) == UNSUPPORTED
    assert go(base=8) == INVALID
    assert go(base=-1) == INVALID
    assert go(T=0.0) == INVALID
    assert go(T=float("nan")) == INVALID
    assert go(cap=-1) == INVALID
    assert go(idx=None) == INVALID
    assert go(idx=None, cnt=None) == INVALID
    assert go(s=None) == INVALID
    assert go(state=None) == INVALID
    assert go(co=None, loss=None, state=None) == INVALID
    assert go(ws=None) == INVALID
    assert go(ws=ODD) == INVALID
    assert go(nb=n - 1) == WORKSPACE
    assert b(A, 0, 8, 1, 1.0, None, A, A, A, None) == OK
    assert b(A, 4, 8, 8, 1.0, None, A, A, A, None) == INVALID
    assert b(A, 4, 8, 1, -1.0, None, A, A, A, None) == INVALID
    assert b(A, 4, 2000, 1, 1.0, None, A, A, A, None) == UNSUPPORTED
    for k in (0, 6, 7, 8):
        args = [A, 4, 8, 1, 1.0, None, A, A, A, None]
        args[k] = None
        assert b(*args) == INVALID, k


def test_c_balance_limits(lib):
    f, b, n = lib.fp_balance_loss_fwd, lib.fp_balance_loss_bwd, lib.fp_balance_workspace_size(4, 8)

    def go(T=1.0, cap=2):
        return f(A, 4, 8, 1, T, None, A, A, cap, None, A, A, A, A, n, None)

    for T in (float("inf"), 1e31, 1e-31):
        assert go(T=T) == INVALID
        assert b(A, 4, 8, 1, T, None, A, A, A, None) == INVALID
    assert go(cap=2 ** 20 + 1) == UNSUPPORTED
