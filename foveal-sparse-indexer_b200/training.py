"""Training operators of the routed parameter-block layers.

* ``checkpoint_mxfp8(x)`` keeps an activation in 8 bits from a forward to its backward pass; ``restore()``
  reads it back.  ``checkpoint="mxfp8"`` of ``triton_fused_swiglu``, ``router_scores`` and
  ``FovealPattentionMLP`` makes their backward passes read such copies instead of the tensors themselves.
* ``router_scores(x, q_proj, block_keys)`` is ``compute_router_scores`` (foveal_pattention.py:257-262) with
  a gradient into x, q_proj and block_keys.
* ``balance_loss(scores, remote_indices, remote_counts, base_blocks=...)`` is the load-balance loss over the
  remote blocks with its gradient into the scores, and the blocks' slot counts; ``block_counts`` gives the
  counts alone (for example to sum them over ranks first).

The reference trains its router by distillation only; these operators have no counterpart there.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import kernels
from ._lib import dtype_code

CHECKPOINTS = (None, "mxfp8")
MAX_CAPACITY = 1 << 20  # slots of a row's route list


def check_checkpoint(checkpoint: Optional[str]) -> Optional[str]:
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"unknown checkpoint {checkpoint!r}; expected one of {CHECKPOINTS}")
    return checkpoint


@dataclass
class MXFP8Checkpoint:
    """An 8-bit copy of a tensor: per 32 consecutive elements (row-major order) one power-of-two scale, the
    smallest with max|x| <= 448 * scale over the block's finite elements, and e4m3 codes rounded to nearest
    even (240 * 2^120 for the magnitudes that would round to 2^128).  NaN and infinities are kept as NaN."""

    buffer: Tensor        # uint8: codes, padded to 16 bytes, then scale bytes
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.buffer.numel()

    @property
    def codes(self) -> Tensor:
        """The e4m3 codes, in the tensor's shape."""
        return self.buffer[:self.shape.numel()].view(torch.float8_e4m3fn).view(self.shape)

    @property
    def scales(self) -> Tensor:
        """One byte per block of 32 elements: the scale's exponent plus 127."""
        return self.buffer[(self.shape.numel() + 15) // 16 * 16:]

    def restore(self) -> Tensor:
        """The values the copy stands for, in the tensor's shape and dtype (exact in fp32 and bf16)."""
        return kernels.mxfp8_dequantize(self.buffer, self.shape, self.dtype)


def checkpoint_mxfp8(x: Tensor) -> MXFP8Checkpoint:
    """An 8-bit copy of ``x`` (fp32 or bf16 CUDA tensor, any shape); no gradient flows through it."""
    return MXFP8Checkpoint(kernels.mxfp8_quantize(x.detach()), x.shape, x.dtype)


def once(backward):
    """``once_differentiable`` where the caller builds a graph of the backward pass, the plain function otherwise (the
    wrapper costs a tenth of a small backward pass).  A second derivative then raises, also where the upstream
    gradient is a constant (``y.sum()``): the gradients still depend on the saved tensors, so the wrapper is given
    an argument that requires a gradient."""
    guarded = once_differentiable(lambda ctx, anchor, *grads: backward(ctx, *grads))

    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        return guarded(ctx, torch.empty(0, requires_grad=True), *grads)

    return run


class _RouterScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, q_proj, block_keys, keep):
        scores, saved, buf = kernels.router_scores_train(x, q_proj, block_keys, keep_mxfp8=keep)
        ctx.dtype = x.dtype
        ctx.save_for_backward(x if ctx.needs_input_grad[1] and not keep else None, buf, q_proj, block_keys, saved)
        return scores

    @staticmethod
    @once
    def backward(ctx, dscores):
        x, buf, q_proj, block_keys, saved = ctx.saved_tensors
        dx, dw, dk = kernels.router_scores_bwd(dscores, x, buf, q_proj, block_keys, saved, ctx.dtype,
                                               ctx.needs_input_grad)
        return dx, dw, dk, None


def check_router(x: Tensor, q_proj: Tensor, block_keys: Tensor) -> None:
    """Refuses what :func:`router_scores` does not take."""
    for t in (x, q_proj, block_keys):
        dtype_code(t.dtype)
    D = x.shape[-1] if x.dim() else 0
    if q_proj.dim() != 2 or q_proj.shape[0] != 16 or q_proj.shape[1] != D or block_keys.dim() != 2 \
            or block_keys.shape[1] != 16:
        raise ValueError(f"shapes: x [..., D], q_proj [16, D], block_keys [NB, 16]; got x {tuple(x.shape)}, "
                         f"q_proj {tuple(q_proj.shape)}, block_keys {tuple(block_keys.shape)}")
    NB = block_keys.shape[0]
    if D == 0 or D % 8 or not 1 <= NB <= 1024:
        raise ValueError(f"the router takes widths that are multiples of 8 and 1 to 1024 blocks, got D {D}, NB {NB}")


def router_scores(x: Tensor, q_proj: Tensor, block_keys: Tensor, *, checkpoint: Optional[str] = None) -> Tensor:
    """``rms_norm(x q_proj^T) block_keys^T / 4`` per token, differentiable in all three: x [..., D] fp32 or
    bf16, q_proj [16, D], block_keys [NB, 16] -> fp32 [..., NB].  q_proj and block_keys are read in x's type (as
    ``compute_router_scores`` does: fp32 weights next to bf16 x are rounded to bf16), their gradients leave in
    their own.  With ``checkpoint="mxfp8"`` the backward pass reads an 8-bit copy of x (it enters q_proj's
    gradient only; where q_proj takes none, neither x nor a copy is kept)."""
    check_checkpoint(checkpoint)
    check_router(x, q_proj, block_keys)
    # only q_proj's gradient reads the tokens: without it neither x nor a copy is kept
    keep = checkpoint is not None and torch.is_grad_enabled() and q_proj.requires_grad
    return _RouterScores.apply(x, q_proj, block_keys, keep)


def _check_routes(remote_indices: Tensor, remote_counts: Tensor) -> None:
    for t in (remote_indices, remote_counts):
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"remote_indices and remote_counts are int32 or int64, got {t.dtype}")
    if remote_indices.dim() < 1 or remote_indices.shape[:-1] != remote_counts.shape:
        raise ValueError(f"shapes: remote_indices [..., capacity], remote_counts [...]; got "
                         f"{tuple(remote_indices.shape)} and {tuple(remote_counts.shape)}")
    if remote_indices.shape[-1] > MAX_CAPACITY:  # partial slot counts have 32 bits
        raise ValueError(f"a route list holds at most {MAX_CAPACITY} slots, got {remote_indices.shape[-1]}")


def _check_valid(valid: Optional[Tensor], lead: torch.Size) -> None:
    if valid is not None and (valid.dtype != torch.bool or valid.shape != lead):
        raise ValueError(f"valid is a bool tensor of shape {tuple(lead)}, got {valid.dtype} {tuple(valid.shape)}")


def _check_blocks(num_blocks: int) -> int:
    if not 1 <= int(num_blocks) <= 1024:
        raise ValueError(f"1 to 1024 blocks, got {num_blocks}")
    return int(num_blocks)


def block_counts(remote_indices: Tensor, remote_counts: Tensor, num_blocks: int, *,
                 valid: Optional[Tensor] = None) -> Tensor:
    """int64 [num_blocks]: how many slots of the route lists name each block.  remote_indices
    [..., capacity], of which row t's first remote_counts[t] count (ids outside [0, num_blocks) do not);
    ``valid`` (bool [...]) leaves rows out, for example padding."""
    NB = _check_blocks(num_blocks)
    _check_routes(remote_indices, remote_counts)
    _check_valid(valid, remote_counts.shape)
    _, counts, _ = kernels.balance_loss_fwd(None, remote_indices, remote_counts, NB, 0, 1.0, valid)
    return counts


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, idx, cnt, base, temperature, valid, counts_in):
        loss, counts, state = kernels.balance_loss_fwd(scores, idx, cnt, scores.shape[-1], base, temperature, valid,
                                                       counts_in)
        ctx.base, ctx.temperature = base, temperature
        ctx.save_for_backward(scores, valid, state)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)  # no zeros for the counts' gradient, which would be a launch
        return loss, counts

    @staticmethod
    @once
    def backward(ctx, dloss, _dcounts):
        if dloss is None:
            return (None,) * 7
        scores, valid, state = ctx.saved_tensors
        ds = kernels.balance_loss_bwd(scores, ctx.base, ctx.temperature, valid, state, dloss)
        return ds, None, None, None, None, None, None


def _check_balance(scores, remote_indices, remote_counts, base_blocks, temperature, valid, counts=None):
    """The arguments of :func:`balance_loss`, refused or in the kernels' types."""
    NB = _check_blocks(scores.shape[-1] if scores.dim() else 0)
    if not 0 <= int(base_blocks) < NB:
        raise ValueError(f"base_blocks must leave a remote block: 0 <= base_blocks < {NB}, got {base_blocks}")
    # beyond these the kernels' fp32 1 / T and R / (T n) would overflow or vanish, and 0 * inf be NaN
    if not 1e-30 <= float(temperature) <= 1e30:
        raise ValueError(f"temperature must be between 1e-30 and 1e30, got {temperature}")
    if not scores.is_floating_point():
        raise TypeError(f"scores must be floating point, got {scores.dtype}")
    lead = scores.shape[:-1]
    if counts is not None:
        if counts.dtype != torch.int64 or counts.shape != (NB,):
            raise ValueError(f"counts is an int64 tensor [{NB}], got {counts.dtype} {tuple(counts.shape)}")
        remote_indices = remote_counts = None
    else:
        if remote_indices is None or remote_counts is None:
            raise ValueError("remote_indices and remote_counts are needed unless counts are given")
        _check_routes(remote_indices, remote_counts)
        if remote_counts.shape != lead:
            raise ValueError(f"routes of {tuple(remote_counts.shape)} rows for scores of {tuple(lead)}")
    _check_valid(valid, lead)
    if scores.dtype != torch.float32:
        scores = scores.float()
    return scores, remote_indices, remote_counts, int(base_blocks), float(temperature)


def checked_balance(scores: Tensor, remote_indices: Tensor, remote_counts: Tensor, base_blocks: int,
                    temperature: float, valid: Optional[Tensor]):
    """(loss, counts, state) of :func:`balance_loss`'s forward, without a graph."""
    scores, idx, cnt, base, T = _check_balance(scores, remote_indices, remote_counts, base_blocks, temperature, valid)
    return kernels.balance_loss_fwd(scores, idx, cnt, scores.shape[-1], base, T, valid)


def balance_loss(scores: Tensor, remote_indices: Optional[Tensor], remote_counts: Optional[Tensor], *,
                 base_blocks: int, temperature: float = 1.0, valid: Optional[Tensor] = None,
                 counts: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """Load-balance loss of a routing and the blocks' slot counts.

    scores [..., NB] are the router's scores (before the temperature), remote_indices [..., capacity] and
    remote_counts [...] the routes chosen from them (``select_blocks``).  With p_t the softmax of
    scores_t / temperature over the R = NB - base_blocks remote blocks, f_b block b's share of the slots and n
    the number of rows, ``loss = R sum_b f_b (1/n) sum_t p_tb``: 1 for an even load, R when one block takes
    everything.  Temperatures from 1e-30 to 1e30, at most 2^20 slots to a list.  The gradient reaches the scores
    through p only.

    Rows whose ``valid`` is False or whose remote scores are all -inf are not counted in n and receive zeros;
    the slots are those of :func:`block_counts`, which leaves out the rows whose ``valid`` is False only.
    ``counts`` (int64 [NB], :func:`block_counts` summed over ranks) replaces the lists' own counts; the
    lists may be None then.  Returns (loss fp32 0-d, counts int64 [NB])."""
    scores, idx, cnt, base, T = _check_balance(scores, remote_indices, remote_counts, base_blocks, temperature, valid,
                                               counts)
    return _BalanceLoss.apply(scores, idx, cnt, base, T, valid, counts)
