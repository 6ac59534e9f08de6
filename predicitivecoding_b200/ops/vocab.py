"""The two ends of a decoder over its vocabulary: the embedding lookup with scaling and its gradient, and the losses
of the output head - softmax cross entropy and distillation from a teacher's top logits - with theirs.

Shapes: tokens and targets [...] int32 or int64, w [V, D] (nn.Linear layout, the embedding's too), x [..., D].

    embed_fwd    x = scale * w[tok]                                      tokens outside [0, V): a zero row
    embed_bwd    dw[v] (+)= scale * sum of dx over the tokens equal to v, in ascending order of place
    ce_fwd       loss_n = logsumexp(x_n w^T) - x_n . w[target_n]
    distill_fwd  loss_n = T^2 sum_k q_k (log q_k - log p_k),  q = softmax(teacher logits / T) over the row's entries,
                 p = softmax(x_n w^T / T) over the whole vocabulary
    head_bwd     the gradients of either loss

The losses take bf16 x and w, multiply on the tensor cores and hold the logits, the softmax statistics and every sum
in fp32; the logits themselves are not stored.  ``head_bwd`` makes them again, ``piece`` columns of the vocabulary
at a time, and keeps the gradient of a piece of them, g, for the two products that read it: 8 N V D operations for a
step instead of 6.  Its workspaces are g, R * piece * 2 bytes with R = N rounded up to a multiple of 256 and at least
512 (``piece`` is by default as large as 256 MiB allow, which may be all of V), and fp32 slabs, (R + 4096) * D * 4 bytes
for dx and up to 19 MiB more where dw has few tiles.  The state keeps N * D * 2 bytes for packed rows.  A vocabulary of up to
512 whose g stays within the bound is the exception: its loss is taken together with g, which the state then keeps.

softmax - target is an operand of the two gradient products in bf16: rounded once for more than 256 counted rows, as
two bf16 terms (2^-14 of it left out) up to there, whatever the type of the results.

Rows that are not counted - a target outside [0, V) or equal to ``ignore_index``, a teacher's list without entries -
have loss 0 and gradient 0, are not read and cost no products; the mean is over the counted rows, and 0 when there
are none.  A teacher's entry is absent when its id is outside [0, V) or its logit is -inf.

The ids of a row's list are meant to differ; entries that repeat an id count as they stand in the loss, and together
in the gradient.  All results are the same from run to run: no sum depends on the order in which atomics arrive.
x and w are read again by ``head_bwd`` and must not change in between; the state keeps them, next to its own buffers, for as
long as it lives (the autograd forms: as long as the graph does, outside the hooks of saved tensors).
A kernel that gives up a wait (which none does unless the device is in trouble) records it in the state: the loss and
the gradients made from it are NaN then, and ``state.status()``, which synchronises, returns the wait's code instead
of 0.  Several backwards of one state may run at the same time.
Kernels: csrc/vocab.cu, csrc/vocab_gemm.cu.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import ext

MAX_TOP_K = 256     # teacher entries per row
HeadState = object  # the extension's record of a loss: what head_bwd needs


# --------------------------------------------------------------------------- embedding
def embed_fwd(tok: torch.Tensor, w: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None,
              dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """scale * w[tok] as ``dtype`` (fp32, the residual stream, or bf16), [..., D]; w fp32 or bf16, rows of any
    stride.  Tokens outside [0, V) - padding - give zero rows."""
    return ext().vocab_embed_fwd(tok, w, scale, out, dtype)


def embed_bwd(tok: torch.Tensor, dx: torch.Tensor, vocab: int, scale: float = 1.0, out: Optional[torch.Tensor] = None,
              dtype: torch.dtype = torch.float32, accumulate: bool = False) -> torch.Tensor:
    """Gradient of :func:`embed_fwd` by w: [vocab, D] of ``dtype``, or into ``out`` (added to it with
    ``accumulate``, as for a matrix that the output head shares).  dx [..., D] fp32 or bf16.  Each row's sum is taken
    in fp32 over its tokens in ascending order of place, in parts of a fixed size where they are many, then rounded once.
    Batches above 1024 tokens (512 into a large matrix) are sorted; their workspace is N * D bytes and some per token."""
    return ext().vocab_embed_bwd(tok, dx, vocab, scale, out, dtype, accumulate)


class Embed(torch.autograd.Function):
    """Autograd form of the lookup; the gradient has w's type, and none of its own (differentiating it raises)."""

    @staticmethod
    def forward(ctx, tok, w, scale, dtype):
        ctx.save_for_backward(tok)
        ctx.w, ctx.scale = (w.shape[0], w.dtype), scale
        return embed_fwd(tok, w, scale, dtype=dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dx):
        tok, = ctx.saved_tensors
        return None, embed_bwd(tok, dx, ctx.w[0], ctx.scale, dtype=ctx.w[1]), None, None


def embedding(tok: torch.Tensor, w: torch.Tensor, scale: float = 1.0,
              dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Differentiable :func:`embed_fwd`."""
    return Embed.apply(tok, w, float(scale), dtype)


# --------------------------------------------------------------------------- head losses
def ce_fwd(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore_index: int = -1,
           reduction: str = "mean", gradient: bool = True) -> Tuple[torch.Tensor, HeadState]:
    """Softmax cross entropy of the head x w^T without its logits: (fp32 loss, state for :func:`head_bwd`).
    ``gradient=False``: no backward will follow."""
    return ext().vocab_ce_fwd(x, w, targets, ignore_index, reduction, gradient)


def distill_fwd(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor, temperature: float = 1.0,
                reduction: str = "mean", gradient: bool = True) -> Tuple[torch.Tensor, HeadState]:
    """Divergence of the student's softmax from the teacher's, which is known by its top logits: ids (int) and logits
    (fp32 or bf16) [..., K], in any order, K <= 256; (fp32 loss, state for :func:`head_bwd`).
    ``gradient=False``: no backward will follow."""
    return ext().vocab_distill_fwd(x, w, ids, logits, temperature, reduction, gradient)


def head_bwd(state: HeadState, gout: Union[float, torch.Tensor] = 1.0, dx: Optional[torch.Tensor] = None,
             dw: Optional[torch.Tensor] = None, need_dx: bool = True, need_dw: bool = True, accumulate: bool = False,
             piece: int = 0) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx [..., D], dw [V, D]) of a mean or summed loss times ``gout`` (a number, or an fp32 CUDA tensor with one
    value).  They are bf16, or go into ``dx`` / ``dw`` (bf16 or fp32; ``accumulate`` adds to ``dw``).  ``piece``: columns of
    the vocabulary at a time (rounded up to a multiple of 256; 0: as many as 256 MiB of g take; a vocabulary of up
    to 512 may be taken whole).  x and w must
    still hold what the loss read."""
    if isinstance(gout, torch.Tensor):
        return ext().vocab_head_bwd(state, 1.0, gout, dx, dw, need_dx, need_dw, accumulate, piece)
    return ext().vocab_head_bwd(state, gout, None, dx, dw, need_dx, need_dw, accumulate, piece)


class _Final(torch.autograd.Function):
    """A gradient made by kernels, as a function of what it depends on that cannot be differentiated."""

    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("the gradients of the vocabulary head's losses cannot be differentiated")


class _HeadLoss(torch.autograd.Function):
    """Autograd form of a mean or summed loss; its gradients have none of their own (differentiating them raises)."""

    @staticmethod
    def forward(ctx, x, w, kind, args, reduction):
        loss, ctx.state = (ce_fwd if kind == "ce" else distill_fwd)(x, w, *args, reduction)
        ctx.save_for_backward(x, w)   # so that a change of either before the backward is noticed
        return loss

    @staticmethod
    def backward(ctx, g):
        sources = ctx.saved_tensors
        with torch.no_grad():
            grads = head_bwd(ctx.state, g.float().contiguous(), need_dx=ctx.needs_input_grad[0],
                             need_dw=ctx.needs_input_grad[1])
        # once_differentiable would not do: it lets a gradient by way of a constant g pass, which yet depends on x and w
        if torch.is_grad_enabled():
            grads = tuple(d if d is None else _Final.apply(d, *sources, g) for d in grads)
        return *grads, None, None, None


class _RowLosses(torch.autograd.Function):
    """Per-row losses.  Their gradient does not exist; asking for it raises, where a detached result would train nothing."""

    @staticmethod
    def forward(ctx, x, w, kind, args):
        return (ce_fwd if kind == "ce" else distill_fwd)(x, w, *args, "none", gradient=False)[0]

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("losses with reduction 'none' have no gradient: take the mean or the sum")


def _differentiated(x: torch.Tensor, w: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and (x.requires_grad or w.requires_grad)


def _head_loss(kind: str, x: torch.Tensor, w: torch.Tensor, args: tuple, reduction: str) -> torch.Tensor:
    if not _differentiated(x, w):
        return (ce_fwd if kind == "ce" else distill_fwd)(x, w, *args, reduction, gradient=False)[0]
    if reduction == "none":
        return _RowLosses.apply(x, w, kind, args)
    return _HeadLoss.apply(x, w, kind, args, reduction)


def cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore_index: int = -1,
                  reduction: str = "mean") -> torch.Tensor:
    """Differentiable :func:`ce_fwd` (mean or sum; a backward through ``none`` raises)."""
    return _head_loss("ce", x, w, (targets, ignore_index), reduction)


def distill(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor, temperature: float = 1.0,
            reduction: str = "mean") -> torch.Tensor:
    """Differentiable :func:`distill_fwd` by x and w (mean or sum; a backward through ``none`` raises); the teacher's
    logits get no gradient."""
    return _head_loss("distill", x, w, (ids, logits, temperature), reduction)


# --------------------------------------------------------------------------- plain statements
def reference_embedding(tok: torch.Tensor, w: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """:func:`embedding` in plain differentiable torch, on any device."""
    live = (tok >= 0) & (tok < w.shape[0])
    return torch.where(live[..., None], w[tok.long().clamp(0, w.shape[0] - 1)] * scale, torch.zeros((), device=w.device))


def _mean_of_rows(rows: torch.Tensor, live: torch.Tensor, reduction: str) -> torch.Tensor:
    rows = torch.where(live, rows, torch.zeros((), device=rows.device, dtype=rows.dtype))
    if reduction == "none":
        return rows
    return rows.sum() / live.sum().clamp(min=1) if reduction == "mean" else rows.sum()


def reference_cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore_index: int = -1,
                            reduction: str = "mean") -> torch.Tensor:
    """:func:`cross_entropy` in plain differentiable torch with the logits in memory, on any device."""
    live = (targets >= 0) & (targets < w.shape[0]) & (targets != ignore_index)
    logp = torch.log_softmax(x @ w.t(), -1)
    at = torch.where(live, targets, torch.zeros_like(targets)).long()
    return _mean_of_rows(-logp.gather(-1, at[..., None])[..., 0], live, reduction)


def reference_distill(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor,
                      temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """:func:`distill` in plain differentiable torch with the student's logits in memory, on any device."""
    there = (ids >= 0) & (ids < w.shape[0]) & (logits != float("-inf"))
    live = there.any(-1)
    t = (logits.to(x.dtype) / temperature).masked_fill(~there, float("-inf"))
    logq = torch.log_softmax(torch.where(live[..., None], t, torch.zeros_like(t)), -1)
    q = torch.exp(logq) * there
    logp = torch.log_softmax(x @ w.t() / temperature, -1).gather(-1, torch.where(there, ids, torch.zeros_like(ids)).long())
    terms = torch.where(q > 0, q * (torch.where(q > 0, logq, torch.zeros_like(q)) - logp), torch.zeros_like(q))
    return _mean_of_rows(temperature ** 2 * terms.sum(-1), live, reduction)
