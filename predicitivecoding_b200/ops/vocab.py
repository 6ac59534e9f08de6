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
in fp32; the logits themselves are never stored.  ``head_bwd`` makes them again, ``piece`` columns of the vocabulary
at a time, which costs 8 N V D operations for a step instead of 6 and needs N * piece * 2 bytes (256 MiB by default)
instead of N * V * 2.  softmax - target is rounded to bf16 once, as an operand of the two gradient products.

Rows that are not counted - a target outside [0, V) or equal to ``ignore_index``, a teacher's list without entries -
have loss 0 and gradient 0, are not read and cost no products; the mean is over the counted rows, and 0 when there
are none.  A teacher's entry is absent when its id is outside [0, V) or its logit is -inf.

All results are the same from run to run: no sum depends on the order in which atomics arrive.
Kernels: csrc/vocab.cu, csrc/vocab_epilogue.cuh, csrc/gemm2_tcgen05.cu.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import ext

MAX_TOP_K = 256     # teacher entries per row
_IDS = (torch.int32, torch.int64)
_FLOATS = (torch.float32, torch.bfloat16)


def _ids(t: torch.Tensor, name: str, what: str) -> torch.Tensor:
    if not t.is_cuda or t.dtype not in _IDS:
        raise ValueError(f"{what}: {name} must be an int32 or int64 CUDA tensor")
    return t


def _same_device(what: str, **tensors) -> None:
    devices = {t.device for t in tensors.values() if t is not None}
    if len(devices) > 1:
        raise ValueError(f"{what}: {', '.join(tensors)} must be on one device")


# --------------------------------------------------------------------------- embedding
def embed_fwd(tok: torch.Tensor, w: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None,
              dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """scale * w[tok] as ``dtype`` (fp32, the residual stream, or bf16), [..., D]; w fp32 or bf16, rows of any
    stride.  Tokens outside [0, V) - padding - give zero rows."""
    _ids(tok, "tok", "embed_fwd")
    if not w.is_cuda or w.dtype not in _FLOATS or w.dim() != 2 or w.stride(1) != 1 or w.numel() == 0:
        raise ValueError("embed_fwd: w must be a [V, D] fp32 or bf16 CUDA tensor with a contiguous inner dimension")
    _same_device("embed_fwd", tok=tok, w=w, out=out)
    shape = (*tok.shape, w.shape[1])
    if out is None:
        if dtype not in _FLOATS:
            raise ValueError("embed_fwd: dtype must be float32 or bfloat16")
        out = torch.empty(shape, device=w.device, dtype=dtype)
    elif out.shape != shape or out.dtype not in _FLOATS or not out.is_contiguous():
        raise ValueError(f"embed_fwd: out must be a contiguous fp32 or bf16 tensor of shape {tuple(shape)}")
    if tok.numel():
        ext().vocab_embed_fwd(tok.contiguous(), w, float(scale), out)
    return out


def embed_bwd(tok: torch.Tensor, dx: torch.Tensor, vocab: int, scale: float = 1.0, out: Optional[torch.Tensor] = None,
              dtype: torch.dtype = torch.float32, accumulate: bool = False) -> torch.Tensor:
    """Gradient of :func:`embed_fwd` by w: [vocab, D] of ``dtype``, or into ``out`` (added to it with
    ``accumulate``, as for a matrix that the output head shares).  dx [..., D] fp32 or bf16.  The tokens are sorted
    and each row's sum is taken in fp32 in ascending order of place, then rounded once."""
    _ids(tok, "tok", "embed_bwd")
    if not dx.is_cuda or dx.dtype not in _FLOATS or dx.dim() < 1 or dx.shape[:-1] != tok.shape or dx.shape[-1] == 0:
        raise ValueError("embed_bwd: dx must be a [*tok.shape, D] fp32 or bf16 CUDA tensor")
    D = dx.shape[-1]
    if out is None:
        if vocab < 1 or dtype not in _FLOATS:
            raise ValueError("embed_bwd: vocab must be positive and dtype float32 or bfloat16")
        if accumulate:
            raise ValueError("embed_bwd: accumulate needs out")
        out = torch.empty(vocab, D, device=dx.device, dtype=dtype)
    elif out.shape != (vocab, D) or out.dtype not in _FLOATS or not out.is_contiguous() or vocab < 1:
        raise ValueError(f"embed_bwd: out must be a contiguous fp32 or bf16 [{vocab}, {D}] tensor")
    _same_device("embed_bwd", tok=tok, dx=dx, out=out)
    if tok.numel() == 0:
        return out if accumulate else out.zero_()
    d2 = dx.reshape(-1, D)
    if d2.stride(1) != 1:
        d2 = d2.contiguous()
    ext().vocab_embed_bwd(tok.contiguous(), d2, float(scale), out, bool(accumulate))
    return out


class Embed(torch.autograd.Function):
    """Autograd form of the lookup; the gradient has w's type."""

    @staticmethod
    def forward(ctx, tok, w, scale, dtype):
        ctx.save_for_backward(tok)
        ctx.w, ctx.scale = (w.shape[0], w.dtype), scale
        return embed_fwd(tok, w, scale, dtype=dtype)

    @staticmethod
    def backward(ctx, dx):
        tok, = ctx.saved_tensors
        return None, embed_bwd(tok, dx, ctx.w[0], ctx.scale, dtype=ctx.w[1]), None, None


def embedding(tok: torch.Tensor, w: torch.Tensor, scale: float = 1.0,
              dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Differentiable :func:`embed_fwd`."""
    return Embed.apply(tok, w, float(scale), dtype)


# --------------------------------------------------------------------------- head losses
@dataclass
class HeadState:
    """What a loss keeps for :func:`head_bwd`: the packed rows, their log-sum-exp and their targets."""
    saved: torch.Tensor
    scalars: torch.Tensor
    w: torch.Tensor
    lead: torch.Size
    N: int
    V: int
    D: int
    K: int
    distill: bool
    temperature: float
    reduction: str


def _head(what: str, x: torch.Tensor, w: torch.Tensor, reduction: str) -> torch.Tensor:
    for name, t in (("x", x), ("w", w)):
        if not t.is_cuda or t.dtype != torch.bfloat16:
            raise ValueError(f"{what}: {name} must be a bf16 CUDA tensor")
    if x.dim() < 1 or w.dim() != 2 or w.stride(1) != 1 or x.shape[-1] != w.shape[1] or w.numel() == 0:
        raise ValueError(f"{what}: x must be [..., D] and w [V, D] with a contiguous inner dimension")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"{what}: reduction must be mean, sum or none")
    x2 = x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(1) == 1 else x2.contiguous()


def _loss(what, x, x2, w, reduction, tgt=None, ignore=-1, ids=None, logits=None, temperature=1.0):
    N, D = x2.shape
    lead, K = x.shape[:-1], 1 if ids is None else ids.shape[1]
    if N == 0:
        loss = torch.zeros(lead if reduction == "none" else (), device=x.device)
        return loss, HeadState(None, None, w, lead, 0, w.shape[0], D, K, ids is not None, temperature, reduction)
    rows, scalars, saved, wr = ext().vocab_fwd(x2, w, tgt, ignore, ids, logits, temperature, reduction == "mean")
    state = HeadState(saved, scalars, wr, lead, N, w.shape[0], D, K, ids is not None, temperature, reduction)
    return (rows.view(lead) if reduction == "none" else scalars[0]), state


def ce_fwd(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore_index: int = -1,
           reduction: str = "mean") -> Tuple[torch.Tensor, HeadState]:
    """Softmax cross entropy of the head x w^T without its logits: (fp32 loss, state for :func:`head_bwd`)."""
    x2 = _head("ce_fwd", x, w, reduction)
    _ids(targets, "targets", "ce_fwd")
    if targets.shape != x.shape[:-1]:
        raise ValueError("ce_fwd: targets must have x's leading shape")
    _same_device("ce_fwd", x=x, w=w, targets=targets)
    return _loss("ce_fwd", x, x2, w, reduction, tgt=targets.contiguous(), ignore=int(ignore_index))


def distill_fwd(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor, temperature: float = 1.0,
                reduction: str = "mean") -> Tuple[torch.Tensor, HeadState]:
    """Divergence of the student's softmax from the teacher's, which is known by its top logits: ids and logits
    [..., K], in any order, K <= 256; (fp32 loss, state for :func:`head_bwd`)."""
    x2 = _head("distill_fwd", x, w, reduction)
    _ids(ids, "ids", "distill_fwd")
    if not logits.is_cuda or logits.dtype not in _FLOATS:
        raise ValueError("distill_fwd: logits must be an fp32 or bf16 CUDA tensor")
    if ids.dim() != x.dim() or ids.shape != logits.shape or ids.shape[:-1] != x.shape[:-1]:
        raise ValueError("distill_fwd: ids and logits must be [*x.shape[:-1], K]")
    K = ids.shape[-1]
    if not 1 <= K <= MAX_TOP_K:
        raise ValueError(f"distill_fwd: between 1 and {MAX_TOP_K} entries per row")
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError("distill_fwd: temperature must be positive and finite")
    _same_device("distill_fwd", x=x, w=w, ids=ids, logits=logits)
    i2, l2 = ids.reshape(-1, K), logits.reshape(-1, K)
    return _loss("distill_fwd", x, x2, w, reduction, ids=i2 if i2.stride(1) == 1 else i2.contiguous(),
                 logits=l2 if l2.stride(1) == 1 else l2.contiguous(), temperature=float(temperature))


def head_bwd(state: HeadState, gout: Union[float, torch.Tensor] = 1.0, dx: Optional[torch.Tensor] = None,
             dw: Optional[torch.Tensor] = None, need_dx: bool = True, need_dw: bool = True, accumulate: bool = False,
             piece: int = 0) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx [..., D], dw [V, D]) of a mean or summed loss times ``gout`` (a number, or an fp32 CUDA tensor with one
    value).  They are bf16, or go into ``dx`` / ``dw`` (bf16 or fp32; ``accumulate`` adds to ``dw``).  ``piece``: columns of
    the vocabulary at a time (rounded up to a multiple of 256; 0: as many as 256 MiB of workspace take)."""
    s = state
    if s.reduction == "none":
        raise ValueError("head_bwd: the gradient is of a mean or summed loss")
    if accumulate and dw is None:
        raise ValueError("head_bwd: accumulate needs dw")
    dev = s.w.device
    for name, t, shape in (("dx", dx, (*s.lead, s.D)), ("dw", dw, (s.V, s.D))):
        if t is not None and (t.shape != shape or t.dtype not in _FLOATS or t.device != dev or t.stride(-1) != 1):
            raise ValueError(f"head_bwd: {name} must be a bf16 or fp32 {tuple(shape)} tensor on w's device with a "
                             "contiguous inner dimension")
    if dx is not None and not dx.is_contiguous() and dx.dim() != 2:
        raise ValueError("head_bwd: dx must be contiguous")
    if isinstance(gout, torch.Tensor) and (gout.dtype != torch.float32 or gout.numel() != 1 or gout.device != dev):
        raise ValueError("head_bwd: gout must be a number or one fp32 value on w's device")
    if piece < 0:
        raise ValueError("head_bwd: piece must not be negative")
    if dx is None and need_dx:
        dx = torch.empty(*s.lead, s.D, device=dev, dtype=torch.bfloat16)
    if dw is None and need_dw:
        dw = torch.empty(s.V, s.D, device=dev, dtype=torch.bfloat16)
    if s.N == 0:
        if dw is not None and not accumulate:
            dw.zero_()
        return dx, dw
    if dx is not None or dw is not None:
        on_device = isinstance(gout, torch.Tensor)
        ext().vocab_bwd(s.saved, s.scalars, s.w, s.N, s.V, s.D, s.K, s.distill, s.temperature, s.reduction == "mean",
                        1.0 if on_device else float(gout), gout if on_device else None,
                        None if dx is None else dx.view(-1, s.D) if dx.dim() != 2 else dx, dw, bool(accumulate),
                        int(piece))
    return dx, dw


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, kind, args, reduction):
        loss, ctx.state = (ce_fwd if kind == "ce" else distill_fwd)(x, w, *args, reduction)
        return loss

    @staticmethod
    def backward(ctx, g):
        dx, dw = head_bwd(ctx.state, g.float().contiguous(), need_dx=ctx.needs_input_grad[0],
                          need_dw=ctx.needs_input_grad[1])
        return dx, dw, None, None, None


def cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore_index: int = -1,
                  reduction: str = "mean") -> torch.Tensor:
    """Differentiable :func:`ce_fwd` (mean or sum; ``none`` has no gradient)."""
    if reduction == "none":
        return ce_fwd(x, w, targets, ignore_index, reduction)[0]
    return _HeadLoss.apply(x, w, "ce", (targets, ignore_index), reduction)


def distill(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor, temperature: float = 1.0,
            reduction: str = "mean") -> torch.Tensor:
    """Differentiable :func:`distill_fwd` by x and w (mean or sum); the teacher's logits get no gradient."""
    if reduction == "none":
        return distill_fwd(x, w, ids, logits, temperature, reduction)[0]
    return _HeadLoss.apply(x, w, "distill", (ids, logits, temperature), reduction)
