"""Sequence-level distillation from a teacher function, and the on-policy (SEED-style) round.

Reference: PredictiveCoding.LLM/Training/LmDistiller.cs:29-166.  ``build_dataset`` asks the
teacher for the completion of every prompt (optionally cached on disk as JSONL); ``step``
trains on prompt + completion with the loss masked to the completion; ``on_policy_round``
lets the student draft, asks the teacher for a corrected completion, and trains on it.

``TopLogitDistiller`` is the token-level form, which the reference has not: the student learns the teacher's top
logits at every position, next to the usual targets.  On a GPU neither loss holds the student's logits
(:mod:`predicitivecoding_b200.ops.vocab`).
"""
from __future__ import annotations

import hashlib
import json
import os
from typing import Callable, List, Optional, Sequence, Tuple

import torch

from ..models.decoder_lm import DecoderLM, mtp_targets
from ..ops import vocab
from ..optim.adam import Adam, clip_global_norm
from .generation import greedy
from .trainer import step as adam_step


def build_dataset(prompts: Sequence[str], teacher: Callable[[str], str],
                  cache_dir: Optional[str] = None) -> List[Tuple[str, str]]:
    out = []
    cache = {}
    path = None
    if cache_dir:
        os.makedirs(cache_dir, exist_ok=True)
        path = os.path.join(cache_dir, "teacher.jsonl")
        if os.path.exists(path):
            for line in open(path, encoding="utf-8"):
                d = json.loads(line)
                cache[d["key"]] = d["completion"]
    for p in prompts:
        k = hashlib.sha256(p.encode("utf-8")).hexdigest()[:16]
        if k not in cache:
            cache[k] = teacher(p)
            if path:
                with open(path, "a", encoding="utf-8") as f:
                    f.write(json.dumps({"key": k, "prompt": p, "completion": cache[k]}) + "\n")
        out.append((p, cache[k]))
    return out


def _example(tok, prompt: str, completion: str, max_seq: int):
    pids = tok.encode(prompt, add_bos=True)
    cids = tok.encode(completion, add_eos=True)
    full = (pids + cids)[: max_seq + 1]
    tokens = full[:-1]
    targets = full[1:]
    for i in range(min(len(pids) - 1, len(targets))):
        targets[i] = -1
    return tokens, targets


def step(model, tok, data, optimizer: Adam, lr: float, clip_norm: float = 1.0) -> float:
    batch = [_example(tok, p, c, model.cfg.max_seq) for p, c in data]
    return adam_step(list(model.parameters()), batch,
                     lambda t, y, tr: model.loss(t.view(1, -1), y.view(1, -1), -1, tr), optimizer, lr, clip_norm)


def on_policy_round(model, tok, prompts: Sequence[str], teacher_correct: Callable[[str, str], str],
                    optimizer: Adam, lr: float, draft_tokens: int = 16, clip_norm: float = 1.0) -> float:
    data = []
    for p in prompts:
        ids = tok.encode(p, add_bos=True)
        out = greedy(model, ids, draft_tokens, tok.eos)
        draft = tok.decode(out[len(ids):])
        data.append((p, teacher_correct(p, draft)))
    return step(model, tok, data, optimizer, lr, clip_norm)


class _Operands(torch.autograd.Function):
    """``t`` as ``n`` operands in bf16, all of one memory, whose gradients are added in fp32."""

    @staticmethod
    def forward(ctx, t, n):
        ctx.set_materialize_grads(False)
        b = t.bfloat16().contiguous()
        return tuple(b.view_as(b) for _ in range(n))

    @staticmethod
    def backward(ctx, *grads):
        return sum(g.float() for g in grads if g is not None), None


class TopLogitDistiller:
    """Trains ``student`` on a teacher's top logits.

    loss = alpha * T^2 KL(q || p_T) + (1 - alpha) * cross entropy + the student's auxiliary terms, q the softmax of the
    teacher's ``top_k`` logits at temperature T, p_T the student's softmax at T over its whole vocabulary.  Both means run
    over the positions whose target is in the vocabulary and not ``ignore_index``.  The auxiliary terms (multi-token
    head, experts' balance) are those of ``DecoderLM.loss``, which this loss is at alpha 0.  ``embed_scale`` multiplies
    the student's embedding rows; given here it becomes the student's (``DecoderLmConfig.embed_scale``), so that the
    network which is trained is the one that is evaluated, served and saved.

    On a GPU the heads' products take the hidden rows and the output matrix in bf16, as the operators do, and each loss
    hands their gradients back in bf16; these are added, and reach the parameters, in the parameters' type.  On the CPU
    everything is in the model's type.
    """

    def __init__(self, student: DecoderLM, top_k: int = 32, temperature: float = 2.0, alpha: float = 0.5,
                 embed_scale: Optional[float] = None, ignore_index: int = -1):
        if not 1 <= top_k <= min(vocab.MAX_TOP_K, student.cfg.vocab):
            raise ValueError(f"top_k must be between 1 and {min(vocab.MAX_TOP_K, student.cfg.vocab)}")
        if not 2.0 ** -126 <= temperature < 2.0 ** 127:   # a positive fp32 number, as the operators take it
            raise ValueError("temperature must be positive and finite")
        if not 0.0 <= alpha <= 1.0:
            raise ValueError("alpha must be between 0 and 1")
        if embed_scale is not None:
            cfg = student.cfg.with_(embed_scale=float(embed_scale))
            cfg.validate()
            student.cfg = cfg
        self.student, self.top_k, self.temperature = student, top_k, float(temperature)
        self.alpha, self.ignore_index = alpha, ignore_index

    @property
    def embed_scale(self) -> float:
        return self.student.cfg.embed_scale

    @torch.no_grad()
    def ask(self, teacher: DecoderLM, tokens: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """The teacher's top logits for tokens [..., S]: (ids int32, logits) [..., S, top_k], to keep or to pass on."""
        top = teacher.forward(tokens).float().topk(self.top_k, dim=-1)
        return top.indices.int(), top.values

    def loss(self, tokens: torch.Tensor, targets: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor,
             training: bool = False) -> torch.Tensor:
        m, c, on_gpu = self.student, self.student.cfg, tokens.is_cuda
        embed = vocab.embedding if on_gpu else vocab.reference_embedding
        ce, kd = (vocab.cross_entropy, vocab.distill) if on_gpu else (vocab.reference_cross_entropy, vocab.reference_distill)
        balance = m.balance_terms()
        hidden = m.hidden(tokens, training, aux_losses=balance, embedded=embed(tokens, m.wemb, c.embed_scale))
        live = (targets >= 0) & (targets < c.vocab) & (targets != self.ignore_index)   # as the cross entropy counts
        ids = torch.where(live[..., None], ids, torch.full_like(ids, -1))
        mixed = (self.alpha < 1.0) + (self.alpha > 0.0)
        second = m.wout_mtp is not None
        operands = _Operands.apply if on_gpu else lambda t, n: (t,) * n
        x, w = list(operands(hidden, mixed + second)), list(operands(m.wout.t(), mixed))
        total = hidden.new_zeros((), dtype=torch.float32)
        if self.alpha < 1.0:
            total = total + (1.0 - self.alpha) * ce(x.pop(), w.pop(), targets, self.ignore_index)
        if self.alpha > 0.0:
            total = total + self.alpha * kd(x.pop(), w.pop(), ids, logits, self.temperature)
        if second:
            w, = operands(m.wout_mtp.t(), 1)
            ahead = mtp_targets(targets, c.mtp_horizon, self.ignore_index)
            total = total + c.mtp_weight * ce(x.pop(), w, ahead, self.ignore_index)
        if balance:
            total = total + c.moe_balance_weight * torch.stack(balance).sum()
        return total

    def step(self, tokens: torch.Tensor, targets: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor,
             optimizer: Adam, lr: float, clip_norm: float = 1.0) -> float:
        """One update on a batch [B, S]; returns its loss."""
        params = list(self.student.parameters())
        for p in params:
            p.grad = None
        loss = self.loss(tokens, targets, ids, logits, training=True)
        loss.backward()
        clip_global_norm(params, clip_norm)
        optimizer.step(params, lr)
        return float(loss.detach())
