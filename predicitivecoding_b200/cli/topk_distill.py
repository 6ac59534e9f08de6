"""Distils a byte-level decoder into a smaller one from its top logits.

Usage: python -m predicitivecoding_b200.cli.topk_distill [--text FILE] [--steps N] [--top-k K] [--temperature T]
       [--alpha A] [--cpu]

A teacher is trained on the text; the student then learns, at every position, the teacher's top logits next to
the text itself.  Prints both models' cross entropy on the last tenth of the text, which neither trains on.
"""
from __future__ import annotations

import argparse
import sys

import torch

from ..llm.distill import TopLogitDistiller
from ..llm.tokenizer import ByteTokenizer
from ..models.config import DecoderLmConfig
from ..models.decoder_lm import DecoderLM
from ..optim.adam import Adam, clip_global_norm

TEXT = ("the night train left the harbour at nine and crossed the river before the rain began. "
        "a lamp moved along the platform, and the guard read the names of the towns aloud. "
        "in the last carriage someone counted the bridges and wrote each number in a small book. ") * 24


def batches(ids: torch.Tensor, seq: int, batch: int, steps: int, seed: int):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        at = torch.randint(0, ids.numel() - seq - 1, (batch,), generator=g)
        rows = torch.stack([ids[i:i + seq + 1] for i in at.tolist()])
        yield rows[:, :-1], rows[:, 1:]


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--text")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--top-k", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=2.0)
    ap.add_argument("--alpha", type=float, default=0.5)
    ap.add_argument("--cpu", action="store_true")
    a = ap.parse_args(argv)
    dev = "cuda" if torch.cuda.is_available() and not a.cpu else "cpu"
    text = open(a.text, encoding="utf-8").read() if a.text else TEXT
    tok = ByteTokenizer()
    ids = torch.tensor(tok.encode(text), device=dev)
    seq, batch = 32, 8
    cut = ids.numel() * 9 // 10
    if cut <= seq + 1 or ids.numel() - cut <= seq:
        print("the text is too short", file=sys.stderr)
        return 1
    shape = dict(vocab=tok.vocab_size, num_heads=4, max_seq=seq, use_rms_norm=True, use_rope=True, ffn="swiglu")
    teacher = DecoderLM(DecoderLmConfig(dim=64, num_blocks=3, ff_dim=128, **shape), seed=1).to(dev)
    student = DecoderLM(DecoderLmConfig(dim=32, num_blocks=1, ff_dim=64, **shape), seed=2).to(dev)

    held = ids[cut:cut + (ids.numel() - cut) // (seq + 1) * (seq + 1)].view(-1, seq + 1)

    def held_out(model) -> float:
        with torch.no_grad():
            return float(model.loss(held[:, :-1], held[:, 1:]))

    adam, params = Adam(), list(teacher.parameters())
    for x, y in batches(ids[:cut], seq, batch, a.steps, 3):
        for p in params:
            p.grad = None
        teacher.loss(x, y).backward()
        clip_global_norm(params, 1.0)
        adam.step(params, 3e-3)
    distiller = TopLogitDistiller(student, a.top_k, a.temperature, a.alpha)
    adam, before, loss = Adam(), held_out(student), float("nan")
    for x, y in batches(ids[:cut], seq, batch, a.steps, 4):
        loss = distiller.step(x, y, *distiller.ask(teacher, x), adam, 3e-3)
    print(f"teacher: held-out cross entropy {held_out(teacher):.4f}")
    print(f"student: held-out cross entropy {before:.4f} -> {held_out(student):.4f}, last step's loss {loss:.4f} ({dev})")
    return 0


if __name__ == "__main__":
    sys.exit(main())
