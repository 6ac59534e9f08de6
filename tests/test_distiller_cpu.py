"""The top-logit distiller's loss next to the student's own, on the CPU."""
import math

import pytest
import torch

from predicitivecoding_b200.llm.distill import TopLogitDistiller
from predicitivecoding_b200.models.config import DecoderLmConfig
from predicitivecoding_b200.models.decoder_lm import DecoderLM

SHAPE = dict(vocab=40, num_heads=2, max_seq=12, use_rms_norm=True, use_rope=True)


def model(seed, dim=16, **kw):
    return DecoderLM(DecoderLmConfig(dim=dim, num_blocks=2, ff_dim=24, **{**SHAPE, **kw}), seed=seed)


def batch(seed=3):
    rows = torch.randint(0, 40, (4, 13), generator=torch.Generator().manual_seed(seed))
    return rows[:, :-1], rows[:, 1:].clone()


@pytest.mark.parametrize("alpha", [0.25, 1.0])
@pytest.mark.parametrize("pad", [-100, 40])
def test_both_terms_run_over_the_same_rows(alpha, pad):
    """A target outside the vocabulary takes its row out of both terms, whatever ignore_index is."""
    teacher, student = model(1, 24), model(2)
    tokens, targets = batch()
    d = TopLogitDistiller(student, top_k=5, temperature=2.0, alpha=alpha)
    ids, logits = d.ask(teacher, tokens)
    padded, ignored = targets.clone(), targets.clone()
    padded[:, :3] = pad
    ignored[:, :3] = -1
    got, want = d.loss(tokens, padded, ids, logits), d.loss(tokens, ignored, ids, logits)
    assert float(got.detach()) == float(want.detach())
