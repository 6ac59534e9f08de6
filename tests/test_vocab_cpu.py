"""The plain statements of the vocabulary-end operators against torch's own losses, the top-logit distiller on the
CPU, and the device entry points' refusal of CPU tensors.  Tolerances: sums of at most 10^3 fp64 terms, 1e-12."""
import math

import pytest
import torch
import torch.nn.functional as F

from predicitivecoding_b200.cli import topk_distill
from predicitivecoding_b200.llm.distill import TopLogitDistiller
from predicitivecoding_b200.models.config import DecoderLmConfig
from predicitivecoding_b200.models.decoder_lm import DecoderLM
from predicitivecoding_b200.ops import vocab
from predicitivecoding_b200.optim.adam import Adam


def rows(N=9, V=13, D=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    return r(N, D).requires_grad_(), r(V, D).requires_grad_(), torch.randint(0, V, (N,), generator=g), g


def close(a, b):
    return bool(((a - b).abs() <= 1e-12 * (1 + b.abs())).all())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reference_cross_entropy(reduction):
    x, w, t, _ = rows()
    t[3] = -1
    loss = vocab.reference_cross_entropy(x, w, t, reduction=reduction)
    ref = F.cross_entropy(x @ w.t(), t, ignore_index=-1, reduction=reduction)
    assert close(loss, ref)
    for a, b in zip(torch.autograd.grad(loss.sum(), (x, w), retain_graph=True), torch.autograd.grad(ref.sum(), (x, w))):
        assert close(a, b)
    none = torch.full_like(t, -1)
    assert float(vocab.reference_cross_entropy(x, w, none).detach()) == 0.0


def test_reference_distill_over_the_whole_vocabulary_is_the_kl_divergence():
    x, w, _, g = rows()
    t = torch.randn(9, 13, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(13, generator=g) for _ in range(9)])
    T = 2.0
    full = torch.zeros_like(t).scatter(1, ids, t)
    loss = vocab.reference_distill(x, w, ids, t, T)
    ref = T * T * F.kl_div(F.log_softmax(x @ w.t() / T, 1), F.log_softmax(full / T, 1), log_target=True,
                           reduction="batchmean")
    assert close(loss, ref)
    for a, b in zip(torch.autograd.grad(loss, (x, w), retain_graph=True), torch.autograd.grad(ref, (x, w))):
        assert close(a, b)


def test_reference_distill_of_lists_with_holes():
    x, w, _, g = rows()
    ids = torch.tensor([[2, -1, 5], [-1, -1, -1], [1, 12, 13]] * 3)
    t = torch.randn(9, 3, generator=g, dtype=torch.float64)
    t[0, 2] = float("-inf")
    loss = vocab.reference_distill(x, w, ids, t, 1.5, "none")
    assert loss[1] == 0 and loss[4] == 0
    logp = torch.log_softmax(x @ w.t() / 1.5, 1)
    assert close(loss[0], -2.25 * logp[0, 2])                    # one entry left: a class target
    q = torch.softmax(t[2, :2] / 1.5, 0)
    assert close(loss[2], 2.25 * (q * (q.log() - logp[2, [1, 12]])).sum())
    gx, gw = torch.autograd.grad(loss.sum(), (x, w))
    assert bool(torch.isfinite(gx).all() and torch.isfinite(gw).all()) and float(gx[1].abs().sum()) == 0.0


def test_reference_embedding():
    _, w, _, _ = rows()
    tok = torch.tensor([[3, -1], [12, 13]])
    x = vocab.reference_embedding(tok, w, 0.5)
    assert close(x[0, 0], 0.5 * w[3]) and close(x[1, 0], 0.5 * w[12])
    x = x.detach()
    assert float(x[0, 1].abs().sum()) == 0.0 and float(x[1, 1].abs().sum()) == 0.0


def models():
    shape = dict(vocab=40, num_heads=2, max_seq=12, use_rms_norm=True, use_rope=True, ffn="swiglu")
    return (DecoderLM(DecoderLmConfig(dim=24, num_blocks=2, ff_dim=32, **shape), seed=1),
            DecoderLM(DecoderLmConfig(dim=16, num_blocks=1, ff_dim=24, **shape), seed=2))


def test_distiller_loss_is_the_mix_of_both_and_falls():
    teacher, student = models()
    g = torch.Generator().manual_seed(3)
    rows_ = torch.randint(0, 40, (4, 13), generator=g)
    tokens, targets = rows_[:, :-1], rows_[:, 1:].clone()
    targets[:, :3] = -1
    d = TopLogitDistiller(student, top_k=5, temperature=2.0, alpha=0.25)
    ids, logits = d.ask(teacher, tokens)
    assert ids.shape == (4, 12, 5) and ids.dtype == torch.int32
    x = student.hidden(tokens)
    live = targets >= 0
    logp = torch.log_softmax(x @ student.wout / 2.0, -1)[live]
    q = torch.softmax(logits[live] / 2.0, -1)
    kd = 4.0 * (q * (q.log() - logp.gather(-1, ids[live].long()))).sum(-1).mean()
    ref = 0.75 * student.loss(tokens, targets) + 0.25 * kd
    assert math.isclose(float(d.loss(tokens, targets, ids, logits).detach()), float(ref.detach()), rel_tol=1e-5)
    adam = Adam()
    losses = [d.step(tokens, targets, ids, logits, adam, 1e-2) for _ in range(30)]
    assert losses[-1] < 0.8 * losses[0]


def test_distiller_refusals():
    _, student = models()
    for kw in ({"top_k": 0}, {"top_k": 41}, {"temperature": 0.0}, {"alpha": 1.5}, {"alpha": -0.1}):
        with pytest.raises(ValueError):
            TopLogitDistiller(student, **{"top_k": 4, **kw})


def test_command(capsys):
    assert topk_distill.main(["--cpu", "--steps", "6", "--top-k", "4"]) == 0
    out = capsys.readouterr().out
    assert "teacher: held-out" in out and "student: held-out" in out


def test_device_entry_points_refuse_cpu_tensors():
    x, w, t = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    ids = torch.zeros(2, 3, dtype=torch.int32)
    for f in (lambda: vocab.ce_fwd(x, w, t), lambda: vocab.distill_fwd(x, w, ids, torch.zeros(2, 3)),
              lambda: vocab.embed_fwd(t, w), lambda: vocab.embed_bwd(t, x, 5)):
        with pytest.raises(ValueError):
            f()
