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


@pytest.mark.parametrize("kw", [
    dict(mtp_weight=0.3), dict(mtp_weight=0.5, mtp_horizon=3), dict(num_experts=3, moe_top_k=2, moe_balance_weight=0.1),
    dict(mtp_weight=0.3, num_experts=2, moe_balance_weight=0.2), {},
])
def test_without_distillation_the_loss_is_the_students_own(kw):
    """alpha 0: value and gradients of DecoderLM.loss, with its multi-token head and its experts' balance.  fp32 sums of
    some hundred terms in another order: 2^-24 sqrt(300) of what they add up, 1e-5 of the largest gradient."""
    teacher, student = model(1, 24), model(2, **kw)
    tokens, targets = batch()
    targets[:, :3] = -1
    d = TopLogitDistiller(student, top_k=5, alpha=0.0)
    params = list(student.parameters())
    grads = lambda loss: torch.autograd.grad(loss, params, allow_unused=True)
    own, got = student.loss(tokens, targets), d.loss(tokens, targets, *d.ask(teacher, tokens))
    assert math.isclose(float(got.detach()), float(own.detach()), rel_tol=1e-5)
    top = max(float(g.abs().max()) for g in grads(student.loss(tokens, targets)) if g is not None)
    for a, b in zip(grads(got), grads(own)):
        assert (a is None) == (b is None)
        assert a is None or float((a - b).abs().max()) <= 1e-5 * top


def test_the_students_auxiliary_terms_stand_beside_the_distillation():
    teacher, student = model(1, 24), model(2, mtp_weight=0.3, num_experts=2, moe_balance_weight=0.2)
    tokens, targets = batch()
    top = TopLogitDistiller(student, top_k=5).ask(teacher, tokens)
    at = lambda alpha: float(TopLogitDistiller(student, top_k=5, alpha=alpha).loss(tokens, targets, *top).detach())
    assert math.isclose(at(0.25), 0.75 * at(0.0) + 0.25 * at(1.0), rel_tol=1e-5)
    x = student.hidden(tokens)
    logp = torch.log_softmax(x @ student.wout / 2.0, -1).gather(-1, top[0].long())
    q = torch.softmax(top[1] / 2.0, -1)
    kd = 4.0 * (q * (q.log() - logp)).sum(-1).mean()
    main = torch.nn.functional.cross_entropy((x @ student.wout).flatten(0, 1), targets.flatten())
    extra = student.loss(tokens, targets) - main      # the auxiliary terms alone
    assert math.isclose(at(1.0), float((kd + extra).detach()), rel_tol=1e-4)


def test_a_scaled_embedding_belongs_to_the_model():
    """The network that is trained with a scale is the one that is evaluated, generated from, served and saved."""
    cfg = DecoderLmConfig(dim=16, num_blocks=2, ff_dim=24, **SHAPE)
    teacher, student = DecoderLM(cfg, seed=1), DecoderLM(cfg, seed=2)
    tokens, targets = batch()
    before = student.forward(tokens)
    d = TopLogitDistiller(student, top_k=5, alpha=0.0, embed_scale=4.0)
    assert d.embed_scale == 4.0 and teacher.cfg.embed_scale == 1.0 and cfg.embed_scale == 1.0
    got, own = d.loss(tokens, targets, *d.ask(teacher, tokens)), student.loss(tokens, targets)
    assert math.isclose(float(got.detach()), float(own.detach()), rel_tol=1e-5)
    logits = student.forward(tokens)
    assert not torch.allclose(logits, before, atol=1e-4)
    # the same network with the scale in its rows
    folded = DecoderLM(cfg, seed=2)
    with torch.no_grad():
        folded.wemb *= 4.0
    assert torch.allclose(folded.forward(tokens), logits, atol=1e-5)
    assert torch.equal(student.embedding_table(), folded.wemb)
    # a second distiller keeps the student's scale
    assert TopLogitDistiller(student, top_k=5).embed_scale == 4.0
    # served: with a KV cache, and step by step
    from predicitivecoding_b200.llm.serving import InferenceModel, export_gpt
    serve = InferenceModel(student, dtype=torch.float32)
    served = serve.prefill(tokens, serve.new_cache(tokens.shape[0]))
    assert torch.allclose(served, logits if served.shape == logits.shape else logits[:, -1], atol=1e-4)
    assert torch.allclose(export_gpt(student).embedding, folded.wemb.detach(), atol=1e-6)


def test_a_scaled_embedding_is_saved_with_the_model(tmp_path):
    from predicitivecoding_b200.llm.facade import PredictiveLlm
    from predicitivecoding_b200.llm.tokenizer import ByteTokenizer
    tok = ByteTokenizer()
    llm = PredictiveLlm(DecoderLmConfig(dim=16, num_blocks=1, ff_dim=24, **{**SHAPE, "vocab": tok.vocab_size}), tok)
    TopLogitDistiller(llm.model, top_k=5, embed_scale=3.0)
    llm.save(str(tmp_path / "m"))
    again = PredictiveLlm.load(str(tmp_path / "m"))
    tokens = torch.randint(0, tok.vocab_size, (1, 9), generator=torch.Generator().manual_seed(0))
    assert again.config.embed_scale == 3.0 and torch.equal(again.model.forward(tokens), llm.model.forward(tokens))
    assert "EmbedScale" not in DecoderLmConfig(dim=16, num_blocks=1, ff_dim=24, **SHAPE).to_json()


def test_trainers_without_a_scaled_lookup_refuse_it():
    from predicitivecoding_b200.engine.fused_trainer import supports
    from predicitivecoding_b200.engine.tp_trainer import tp_supports
    from predicitivecoding_b200.llm.pc_trainer import PcDecoderTrainer
    cfg = DecoderLmConfig(64, 128, 1, 2, 128, 128, use_rms_norm=True, use_rope=True, ffn="swiglu")
    assert supports(cfg) and tp_supports(cfg, 2, 128, 1)
    assert not supports(cfg.with_(embed_scale=2.0)) and not tp_supports(cfg.with_(embed_scale=2.0), 2, 128, 1)
    with pytest.raises(NotImplementedError):
        PcDecoderTrainer(model(1, embed_scale=2.0))
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            cfg.with_(embed_scale=bad).validate()


def test_gradients_of_shared_operands_are_added_in_fp32():
    from predicitivecoding_b200.llm.distill import _Operands
    t = torch.tensor([[1.0, -3.0], [0.5, 2.0]], requires_grad=True)
    a, b, unused = _Operands.apply(t.t(), 3)
    assert a.dtype == torch.bfloat16 and a.is_contiguous() and a.data_ptr() == b.data_ptr() == unused.data_ptr()
    assert torch.equal(a.float(), t.t())
    big = torch.tensor([[1.0, 2.0], [3.0, 4.0]])
    small = big * 2.0 ** -10                         # lost in a sum of 8 bits
    ((a.float() * big).sum() + (b.float() * small).sum()).backward()
    assert torch.equal(t.grad, (big + small).t())


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("inf"), float("nan"), 1e-60, 1e60])
def test_what_is_no_temperature_is_refused(temperature):
    with pytest.raises(ValueError):
        TopLogitDistiller(model(2), top_k=5, temperature=temperature)
