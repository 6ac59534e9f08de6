"""The vocabulary-end kernels on either side of the sizes where another variant takes over: sums of logits in two halves,
both terms of the gradient of the logits from each kernel that makes it, and the sort's widths."""
import pytest
import torch

from predicitivecoding_b200.ops import vocab
from test_vocab_gpu import DEV, E, U, check_embedding_grad, check_head, gen, head, targets64, teacher, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [5, 128, 255, 256, 257])
@pytest.mark.parametrize("D", [1016, 1024, 1032, 2048])
@pytest.mark.parametrize("V,K", [(300, 0), (1500, 0), (1500, 40)])
def test_logits_in_two_halves(N, D, V, K):
    """Up to 256 rows of 1024 or more columns: two accumulators take half of the sum each; an odd number of k-blocks, row
    blocks of one and of both CTAs, rows not counted, pieces."""
    x, w, own, g = head(N, V, D, N + V + D + K)
    if K:
        ids, t = teacher(N, V, K, own, g, torch.bfloat16)
        q, live = targets64(V, ids=ids, t=t, T=2.0)
        T, fwd = 2.0, lambda r: vocab.distill_fwd(x, w, ids, t, 2.0, r)
    else:
        own[1::4] = -1
        q, live = targets64(V, tgt=own)
        T, fwd = 1.0, lambda r: vocab.ce_fwd(x, w, own, reduction=r)
    x[~live] = float("nan")
    for reduction, piece in (("mean", 0), ("sum", 0), ("mean", 256)):
        check_head(x, w, q, live, T, fwd, reduction, gout=0.7, piece=piece)
    loss, state = fwd("sum")
    first = vocab.head_bwd(state)
    assert all(torch.equal(a, b) for a, b in zip(first, vocab.head_bwd(fwd("sum")[1])))
    assert state.status() == 0


@pytest.mark.parametrize("N,V,D", [
    (1, 3000, 256), (4, 3000, 1032),        # the FMA units
    (5, 3000, 256), (256, 3000, 256),       # pair products
    (5, 3000, 1024), (256, 700, 2048),      # in two halves
    (5, 400, 256), (256, 512, 64),          # whole vocabularies
    (700, 400, 64), (700, 3000, 256),       # few counted rows of many
])
@pytest.mark.parametrize("kind", ["ce", "distill"])
def test_both_terms_reach_the_gradient(N, V, D, kind):
    """Up to 256 counted rows p - q has two bf16 terms, 2^-14 of it left out.  With 3 rows counted at most, x small (so
    that the logits' error, 2 (D / 16 + 4) e |x| |w|, is small too) and an fp32 result, every element of dw shows a missing
    second term, which is up to 2^-9 of p - q."""
    x, w, own, g = head(N, V, D, N + V + D)
    x = (x.float() / 32).bfloat16()
    counted = torch.zeros(N, dtype=torch.bool, device=DEV)
    counted[torch.tensor([0, N // 2, N - 1], device=DEV)] = True
    if kind == "ce":
        own[~counted] = -1
        q, live = targets64(V, tgt=own)
        T, state = 1.0, vocab.ce_fwd(x, w, own, reduction="sum")[1]
    else:
        ids, t = teacher(N, V, 9, own, g, torch.float32, ragged=False)
        ids[~counted] = -1
        q, live = targets64(V, ids=ids, t=t, T=2.0)
        T, state = 2.0, vocab.distill_fwd(x, w, ids, t, 2.0, "sum")[1]
    dw = vocab.head_bwd(state, need_dx=False, dw=torch.empty(V, D, device=DEV))[1].double()
    xs, n = x[live].double(), int(live.sum())
    p = torch.softmax(xs @ w.double().T / T, 1)
    G = p - q[live]
    dl = 2 * (D / 16 + 4) * E * xs.norm(dim=1) * float(w.double().norm(dim=1).max())
    rel = (2 * dl / T + 2.0 ** -18)[:, None]
    B = T * (2.0 ** -14 * G.abs() + rel * (G.abs() + p + q[live]))
    bound = B.T @ xs.abs() + 4 * n * E * T * (G.abs().T @ xs.abs())
    exact = T * G.T @ xs
    assert bool(((dw - exact).abs() <= bound).all())
    one = T * G.float().bfloat16().double().T @ xs              # the first terms alone
    assert float(((one - exact).abs() > bound).double().mean()) > 0.05


@pytest.mark.parametrize("N", [8192, 8193, 16384, 16385, 32768, 32769, 65536, 65537])
@pytest.mark.parametrize("V,D", [(200, 40), (70001, 12)])
def test_embedding_gradient_at_the_sorts_widths(N, V, D):
    """1, 2, 4 and 8 keys a thread, and the first batch that no cluster holds; one to three digits a key."""
    g = gen(N + V)
    dx = torch.randn(N, D, device=DEV, generator=g)
    for kind in ("zipf", "pad"):
        check_embedding_grad(tokens(N, V, kind, g), V, dx, torch.float32)
    check_embedding_grad(torch.arange(N, device=DEV).flip(0) * 7 % V, V, dx.bfloat16(), torch.bfloat16)


def test_top_logit_distiller_with_a_second_head_on_the_device():
    """Value and gradients against the CPU's, with a multi-token head: operands of both heads rounded to bf16 (2^-8 each,
    logits of size |x| |w|; their terms weigh 1 + 0.3 together)."""
    from predicitivecoding_b200.llm.distill import TopLogitDistiller
    from predicitivecoding_b200.models.config import DecoderLmConfig
    from predicitivecoding_b200.models.decoder_lm import DecoderLM
    cfg = DecoderLmConfig(vocab=260, dim=64, num_blocks=2, num_heads=4, ff_dim=96, max_seq=32, use_rms_norm=True,
                          use_rope=True, ffn="swiglu", mtp_weight=0.3)
    teacher_, student = DecoderLM(cfg, seed=1), DecoderLM(cfg, seed=2)
    rows = torch.randint(0, 260, (3, 33), generator=torch.Generator().manual_seed(1))
    x, y = rows[:, :-1], rows[:, 1:].clone()
    y[0, :9] = -100
    d = TopLogitDistiller(student, top_k=7, temperature=2.0, alpha=0.4, embed_scale=8.0)
    ids, logits = d.ask(teacher_, x)
    params = lambda: (student.wemb, student.wout, student.wout_mtp)
    want = d.loss(x, y, ids, logits)
    grads = torch.autograd.grad(want, params())
    norms = max(float(w.norm(dim=0).max().detach()) for w in (student.wout, student.wout_mtp))
    size = float(student.hidden(x).norm(dim=-1).max().detach()) * norms
    student.to(DEV)
    got = d.loss(x.to(DEV), y.to(DEV), ids.to(DEV), logits.to(DEV))
    assert abs(float(got.detach()) - float(want.detach())) <= 1.3 * 2 * 2 * U * size + 1e-4
    for a, b in zip(torch.autograd.grad(got, params()), grads):
        assert float((a.cpu() - b).norm() / b.norm()) <= 8 * U


def test_the_distillers_two_heads_are_added_without_another_rounding():
    """With weights of 1/2 (exact) the gradient of the output matrix is half of the two terms' own, added in fp32."""
    from predicitivecoding_b200.llm.distill import TopLogitDistiller
    from predicitivecoding_b200.models.config import DecoderLmConfig
    from predicitivecoding_b200.models.decoder_lm import DecoderLM
    cfg = DecoderLmConfig(vocab=900, dim=64, num_blocks=1, num_heads=4, ff_dim=96, max_seq=32, use_rms_norm=True, use_rope=True)
    student, teacher_ = DecoderLM(cfg, seed=2).to(DEV), DecoderLM(cfg, seed=1).to(DEV)
    rows = torch.randint(0, 900, (3, 33), generator=torch.Generator().manual_seed(1)).to(DEV)
    x, y = rows[:, :-1], rows[:, 1:]
    top = TopLogitDistiller(student, top_k=7).ask(teacher_, x)
    grad = lambda alpha: torch.autograd.grad(TopLogitDistiller(student, top_k=7, alpha=alpha).loss(x, y, *top), student.wout)[0]
    assert torch.equal(grad(0.5), 0.5 * grad(0.0) + 0.5 * grad(1.0))
