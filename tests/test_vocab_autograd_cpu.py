"""What the autograd forms of the vocabulary-end operators promise around their kernels, on the CPU: the extension's
entry points are replaced by plain stand-ins of the same formulas."""
import pytest
import torch

from predicitivecoding_b200.ops import vocab


@pytest.fixture
def plain(monkeypatch):
    """Entry points in plain torch; a loss's state is the tensors that its gradient needs."""
    def embed_bwd(tok, dx, vocab_size, scale=1.0, out=None, dtype=torch.float32, accumulate=False):
        return torch.zeros(vocab_size, dx.shape[-1], dtype=dx.dtype).index_add_(0, tok, dx * scale).to(dtype)

    def fwd(reference):
        def call(x, w, *args, gradient=True):
            *args, reduction = args
            return reference(x, w, *args, reduction), (reference, x, w, args, reduction)
        return call

    def head_bwd(state, gout=1.0, need_dx=True, need_dw=True, **_):
        reference, x, w, args, reduction = state
        with torch.enable_grad():
            x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
            dx, dw = torch.autograd.grad(reference(x, w, *args, reduction), (x, w), gout.to(x.dtype))
        return dx if need_dx else None, dw if need_dw else None

    monkeypatch.setattr(vocab, "embed_fwd", lambda tok, w, scale=1.0, out=None, dtype=torch.float32: (w[tok] * scale).to(dtype))
    monkeypatch.setattr(vocab, "embed_bwd", embed_bwd)
    monkeypatch.setattr(vocab, "ce_fwd", fwd(vocab.reference_cross_entropy))
    monkeypatch.setattr(vocab, "distill_fwd", fwd(vocab.reference_distill))
    monkeypatch.setattr(vocab, "head_bwd", head_bwd)


def operands(N=6, V=11, D=4, K=3):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(N, D, generator=g).requires_grad_()
    w = torch.randn(V, D, generator=g).requires_grad_()
    return x, w, torch.randint(0, V, (N,), generator=g), torch.randint(0, V, (N, K), generator=g), torch.randn(N, K, generator=g)


def scalar_forms(x, w, tgt, ids, logits):
    return {
        "embedding": lambda: (vocab.embedding(tgt, w, 2.0) ** 2).sum(),
        "cross_entropy": lambda: vocab.cross_entropy(x, w, tgt),
        "distill": lambda: vocab.distill(x, w, ids, logits, 2.0, "sum"),
    }


@pytest.mark.parametrize("form", ["embedding", "cross_entropy", "distill"])
def test_a_gradient_of_a_gradient_is_refused(plain, form):
    """The backwards are kernels without a gradient of their own: a penalty on a gradient raises instead of
    contributing nothing."""
    x, w, *rest = operands()
    f = scalar_forms(x, w, *rest)[form]
    first, = torch.autograd.grad(f(), w)
    graph, = torch.autograd.grad(f(), w, create_graph=True)
    assert torch.equal(first, graph)
    with pytest.raises(RuntimeError, match="differentia"):
        ((graph ** 2).sum() + (w ** 2).sum()).backward()


@pytest.mark.parametrize("form", ["cross_entropy", "distill"])
def test_a_gradient_of_row_losses_is_refused(plain, form):
    """Per-row losses have no gradient: weighted rows in a sum with another loss raise instead of training nothing.
    Without a gradient wanted they are plain values."""
    x, w, tgt, ids, logits = operands()
    f = ((lambda: vocab.cross_entropy(x, w, tgt, reduction="none")) if form == "cross_entropy" else
         (lambda: vocab.distill(x, w, ids, logits, 2.0, "none")))
    rows = f()
    weights = torch.arange(6.0)
    with pytest.raises(RuntimeError, match="none"):
        ((rows * weights).sum() + (x ** 2).sum()).backward()
    with torch.no_grad():
        alone = f()
    assert not alone.requires_grad and torch.equal(alone, rows.detach())
