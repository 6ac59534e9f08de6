"""The vocabulary ends of a decoder on the device (embedding lookup and gradient, cross entropy and distillation
without the logits) against plain statements of the same formulas in 64 bits.

Bounds.  u = 2^-8 is half a bf16 unit in the last place (relative), e = 2^-24 half an fp32 one.
  lookup        one fp32 product, one rounding: equal bit for bit
  embed grad    an fp32 sum of n terms: (n + 2) e sum |scale dx|, and u |dw| more for a bf16 result
  logits        products exact, D / 16 fp32 accumulations on the tensor cores, each off by at most one unit of the
                partial sum, which |x| |w| bounds: dl = 2 (D / 16 + 4) e |x| |w|
  losses        2 dl / T (logit and log-sum-exp) and 2^-20 of the largest logarithm in it, times T^2
  gradients     (u + 2 dl / T + 2^-18) of c (|p - q| |w|) - the rounding of p - q, the error of p - and, with p + q in
                the place of |p - q|, 2 dl / T + 2^-18 again; (V or N) e for the sums; u |dx| for a bf16 result
"""
import math

import pytest
import torch

from predicitivecoding_b200 import ops
from predicitivecoding_b200.ops import vocab

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, E = 2.0 ** -8, 2.0 ** -24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------------------ embedding
def tokens(N, V, kind, g):
    if kind == "one":
        return torch.full((N,), V // 2, device=DEV)
    if kind == "pad":
        t = torch.randint(0, V, (N,), device=DEV, generator=g)
        return torch.where(torch.rand(N, device=DEV, generator=g) < 0.5, torch.full_like(t, -1), t)
    if kind == "none":
        t = torch.full((N,), -1, device=DEV)
        t[::2] = V       # past the table
        return t
    return (torch.exp(torch.rand(N, device=DEV, generator=g) * math.log(V)) - 1).long().clamp(0, V - 1)


@pytest.mark.parametrize("N,V,D,kind", [
    (1, 1, 1, "zipf"), (1, 300, 7, "zipf"), (31, 2, 64, "zipf"), (33, 257, 100, "pad"), (2048, 32000, 96, "zipf"),
    (2049, 65536, 12, "zipf"), (5000, 70001, 33, "pad"), (4097, 77, 260, "one"), (100, 50, 32, "none"),
    (70000, 1000, 8, "zipf"), (9000, 3, 40, "one"), (640, 20, 2052, "zipf"),
])
@pytest.mark.parametrize("wt,xt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("idt", [torch.int64, torch.int32])
def test_embedding(N, V, D, kind, wt, xt, idt):
    g = gen(N + V + D)
    tok = tokens(N, V, kind, g).to(idt)
    w = torch.randn(V, D, device=DEV, generator=g).to(wt)
    scale = 1.7
    x = vocab.embed_fwd(tok, w, scale, dtype=xt)
    live = (tok >= 0) & (tok < V)
    ref = torch.where(live[:, None], w[tok.long().clamp(0, V - 1)].float() * torch.tensor(scale, device=DEV), torch.zeros((), device=DEV)).to(xt)
    assert x.dtype == xt and torch.equal(x, ref)

    dx = torch.randn(N, D, device=DEV, generator=g).to(xt)
    dx[~live] = float("nan")           # never read
    dw = vocab.embed_bwd(tok, dx, V, scale, dtype=wt)
    at = torch.nonzero(live)[:, 0]
    exact = torch.zeros(V, D, device=DEV, dtype=torch.float64)
    exact.index_add_(0, tok[at].long(), dx[at].double() * scale)
    size = torch.zeros_like(exact).index_add_(0, tok[at].long(), dx[at].double().abs() * scale)
    n = torch.bincount(tok[at].long(), minlength=V)[:, None]
    bound = (n + 2) * E * size + (U * exact.abs() if wt == torch.bfloat16 else 0)
    assert bool(((dw.double() - exact).abs() <= bound).all())
    assert torch.equal(dw, vocab.embed_bwd(tok, dx, V, scale, dtype=wt))

    start = torch.randn(V, D, device=DEV, generator=g).to(wt)
    acc = vocab.embed_bwd(tok, dx, V, scale, out=start.clone(), accumulate=True)
    exact = exact + start.double()
    bound = (n + 3) * E * (size + start.double().abs()) + (U * exact.abs() if wt == torch.bfloat16 else 0)
    assert bool(((acc.double() - exact).abs() <= bound).all())
    untouched = (n == 0).flatten()
    assert torch.equal(acc[untouched], start[untouched])


def check_embedding_grad(tok, V, dx, wt, scale=0.6):
    exact = torch.zeros(V, dx.shape[1], device=DEV, dtype=torch.float64)
    at = torch.nonzero((tok >= 0) & (tok < V))[:, 0]
    exact.index_add_(0, tok[at], dx[at].double() * scale)
    size = torch.zeros_like(exact).index_add_(0, tok[at], dx[at].double().abs() * scale)
    n = torch.bincount(tok[at], minlength=V)[:, None]
    out = torch.full((V, dx.shape[1]), float("nan"), device=DEV, dtype=wt)    # every element is written
    dw = vocab.embed_bwd(tok, dx, V, scale, out=out)
    bound = (n + 2) * E * size + (U * exact.abs() if wt == torch.bfloat16 else 0)
    assert bool(((dw.double() - exact).abs() <= bound).all())
    assert torch.equal(dw, vocab.embed_bwd(tok, dx, V, scale, dtype=wt))
    return dw


@pytest.mark.parametrize("N", [15, 16, 17, 511, 512, 513, 1023, 1024, 1025])
@pytest.mark.parametrize("V,D", [(3, 129), (2500, 40), (40000, 210)])
def test_embedding_gradient_of_few_tokens(N, V, D):
    """Either side of the sizes up to which nothing is sorted (1024 tokens, 512 into a large matrix); tokens of 16 and 17
    places, of a whole batch, met first in one part of the batch."""
    g = gen(N + V)
    dx = torch.randn(N, D, device=DEV, generator=g)
    for kind in ("zipf", "one", "pad"):
        check_embedding_grad(tokens(N, V, kind, g), V, dx, torch.float32)
    tok = torch.arange(N, device=DEV) // 17 % V                              # runs of 17, the last one shorter
    fp32 = check_embedding_grad(tok, V, dx, torch.float32)
    check_embedding_grad((torch.arange(N, device=DEV) * 7) % min(V, N // 16 + 1), V, dx.bfloat16(), torch.bfloat16)
    base = torch.randn(V, D, device=DEV, generator=g)
    both = vocab.embed_bwd(tok, dx, V, 0.6, out=base.clone(), accumulate=True)
    assert float((both - (base + fp32)).abs().max()) <= 4 * E * float((base.abs() + fp32.abs()).max())


def test_embedding_strides_and_shapes():
    g = gen(3)
    w = torch.randn(50, 80, device=DEV, generator=g)[:, 3:40]           # rows apart, unaligned
    tok = torch.randint(-1, 50, (4, 6, 2), device=DEV, generator=g)[..., 0]
    x = vocab.embed_fwd(tok, w)
    assert x.shape == (4, 6, 37)
    assert torch.equal(x, torch.where(tok[..., None] >= 0, w[tok.clamp(min=0)], torch.zeros((), device=DEV)))
    wide = torch.randn(4, 6, 96, device=DEV, generator=g)
    dx = wide[..., 8:45]
    one = torch.ones(1, 1, 1, device=DEV).expand(4, 6, 37)              # a broadcast gradient
    for d in (dx, one):
        dw = vocab.embed_bwd(tok, d, 50)
        ref = torch.zeros(50, 37, device=DEV, dtype=torch.float64)
        ref.index_add_(0, tok.clamp(min=0).flatten(), (d * (tok >= 0)[..., None]).reshape(-1, 37).double())
        assert float((dw - ref).abs().max()) <= 30 * E * float(d.abs().max()) * 24
    assert vocab.embed_fwd(tok[:0], w).shape == (0, 6, 37)
    assert float(vocab.embed_bwd(tok[:0], dx[:0], 50).abs().sum()) == 0.0


def test_embedding_autograd():
    g = gen(4)
    w = torch.randn(40, 24, device=DEV, generator=g, requires_grad=True)
    tok = torch.randint(0, 40, (3, 50), device=DEV, generator=g)
    coef = torch.randn(3, 50, 24, device=DEV, generator=g)
    (vocab.embedding(tok, w, 2.0) * coef).sum().backward()
    ref = torch.zeros(40, 24, device=DEV, dtype=torch.float64).index_add_(0, tok.flatten(), 2.0 * coef.reshape(-1, 24).double())
    assert float((w.grad - ref).abs().max()) <= 150 * E * 2 * float(coef.abs().max()) * 30


# ------------------------------------------------------------------------------------------------ head losses
def head(N, V, D, seed, spread=1.5):
    g = gen(seed)
    w = (torch.randn(V, D, device=DEV, generator=g) * (spread / math.sqrt(D))).bfloat16()
    own = torch.randint(0, V, (N,), device=DEV, generator=g)
    x = (torch.randn(N, D, device=DEV, generator=g) + w[own].float() * torch.rand(N, 1, device=DEV, generator=g)).bfloat16()
    return x, w, own, g


def teacher(N, V, K, own, g, dtype, ragged=True):
    ids = torch.stack([torch.randperm(V, device=DEV, generator=g)[:K] for _ in range(min(N, 64))])
    ids = ids.repeat((N + ids.shape[0] - 1) // ids.shape[0], 1)[:N].clone()
    t = (torch.randn(N, K, device=DEV, generator=g) * 2).to(dtype)
    if ragged:
        count = torch.randint(0, K + 1, (N,), device=DEV, generator=g)
        ids[torch.arange(K, device=DEV)[None] >= count[:, None]] = -1
        if N > 3 and K > 1:
            t[1, 0] = float("-inf")
            ids[2] = V                # none of the vocabulary's
    return ids, t


def targets64(V, tgt=None, ids=None, t=None, T=1.0, ignore=-1):
    """Dense target distribution and the counted rows."""
    if tgt is not None:
        live = (tgt >= 0) & (tgt < V) & (tgt != ignore)
        q = torch.zeros(tgt.numel(), V, device=DEV, dtype=torch.float64)
        q[live, tgt[live].long()] = 1.0
        return q, live
    there = (ids >= 0) & (ids < V) & (t.float() != float("-inf"))
    live = there.any(1)
    s = (t.double() / T).masked_fill(~there, float("-inf"))
    s[~live] = 0.0
    p = torch.softmax(s, 1) * there
    q = torch.zeros(ids.shape[0], V, device=DEV, dtype=torch.float64)
    q.scatter_add_(1, ids.clamp(0, V - 1).long(), p)
    return q, live


def check_head(x, w, q, live, T, fwd, reduction, gout=1.0, piece=0, dx_out=None, dw_out=None):
    N, D = x.shape
    V = w.shape[0]
    xs = torch.where(live[:, None], x.double(), torch.zeros((), device=DEV, dtype=torch.float64))
    z = xs @ w.double().T / T
    logp = torch.log_softmax(z, 1)
    rows = T * T * (torch.special.xlogy(q, q) - q * logp).sum(1) * live
    n = int(live.sum())
    dl = 2 * (D / 16 + 4) * E * xs.norm(dim=1) * float(w.double().norm(dim=1).max())
    logs = logp.abs().amax(1) + torch.where(q > 0, q.log().abs(), q).amax(1) + z.abs().amax(1)
    tol = (T * T * (2 * dl / T + 2.0 ** -20 * (1 + logs))) * live
    loss, state = fwd(reduction)
    if reduction == "none":
        assert loss.shape == (N,) and bool(((loss.double() - rows).abs() <= tol).all())
        return
    f = 1.0 / max(n, 1) if reduction == "mean" else 1.0
    assert loss.shape == () and abs(float(loss) - float(rows.sum() * f)) <= float(tol.sum() * f) + 1e-6 * abs(float(loss))
    dx, dw = vocab.head_bwd(state, gout, dx=dx_out, dw=dw_out, piece=piece)
    c = float(gout) * f * T
    p = torch.exp(logp)
    G = (p - q) * live[:, None]
    rel = (2 * dl / T + 2.0 ** -18)[:, None]
    B = (U * G.abs() + rel * (G.abs() + (p + q) * live[:, None])) * abs(c)
    wa, xa = w.double().abs(), xs.abs()
    for name, got, ref, bound in (("dx", dx, c * (G @ w.double()), (B + V * E * abs(c) * G.abs()) @ wa),
                                  ("dw", dw, c * (G.T @ xs), (B + N * E * abs(c) * G.abs()).T @ xa)):
        if got.dtype == torch.bfloat16:
            bound = bound + U * (ref.abs() + bound)
        over = (got.double() - ref).abs() - bound - 1e-30
        assert bool((over <= 0).all()), (name, float(over.max()))
    assert not bool(dx[~live].float().abs().sum())


SHAPES = [
    (1, 2, 8), (1, 257, 64), (2, 256, 8), (63, 1000, 40), (65, 255, 136), (255, 513, 72), (257, 300, 33), (300, 130, 256),
    (513, 1025, 7), (640, 4111, 264), (1100, 260, 512), (3, 20000, 384),
]


@pytest.mark.parametrize("N,V,D", SHAPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("mask", ["all", "some", "none"])
def test_cross_entropy(N, V, D, reduction, mask):
    x, w, tgt, g = head(N, V, D, N + V + D)
    if mask == "some":
        tgt = torch.where(torch.rand(N, device=DEV, generator=g) < 0.5, torch.full_like(tgt, -1), tgt)
        tgt[0] = V + 5
    elif mask == "none":
        tgt = torch.full_like(tgt, -100)
    q, live = targets64(V, tgt=tgt)
    x[~live] = float("nan")             # rows that are not counted are never read
    check_head(x, w, q, live, 1.0, lambda r: vocab.ce_fwd(x, w, tgt.to(torch.int32 if N % 2 else torch.int64), reduction=r),
               reduction, gout=0.7)


@pytest.mark.parametrize("N,V,D", SHAPES)
@pytest.mark.parametrize("K,T,dtype", [(1, 1.0, torch.float32), (7, 2.0, torch.bfloat16), (64, 0.5, torch.float32),
                                       (256, 4.0, torch.float32)])
def test_distillation(N, V, D, K, T, dtype):
    K = min(K, V)
    x, w, own, g = head(N, V, D, N + V + D + K)
    ids, t = teacher(N, V, K, own, g, dtype)
    q, live = targets64(V, ids=ids, t=t, T=T)
    x[~live] = float("inf")
    for reduction in ("mean", "none"):
        check_head(x, w, q, live, T, lambda r: vocab.distill_fwd(x, w, ids.to(torch.int32 if K % 2 else torch.int64), t, T, r),
                   reduction)


def test_distillation_repeated_ids():
    x, w, own, g = head(40, 300, 64, 9)
    ids = torch.randint(0, 6, (40, 12), device=DEV, generator=g)
    t = torch.randn(40, 12, device=DEV, generator=g)
    q, live = targets64(300, ids=ids, t=t, T=2.0)
    # log q of the entries, not of their sums: the entropy term differs, the gradient does not
    _, state = vocab.distill_fwd(x, w, ids, t, 2.0)
    dx, dw = vocab.head_bwd(state)
    p = torch.softmax(x.double() @ w.double().T / 2.0, 1)
    ref = 2.0 / 40 * (p - q) @ w.double()
    assert float((dx.double() - ref).norm() / ref.norm()) <= 2 * U


@pytest.mark.parametrize("piece", [1, 256, 700, 1 << 20])
def test_pieces_and_outputs(piece):
    x, w, tgt, g = head(333, 1500, 200, 5)
    tgt[::3] = -1
    q, live = targets64(1500, tgt=tgt)
    big = torch.zeros(333, 264, device=DEV)
    dx = big[:, 32:232]                                      # rows apart, fp32
    dw = torch.empty(1500, 200, device=DEV)
    check_head(x, w, q, live, 1.0, lambda r: vocab.ce_fwd(x, w, tgt, reduction=r), "mean", gout=-3.0, piece=piece,
               dx_out=dx, dw_out=dw)
    # accumulation into the shared matrix's gradient, fp32 and bf16
    _, state = vocab.ce_fwd(x, w, tgt)
    one = vocab.head_bwd(state, piece=piece, dw=torch.empty_like(dw))[1]
    for dt in (torch.float32, torch.bfloat16):
        start = torch.randn(1500, 200, device=DEV, generator=g).to(dt)
        acc = vocab.head_bwd(state, dw=start.clone(), accumulate=True, piece=piece)[1]
        ref = one.double() + start.double()
        tol = (U if dt == torch.bfloat16 else 2 * E) * ref.abs() + 2 * E * (one.abs() + start.abs())
        assert bool(((acc.double() - ref).abs() <= tol).all())
    only_dx, none = vocab.head_bwd(state, need_dw=False, piece=piece)
    assert none is None and torch.equal(only_dx, vocab.head_bwd(state, piece=piece)[0])
    none, only_dw = vocab.head_bwd(state, need_dx=False, piece=piece)
    assert none is None and torch.equal(only_dw, vocab.head_bwd(state, piece=piece)[1])


@pytest.mark.parametrize("N,V", [(256, 512), (255, 511), (257, 385), (513, 512), (900, 320), (40000, 257), (5, 33)])
@pytest.mark.parametrize("K", [0, 5, 33])
def test_vocabularies_taken_whole(N, V, K):
    """Row blocks that end inside a tile, columns that end in each of its parts, one and several blocks a pair of SMs,
    one and two terms; more targets in 32 columns than are held ahead; the loss without its gradient is the same."""
    x, w, own, g = head(N, V, 48, N + V + K)
    if K:
        ids, t = teacher(N, V, K, own, g, torch.float32)
        q, live = targets64(V, ids=ids, t=t, T=1.5)
        T, fwd = 1.5, lambda r, **k: vocab.distill_fwd(x, w, ids, t, 1.5, r, **k)
    else:
        own[1::7] = -1
        q, live = targets64(V, tgt=own)
        T, fwd = 1.0, lambda r, **k: vocab.ce_fwd(x, w, own, reduction=r, **k)
    x[~live] = float("nan")
    check_head(x, w, q, live, T, fwd, "mean", gout=1.5)
    loss, state = fwd("sum")
    first = vocab.head_bwd(state)
    for a, b in zip(first, vocab.head_bwd(state, piece=256)):   # again, from the same state
        assert torch.equal(a, b)
    alone, refused = fwd("sum", gradient=False)
    rows = fwd("none")[0].double()
    assert abs(float(alone) - float(loss)) <= 2.0 ** -19 * float(rows.abs().sum()) + 1e-5 * N
    with pytest.raises(ValueError):
        vocab.head_bwd(refused)
    assert state.status() == 0


@pytest.mark.parametrize("N", [5, 17, 32, 33])
@pytest.mark.parametrize("V,D", [(1, 8), (127, 64), (128, 72), (129, 33), (1000, 448), (4099, 520), (300, 2112)])
@pytest.mark.parametrize("K", [0, 3, 70])
def test_scoring_a_few_rows(N, V, D, K):
    """The loss of a few rows without its gradient: one to more k-blocks than a ring holds, fewer k-blocks than partial
    sums, columns that end inside a block, rows not counted, in place and from rows apart."""
    x, w, own, g = head(N, V, D, N + V + D + K)
    K = min(K, V)
    if K:
        ids, t = teacher(N, V, K, own, g, torch.float32)
        q, live = targets64(V, ids=ids, t=t, T=0.7)
        T, fwd = 0.7, lambda x, **k: vocab.distill_fwd(x, w, ids, t, 0.7, **k)
    else:
        own[1::5] = -1
        q, live = targets64(V, tgt=own)
        T, fwd = 1.0, lambda x, **k: vocab.ce_fwd(x, w, own, **k)
    x[~live] = float("nan")
    apart = torch.full((N, D + 24), float("nan"), device=DEV).bfloat16()
    apart[:, 8:8 + D] = x
    for v in (x, apart[:, 8:8 + D]):
        check_head(v, w, q, live, T, lambda r: fwd(v, reduction=r), "none")
    rows, state = fwd(x, reduction="none")
    mean, alone = fwd(x, gradient=False)
    assert state.status() == 0 and alone.status() == 0
    assert abs(float(mean) - float(rows.double().sum()) / max(int(live.sum()), 1)) <= 2.0 ** -22 * float(rows.abs().max())
    assert torch.equal(rows, fwd(x, reduction="none")[0])


def test_a_whole_vocabulary_with_infinities():
    """Logits of -inf and +inf in one row reach that row's loss and gradient, and no other row's."""
    x, w, tgt, g = head(300, 300, 64, 3)
    clean_loss = vocab.ce_fwd(x, w, tgt, reduction="none")[0]
    dx = vocab.head_bwd(vocab.ce_fwd(x, w, tgt, reduction="sum")[1], need_dw=False)[0]
    x[17] = float("inf")
    loss, state = vocab.ce_fwd(x, w, tgt, reduction="sum")
    bad = vocab.head_bwd(state, need_dw=False)[0]
    keep = torch.arange(300, device=DEV) != 17
    assert not bool(torch.isfinite(loss)) and not bool(torch.isfinite(bad[17].float()).all())
    assert torch.equal(bad[keep], dx[keep]) and bool(torch.isfinite(clean_loss).all())


@pytest.mark.parametrize("rows,ignored", [(9000, 0.5), (8193, 0.99), (600, 0.0), (257, 0.0), (256, 0.0)])
@pytest.mark.parametrize("V,piece", [(40, 0), (700, 256)])
def test_long_batches_and_the_edge_of_two_terms(rows, ignored, V, piece):
    """More rows than a block counts for itself; 256 counted rows (two-term gradients) and one more; pieces whose last
    one is short."""
    x, w, tgt, g = head(rows, V, 72, rows + V)
    tgt = torch.where(torch.rand(rows, device=DEV, generator=g) < ignored, torch.full_like(tgt, -1), tgt)
    q, live = targets64(V, tgt=tgt)
    check_head(x, w, q, live, 1.0, lambda r: vocab.ce_fwd(x, w, tgt, reduction=r), "mean", piece=piece)
    _, state = vocab.ce_fwd(x, w, tgt)
    vocab.head_bwd(state, piece=piece)
    assert state.status() == 0


@pytest.mark.parametrize("N", [1, 2, 3, 4])
@pytest.mark.parametrize("V,D,K", [(1, 8, 1), (127, 1603, 5), (129, 40, 129), (5000, 2048, 64), (300, 16, 256)])
def test_few_rows(N, V, D, K):
    """Up to 4 rows take the FMA units: losses to 2^-19 of the logarithms in them (a few roundings of sums of D
    products in nearest fp32, D^0.5 2^-24 |x| |w|), gradients with one rounding; some rows not counted; pieces."""
    x, w, tgt, g = head(N, V, D, 100 * N + V)
    ids, t = teacher(N, V, min(K, V), tgt, g, torch.float32, ragged=False)
    if N > 2:
        tgt[1] = -1
        ids[2] = -1
    for q, live, T, fwd in ((*targets64(V, tgt=tgt), 1.0, lambda r: vocab.ce_fwd(x, w, tgt, reduction=r)),
                            (*targets64(V, ids=ids, t=t, T=2.0), 2.0, lambda r: vocab.distill_fwd(x, w, ids, t, 2.0, r))):
        loss, _ = fwd("none")
        z = x.double() @ w.double().T / T
        logp = torch.log_softmax(z, 1)
        rows = T * T * (torch.special.xlogy(q, q) - q * logp).sum(1) * live
        logs = logp.abs().amax(1) + z.abs().amax(1) + torch.where(q > 0, q.log().abs(), q).amax(1)
        tol = T * T * (2.0 ** -19 * (1 + logs) + 8 * D ** 0.5 * E * x.double().norm(dim=1) * w.double().norm(dim=1).max())
        assert bool(((loss.double() - rows).abs() <= tol).all())
        for piece in (0, 256):
            check_head(x, w, q, live, T, fwd, "mean", gout=0.5, piece=piece)
    wide = torch.randn(V, D + 13, device=DEV, generator=g).bfloat16()      # rows of w that no vector fits
    wide[:, 3:D + 3] = w
    a, b = vocab.ce_fwd(x, wide[:, 3:D + 3], tgt)[0], vocab.ce_fwd(x, w, tgt)[0]
    assert torch.equal(a, b)


def test_few_rows_round_the_gradient_once():
    """Up to 256 counted rows p - q has two terms: the bf16 result is off by its own rounding and 2^-14 more."""
    x, w, tgt, g = head(5, 3000, 256, 21)
    _, state = vocab.ce_fwd(x, w, tgt)
    dx, dw = vocab.head_bwd(state)
    q, live = targets64(3000, tgt=tgt)
    G = (torch.softmax(x.double() @ w.double().T, 1) - q) / 5
    for got, ref, size in ((dx, G @ w.double(), G.abs() @ w.double().abs()), (dw, G.T @ x.double(), G.T.abs() @ x.double().abs())):
        assert bool(((got.double() - ref).abs() <= U * ref.abs() + 2.0 ** -14 * size).all())


def test_top_logit_distiller_on_the_device():
    """The distiller's loss and gradients on the device against the CPU's.  The device rounds the head's operands to
    bf16 (2^-8 each, logits of size |x| |w|) and takes its matrix products in fp32."""
    from predicitivecoding_b200.llm.distill import TopLogitDistiller
    from predicitivecoding_b200.models.config import DecoderLmConfig
    from predicitivecoding_b200.models.decoder_lm import DecoderLM
    cfg = DecoderLmConfig(vocab=260, dim=64, num_blocks=2, num_heads=4, ff_dim=96, max_seq=32, use_rms_norm=True,
                          use_rope=True, ffn="swiglu")
    teacher, student = DecoderLM(cfg, seed=1), DecoderLM(cfg, seed=2)
    tokens = torch.randint(0, 260, (3, 33), generator=torch.Generator().manual_seed(1))
    x, y = tokens[:, :-1], tokens[:, 1:].clone()
    y[0, :9] = -1
    d = TopLogitDistiller(student, top_k=7, temperature=2.0, alpha=0.4, embed_scale=8.0)
    ids, logits = d.ask(teacher, x)
    want = d.loss(x, y, ids, logits)
    grads = torch.autograd.grad(want, (student.wemb, student.wout))
    size = float((student.hidden(x).norm(dim=-1).max() * student.wout.norm(dim=0).max()).detach())
    student.to(DEV)
    got = d.loss(x.to(DEV), y.to(DEV), ids.to(DEV), logits.to(DEV))
    assert abs(float(got.detach()) - float(want.detach())) <= 2 * 2 * U * size + 1e-4
    for a, b in zip(torch.autograd.grad(got, (student.wemb, student.wout)), grads):
        assert float((a.cpu() - b).norm() / b.norm()) <= 8 * U


def test_strides_and_leading_shapes():
    x, w, tgt, g = head(96, 700, 48, 6)
    wide = torch.randn(700, 101, device=DEV, generator=g).bfloat16()
    wide[:, 5:53] = w
    big = torch.randn(4, 24, 111, device=DEV, generator=g).bfloat16()
    big[..., 1:49] = x.view(4, 24, 48)
    loss0, s0 = vocab.ce_fwd(x, w, tgt)
    loss1, s1 = vocab.ce_fwd(big[..., 1:49], wide[:, 5:53], tgt.view(4, 24))
    assert torch.equal(loss0, loss1)
    for a, b in zip(vocab.head_bwd(s0), vocab.head_bwd(s1)):
        assert torch.equal(a.flatten(), b.flatten())
    # one row for all: a broadcast x and a broadcast w
    xb, wb = x[:1].expand(96, 48), w[:1].expand(700, 48)
    check_head(xb, wb, *targets64(700, tgt=tgt), 1.0, lambda r: vocab.ce_fwd(xb, wb, tgt, reduction=r), "mean")
    none = vocab.ce_fwd(x[:0], w, tgt[:0], reduction="none")
    assert none[0].shape == (0,)
    loss, s = vocab.ce_fwd(x[:0], w, tgt[:0])
    dx, dw = vocab.head_bwd(s)
    assert float(loss) == 0.0 and dx.shape == (0, 48) and not bool(dw.float().abs().sum())


def test_ignore_index_in_the_vocabulary():
    x, w, tgt, g = head(200, 64, 32, 8)
    tgt[5] = 3
    q, live = targets64(64, tgt=tgt, ignore=3)
    check_head(x, w, q, live, 1.0, lambda r: vocab.ce_fwd(x, w, tgt, 3, r), "mean")


@pytest.mark.parametrize("scale", [1e-3, 30.0, 300.0])
def test_extreme_logits(scale):
    """Flat and one-hot softmaxes: logits of a few thousand neither overflow nor leave a NaN."""
    x, w, tgt, g = head(130, 900, 64, 10)
    x = (x.float() * scale).bfloat16()
    q, live = targets64(900, tgt=tgt)
    check_head(x, w, q, live, 1.0, lambda r: vocab.ce_fwd(x, w, tgt, reduction=r), "mean")


def test_nan_reaches_its_row_only():
    x, w, tgt, g = head(70, 300, 32, 11)
    x[7, 3] = float("nan")
    loss, _ = vocab.ce_fwd(x, w, tgt, reduction="none")
    bad = torch.isnan(loss)
    assert bool(bad[7]) and int(bad.sum()) == 1
    ids, t = teacher(70, 300, 5, tgt, g, torch.float32, ragged=False)
    t[9, 2] = float("nan")
    loss, _ = vocab.distill_fwd(x, w, ids, t, 1.0, "none")
    assert sorted(torch.nonzero(torch.isnan(loss))[:, 0].tolist()) == [7, 9]


def test_gradient_against_differences():
    """d loss / d t along x + t a and w + t b, a and b exact in bf16, against central differences of the device's
    own loss.  With E = max |logit change| per unit t, the third derivative of a row's loss is at most 8 E^3 and its
    rounding is bounded as in check_head."""
    N, V, D, h = 24, 90, 16, 2.0 ** -5
    g = gen(12)
    q8 = lambda s, n: torch.randint(-n, n + 1, s, device=DEV, generator=g).float()
    x, w = q8((N, D), 8) / 8, q8((V, D), 8) / 16
    a, b = q8((N, D), 1) / 4, q8((V, D), 1) / 8
    tgt = torch.randint(0, V, (N,), device=DEV, generator=g)
    ids, t = teacher(N, V, 6, tgt, g, torch.float32)
    for fwd, T in ((lambda x, w: vocab.ce_fwd(x, w, tgt, reduction="sum"), 1.0),
                   (lambda x, w: vocab.distill_fwd(x, w, ids, t, 2.0, "sum"), 2.0)):
        for da, db in ((a, None), (None, b)):
            at = lambda s: (x if da is None else x + s * da, w if db is None else w + s * db)
            losses = []
            for s in (h, -h):
                xs, ws = at(s)
                assert torch.equal(xs.bfloat16().float(), xs) and torch.equal(ws.bfloat16().float(), ws)
                losses.append(float(fwd(xs.bfloat16(), ws.bfloat16())[0]))
            _, state = fwd(x.bfloat16(), w.bfloat16())
            dx, dw = vocab.head_bwd(state, dx=torch.empty(N, D, device=DEV), dw=torch.empty(V, D, device=DEV))
            got = float((dx * da).sum() if da is not None else (dw * db).sum())
            e = float(((da @ w.T) if da is not None else (x @ db.T)).abs().max()) / T
            third = N * T * T * 8 * e ** 3 * h * h / 6
            rounding = 2 * N * T * T * 2.0 ** -18 / (2 * h)
            grads = U * 2 * N * T * T * e * 2
            assert abs((losses[0] - losses[1]) / (2 * h) - got) <= third + rounding + grads


def test_autograd_and_other_stream():
    x, w, tgt, g = head(128, 500, 64, 13)
    ids, t = teacher(128, 500, 9, tgt, g, torch.float32)
    for f, s in ((lambda x, w: vocab.cross_entropy(x, w, tgt), lambda: vocab.ce_fwd(x, w, tgt)),
                 (lambda x, w: vocab.distill(x, w, ids, t, 3.0), lambda: vocab.distill_fwd(x, w, ids, t, 3.0))):
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        f(xg, wg).backward()
        loss, state = s()
        dx, dw = vocab.head_bwd(state)
        assert torch.equal(xg.grad, dx) and torch.equal(wg.grad, dw)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            loss2, state2 = s()
            dx2, dw2 = vocab.head_bwd(state2)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(loss, loss2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
        xg.grad = None
        (f(xg, wg) * 0.5).backward()
        half = vocab.head_bwd(state, torch.tensor(0.5, device=DEV))[0]
        assert torch.equal(xg.grad, half)


def test_graph_capture():
    x, w, tgt, g = head(256, 600, 64, 14)
    tok = torch.randint(0, 600, (256,), device=DEV, generator=g)
    step = lambda: (vocab.embed_fwd(tok, w, 2.0), *vocab.head_bwd(vocab.ce_fwd(x, w, tgt)[1]),
                    vocab.embed_bwd(tok, x, 600, 2.0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    tgt.copy_(torch.where(torch.arange(256, device=DEV) % 2 == 0, tgt, torch.full_like(tgt, -1)))   # other counted rows
    graph.replay()
    for a, b in zip(outs, step()):
        assert torch.equal(a, b)


def test_refusals():
    x, w, tgt, g = head(8, 40, 16, 15)
    ids, t = teacher(8, 40, 4, tgt, g, torch.float32)
    bad = [
        lambda: vocab.ce_fwd(x.float(), w, tgt), lambda: vocab.ce_fwd(x, w.float(), tgt), lambda: vocab.ce_fwd(x, w, tgt.float()),
        lambda: vocab.ce_fwd(x, w[:, :8], tgt), lambda: vocab.ce_fwd(x, w, tgt[:4]), lambda: vocab.ce_fwd(x, w, tgt, reduction="max"),
        lambda: vocab.ce_fwd(x.cpu(), w, tgt), lambda: vocab.ce_fwd(x, w, tgt.cpu()), lambda: vocab.ce_fwd(x, w[:0], tgt),
        lambda: vocab.distill_fwd(x, w, ids, t, 0.0), lambda: vocab.distill_fwd(x, w, ids, t, float("inf")),
        lambda: vocab.distill_fwd(x, w, ids, t[:, :2]), lambda: vocab.distill_fwd(x, w, ids[:, :0], t[:, :0]),
        lambda: vocab.distill_fwd(x, w, ids.repeat(1, 65), t.repeat(1, 65)), lambda: vocab.distill_fwd(x, w, ids, t.half()),
        lambda: vocab.head_bwd(vocab.ce_fwd(x, w, tgt, reduction="none")[1]),
        lambda: vocab.head_bwd(vocab.ce_fwd(x, w, tgt)[1], accumulate=True),
        lambda: vocab.head_bwd(vocab.ce_fwd(x, w, tgt)[1], dx=torch.empty(8, 8, device=DEV)),
        lambda: vocab.head_bwd(vocab.ce_fwd(x, w, tgt)[1], dw=torch.empty(40, 16)),
        lambda: vocab.head_bwd(vocab.ce_fwd(x, w, tgt)[1], gout=torch.ones(2, device=DEV)),
        lambda: vocab.head_bwd(vocab.ce_fwd(x, w, tgt)[1], piece=-1),
        lambda: vocab.embed_fwd(tgt.float(), w), lambda: vocab.embed_fwd(tgt, w.half()), lambda: vocab.embed_fwd(tgt, w.t()),
        lambda: vocab.embed_fwd(tgt, w, dtype=torch.float16), lambda: vocab.embed_fwd(tgt, w, out=torch.empty(8, 4, device=DEV)),
        lambda: vocab.embed_fwd(tgt, w[0]), lambda: vocab.embed_fwd(tgt.cpu(), w),
        lambda: vocab.embed_bwd(tgt, x[:4], 40), lambda: vocab.embed_bwd(tgt, x, 0), lambda: vocab.embed_bwd(tgt, x.half(), 40),
        lambda: vocab.embed_bwd(tgt, x, 40, out=torch.empty(40, 8, device=DEV)),
        lambda: vocab.embed_bwd(tgt, x, 40, accumulate=True), lambda: vocab.embed_bwd(tgt.cpu(), x, 40),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    torch.cuda.synchronize()
    assert ops.launch_count() > 0
