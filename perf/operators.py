"""Cases of the operators at the two ends of a decoder: the embedding lookup and its gradient, the softmax cross
entropy over a large vocabulary, and the distillation from a teacher's top logits.

Each case names an operator and a direction:

    embed    lookup (x = scale * w[tok]), grad (dw from dx), both
    ce       score (per-row losses, nothing kept for a gradient), train (mean loss and the gradients of x and w)
    distill  score, train; the teacher is a list of ids and logits per row, padded with id -1

``run`` computes them in plain torch in 32 bits, or, with ``own`` set, through ``predicitivecoding_b200.ops.vocab``.
"""
import math

import torch

own = False

#: upper ends of the drawn ranges; a drawn case never asks for more than the largest listed one
MAX_EMBED = 16384 * 768          # tokens * width of a lookup with its gradient
MAX_HEAD = 4096 * 2048 * 32000   # rows * width * vocabulary of a loss with its gradient


def listed():
    return [
        # a decode step of 32 sequences at the 1.3B decoder's width: bf16 table in, fp32 residual stream out
        {"name": "embed_decode", "op": "embed", "mode": "lookup", "N": 32, "V": 32000, "D": 2048, "w": "bf16",
         "x": "fp32", "pad": 0.0, "scale": math.sqrt(2048)},
        # the 124M decoder's training batch, 16 sequences of 1024: fp32 stream and fp32 gradient arena
        {"name": "embed_train_124m", "op": "embed", "mode": "both", "N": 16384, "V": 32000, "D": 768, "w": "bf16",
         "x": "fp32", "pad": 0.0, "scale": math.sqrt(768)},
        # 2 sequences of 2048 at the 1.3B decoder's width with 16-bit activations and gradients
        {"name": "embed_grad_1p3b", "op": "embed", "mode": "grad", "N": 4096, "V": 32000, "D": 2048, "w": "bf16",
         "x": "bf16", "pad": 0.0, "scale": 1.0},
        # a ragged fp32 batch with padding, a width that fills no vector, a small odd vocabulary
        {"name": "embed_ragged", "op": "embed", "mode": "both", "N": 999, "V": 5003, "D": 101, "w": "fp32",
         "x": "fp32", "pad": 0.25, "scale": 1.0},
        # log probabilities of 32 candidate continuations (one row each) at the 1.3B decoder's head
        {"name": "ce_score_32", "op": "ce", "mode": "score", "N": 32, "V": 32000, "D": 2048, "ignored": 0.0},
        # the byte language model's head: 8 windows of 256 bytes
        {"name": "ce_byte_lm", "op": "ce", "mode": "train", "N": 2048, "V": 256, "D": 256, "ignored": 0.0},
        # the 124M decoder's head on 4 sequences of 1024
        {"name": "ce_train_124m", "op": "ce", "mode": "train", "N": 4096, "V": 32000, "D": 768, "ignored": 0.0},
        # fine-tuning with masked prompts on the small preset: ragged rows, an odd vocabulary, 60% of the rows ignored
        {"name": "ce_masked_small", "op": "ce", "mode": "train", "N": 3001, "V": 16001, "D": 384, "ignored": 0.6},
        # the 1.3B decoder's head on 2 sequences of 2048
        {"name": "ce_train_1p3b", "op": "ce", "mode": "train", "N": 4096, "V": 32000, "D": 2048, "ignored": 0.0},
        # a byte-level student (256 bytes and 4 specials) and 16 logits a row
        {"name": "distill_byte", "op": "distill", "mode": "train", "N": 512, "V": 260, "D": 256, "K": 16, "T": 2.0,
         "t": "fp32"},
        # the 124M decoder as the student of 64 stored 16-bit logits a row, 2 sequences of 1024
        {"name": "distill_124m", "op": "distill", "mode": "train", "N": 2048, "V": 32000, "D": 768, "K": 64, "T": 2.0,
         "t": "bf16"},
        # the divergence alone, on a held-out set: the small preset, an odd vocabulary
        {"name": "distill_score", "op": "distill", "mode": "score", "N": 1023, "V": 16001, "D": 384, "K": 32, "T": 1.0,
         "t": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "ce", "distill"])
    V = _log_int(rng, 200, 50000)
    D = _log_int(rng, 8, 256) * 8 if rng.random() < 0.8 else _log_int(rng, 33, 2047)
    V = min(V, max(200, 32000 * 2048 // D))
    if op == "embed":
        mode = rng.choice(["lookup", "grad", "both"])
        N = min(_log_int(rng, 1, 65536), max(1, MAX_EMBED // D))
        return {"op": op, "mode": mode, "N": N, "V": V, "D": D, "w": rng.choice(["bf16", "fp32"]),
                "x": rng.choice(["bf16", "fp32"]), "pad": rng.choice([0.0, 0.0, 0.3]),
                "scale": rng.choice([1.0, math.sqrt(D)])}
    mode = rng.choice(["train", "train", "score"])
    N = min(_log_int(rng, 1, 8192), max(1, MAX_HEAD // (V * D)))
    if op == "ce":
        return {"op": op, "mode": mode, "N": N, "V": V, "D": D, "ignored": rng.choice([0.0, 0.0, 0.3, 0.9])}
    return {"op": op, "mode": mode, "N": N, "V": V, "D": D, "K": _log_int(rng, 1, 128),
            "T": rng.choice([1.0, 1.5, 2.0, 4.0]), "t": rng.choice(["bf16", "fp32"])}


_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, V, D = case["N"], case["V"], case["D"]

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)

    def rand(*s):
        return torch.rand(*s, device="cuda", generator=g)

    def zipf(*s):   # token ids as text has them: p(id) falls off as 1 / (id + 1)
        return (torch.exp(rand(*s) * math.log(V)) - 1.0).long().clamp(0, V - 1)

    st = {"case": dict(case)}
    if case["op"] == "embed":
        tok = zipf(N)
        if case["pad"]:
            tok = torch.where(rand(N) < case["pad"], torch.full_like(tok, -1), tok)
        st["tok"] = tok
        st["w"] = (randn(V, D) * 0.02).to(_DT[case["w"]])
        if case["mode"] != "lookup":
            st["dx"] = (randn(N, D) * 1e-2).to(_DT[case["x"]])
        return st
    # a head that has learnt something: each row leans towards its own token, so its probability spreads over (0, 1)
    w = randn(V, D) * (2.0 / math.sqrt(D))
    own_token = zipf(N)
    x = randn(N, D) + w[own_token] * (rand(N, 1) * 2.0)
    st["w"], st["x"] = w.bfloat16(), x.bfloat16()
    if case["op"] == "ce":
        st["tgt"] = torch.where(rand(N) < case["ignored"], torch.full_like(own_token, -1), own_token)
        return st
    # the teacher's ids: the row's own token with the largest logit, and others spread over the vocabulary
    K, blocks = case["K"], min(V, 4 * case["K"] + 64)
    step = V // blocks
    order = rand(N, blocks).scatter_(1, (own_token // step).clamp(max=blocks - 1)[:, None], -1.0)
    ids = torch.topk(order, K, dim=1).indices * step + torch.randint(0, step, (N, K), device="cuda", generator=g)
    logits = randn(N, K) * 2.0 + 4.0
    ids[:, 0], logits[:, 0] = own_token, 11.0 + randn(N)
    shuffle = torch.argsort(rand(N, K), 1)
    ids, logits = torch.gather(ids, 1, shuffle), torch.gather(logits, 1, shuffle).to(_DT[case["t"]])
    # half of the rows have fewer than K entries, some of them none
    count = torch.where(rand(N) < 0.5, torch.full((N,), float(K), device="cuda"), torch.floor(rand(N) * (K + 1)))
    ids = torch.where(torch.arange(K, device="cuda")[None] < count[:, None], ids, torch.full_like(ids, -1))
    st["ids"], st["logits"] = ids.int(), logits
    return st


# ------------------------------------------------------------------------------------------------ the framework's
def _run_own(st):
    from predicitivecoding_b200.ops import vocab

    c = st["case"]
    if c["op"] == "embed":
        out = {}
        if c["mode"] != "grad":
            out["x"] = vocab.embed_fwd(st["tok"], st["w"], c["scale"], dtype=_DT[c["x"]])
        if c["mode"] != "lookup":
            out["dw"] = vocab.embed_bwd(st["tok"], st["dx"], c["V"], c["scale"], dtype=_DT[c["w"]])
        return out
    reduction = "none" if c["mode"] == "score" else "mean"
    if c["op"] == "ce":
        loss, saved = vocab.ce_fwd(st["x"], st["w"], st["tgt"], reduction=reduction)
    else:
        loss, saved = vocab.distill_fwd(st["x"], st["w"], st["ids"], st["logits"], c["T"], reduction=reduction)
    if c["mode"] == "score":
        return {"loss": loss}
    dx, dw = vocab.head_bwd(saved)
    return {"loss": loss, "dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------------------ plain forms
def _embed_plain(st):
    c, tok, out = st["case"], st["tok"], {}
    keep = (tok >= 0)[:, None]
    at = tok.clamp(min=0)
    if c["mode"] != "grad":
        out["x"] = (st["w"][at].float() * c["scale"] * keep).to(_DT[c["x"]])
    if c["mode"] != "lookup":
        dw = torch.zeros(c["V"], c["D"], device="cuda")
        dw.index_add_(0, at, st["dx"].float() * keep)
        out["dw"] = (dw * c["scale"]).to(_DT[c["w"]])
    return out


def _head_plain(st):
    c = st["case"]
    x, w = st["x"].float(), st["w"].float()
    T = c.get("T", 1.0)
    z = (x @ w.T) / T
    z = z - z.max(1, keepdim=True).values
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    logp = z - torch.log(s)
    if c["op"] == "ce":
        keep = st["tgt"] >= 0
        at = st["tgt"].clamp(min=0)[:, None]
        q = torch.ones_like(s)
        rows = -torch.gather(logp, 1, at)[:, 0]
    else:
        there = st["ids"] >= 0
        keep = there.any(1)
        at = st["ids"].clamp(min=0).long()
        t = torch.where(there, st["logits"].float() / T, torch.full_like(st["logits"].float(), -1e30))
        q = torch.exp(t - t.max(1, keepdim=True).values) * there
        q = q / q.sum(1, keepdim=True).clamp(min=1e-30)
        rows = T * T * (q * (torch.log(q.clamp(min=1e-38)) - torch.gather(logp, 1, at))).sum(1)
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    if c["mode"] == "score":
        return {"loss": rows}
    n = keep.sum().clamp(min=1)
    g = (e / s).scatter_add_(1, at, -q) * (keep[:, None] * (T / n))
    return {"loss": rows.sum() / n, "dx": (g @ w).bfloat16(), "dw": (g.T @ x).bfloat16()}


def run(st):
    if own:
        return _run_own(st)
    return _embed_plain(st) if st["case"]["op"] == "embed" else _head_plain(st)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "embed":
        out = {}
        valid = st["tok"] >= 0
        if case["mode"] != "grad":
            x = torch.zeros(case["N"], case["D"], device="cuda", dtype=torch.float64)
            x[valid] = st["w"].index_select(0, st["tok"][valid]).double() * case["scale"]
            out["x"] = x
        if case["mode"] != "lookup":
            pick = torch.nonzero(valid)[:, 0]
            dw = torch.zeros(case["V"], case["D"], device="cuda", dtype=torch.float64)
            dw.index_add_(0, st["tok"][pick], st["dx"][pick].double(), alpha=case["scale"])
            out["dw"] = dw
        return out
    N, V, D, T = case["N"], case["V"], case["D"], case.get("T", 1.0)
    w = st["w"].double()
    loss = torch.zeros(N, device="cuda", dtype=torch.float64)
    dx = torch.zeros(N, D, device="cuda", dtype=torch.float64)
    dw = torch.zeros(V, D, device="cuda", dtype=torch.float64)
    counted = (st["tgt"] >= 0) if case["op"] == "ce" else (st["ids"] >= 0).any(1)
    n = max(1, int(counted.sum()))
    block = max(1, min(N, 50_000_000 // V))
    for r in range(0, N, block):
        rows = torch.arange(r, min(N, r + block), device="cuda")
        rows = rows[counted[rows]]
        if not rows.numel():
            continue
        x = st["x"][rows].double()
        p = torch.zeros(rows.numel(), V, device="cuda", dtype=torch.float64)
        if case["op"] == "ce":
            p[torch.arange(rows.numel(), device="cuda"), st["tgt"][rows]] = 1.0
        else:
            ids = st["ids"][rows].long()
            t = (st["logits"][rows].double() / T).masked_fill(ids < 0, float("-inf"))
            t = torch.softmax(t, 1)
            p.scatter_add_(1, ids.clamp(min=0), t)
        logq = torch.log_softmax(x @ w.T / T, 1)
        ent = torch.special.xlogy(p, p).sum(1)
        loss[rows] = T * T * (ent - (p * logq).sum(1))
        if case["mode"] == "train":
            d = (torch.exp(logq) - p) * (T / n)
            dx[rows] = d @ w
            dw += d.T @ x
    if case["mode"] == "score":
        return {"loss": loss}
    return {"loss": loss.sum() / n, "dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    N, V, D = case["N"], case["V"], case["D"]
    if case["op"] == "embed":
        w, x = (2 if case["w"] == "bf16" else 4), (2 if case["x"] == "bf16" else 4)
        live = N * (1 - case["pad"])
        # ids are log-uniform over the vocabulary: the rows that a lookup touches, each read once
        touched = min(V, live, sum(1 - (1 - math.log1p(1 / (i + 1)) / math.log(V)) ** live for i in range(V)))
        b = f = 0
        if case["mode"] != "grad":
            b += 8 * N + touched * D * w + N * D * x
            f += live * D
        if case["mode"] != "lookup":
            b += 8 * N + live * D * x + V * D * w
            f += live * D
        return {"bytes": b, "flops": f}
    live = N * (1 - case["ignored"]) if case["op"] == "ce" else N * (1 - 0.5 / (case["K"] + 1))
    per_row = 8 if case["op"] == "ce" else case["K"] * (4 + (2 if case["t"] == "bf16" else 4))
    b = live * D * 2 + V * D * 2 + N * per_row + 4 * N
    f = 2 * live * V * D
    if case["mode"] == "train":
        b += N * D * 2 + V * D * 2
        f += 4 * live * V * D
    return {"bytes": b, "flops": f}
