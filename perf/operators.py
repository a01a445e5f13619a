"""Performance cases of the model-side operators: the token embedding, the router of a mixture-of-experts layer and the loss over
the vocabulary, with their gradients.  They stand around the tensor-parallel layers and the expert exchange of `perf/cases.py`.

listed() names the cases, draw() makes more of the same ranges.  run() computes them in their plain form (elementary torch
operations in 32 bits, rounded once at the end), or, where `own` is true, with the library's kernels; exact() states them in 64 bits.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
IGNORE = -100


def listed():
    return [
        # a decode step of eight sequences: one row each, the call's latency is all there is
        {"name": "embed_decode_8", "kind": "embed", "tokens": 8, "vocab": 32000, "hidden": 4096, "dtype": "bfloat16", "scale": 1.0},
        # a prefill batch at the hidden size of the benchmark's MLP, scaled by sqrt(hidden)
        {"name": "embed_prefill_16384", "kind": "embed", "tokens": 16384, "vocab": 128256, "hidden": 8192, "dtype": "bfloat16", "scale": 90.5},
        # gradient of a small batch in fp32: rows that are not whole vectors, most of the table untouched
        {"name": "embed_grad_odd_fp32", "kind": "embed_grad", "tokens": 1531, "vocab": 50257, "hidden": 1001, "dtype": "float32", "scale": 1.0},
        # gradient of a training batch: frequent tokens repeat thousands of times
        {"name": "embed_grad_32768", "kind": "embed_grad", "tokens": 32768, "vocab": 128256, "hidden": 4096, "dtype": "bfloat16", "scale": 64.0},
        # scores of a few tokens (likelihood of an answer): the weights are read once
        {"name": "loss_eval_7", "kind": "loss", "tokens": 7, "vocab": 32000, "hidden": 4096},
        # evaluation of a batch: loss per token, no gradients
        {"name": "loss_eval_4096", "kind": "loss", "tokens": 4096, "vocab": 128256, "hidden": 4096},
        # training with odd sizes and a weight for each token
        {"name": "loss_train_odd", "kind": "loss_grad", "tokens": 1531, "vocab": 50257, "hidden": 1000, "weighted": True},
        # training step of a batch: the largest products
        {"name": "loss_train_8192", "kind": "loss_grad", "tokens": 8192, "vocab": 128256, "hidden": 4096, "weighted": False},
        # router of a decode batch
        {"name": "route_decode_16", "kind": "route", "tokens": 16, "experts": 64, "topk": 8, "dtype": "float32", "masked": False},
        # router of the benchmark's exchange: 8192 tokens, 256 experts, top 8
        {"name": "route_prefill_8192", "kind": "route", "tokens": 8192, "experts": 256, "topk": 8, "dtype": "float32", "masked": False},
        # router of a padded batch in training, odd sizes, logits as a bf16 layer leaves them: equal logits occur
        {"name": "route_train_odd", "kind": "route_grad", "tokens": 2371, "experts": 60, "topk": 4, "dtype": "bfloat16", "masked": True},
        # router of a large training batch, with gradients
        {"name": "route_train_65536", "kind": "route_grad", "tokens": 65536, "experts": 256, "topk": 8, "dtype": "float32", "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "loss", "loss_grad", "loss_grad", "route", "route_grad"])
    if kind in ("embed", "embed_grad"):
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        while True:
            hidden = rng.choice([64 * rng.randint(1, 128), 8 * rng.randint(8, 1024), rng.randint(64, 8192)])
            vocab, tokens = _log(rng, 1000, 160000), _log(rng, 1, 32768)
            if vocab * hidden * SIZE[dtype] <= 128256 * 8192 * 2 and tokens * hidden * SIZE[dtype] <= 32768 * 8192 * 2:
                break
        return {"kind": kind, "tokens": tokens, "vocab": vocab, "hidden": hidden, "dtype": dtype, "scale": rng.choice([1.0, round(math.sqrt(hidden), 2)])}
    if kind in ("loss", "loss_grad"):
        while True:
            tokens, vocab = _log(rng, 1, 16384), _log(rng, 1000, 160000)
            hidden = 8 * _log(rng, 16, 1024)
            if rng.random() < 0.5:
                hidden = (hidden + 63) // 64 * 64
            work = tokens * vocab * hidden
            if work <= 8192 * 128256 * 4096 and tokens * vocab <= 8192 * 128256 and vocab * hidden <= 128256 * 4096:
                break
        case = {"kind": kind, "tokens": tokens, "vocab": vocab, "hidden": hidden}
        if kind == "loss_grad":
            case["weighted"] = rng.random() < 0.3
        return case
    experts = rng.choice([8, 16, 64, 128, 256, 512, rng.randint(8, 512)])
    return {"kind": kind, "tokens": _log(rng, 1, min(65536, 65536 * 256 // experts)), "experts": experts, "topk": min(experts, rng.choice([1, 2, 4, 6, 8])),
            "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]), "masked": rng.random() < 0.3}


# ---------------------------------------------------------------------------------------------------------- inputs
def _words(n, vocab, g):
    """Token ids as text has them: frequencies fall as the inverse of the rank, the most frequent one is about six in a hundred."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    rank = (float(vocab) ** u).long().clamp_(1, vocab) - 1
    return (rank * 7919) % vocab if vocab % 7919 else rank


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s, kind = dict(case), case["kind"]
    T = case["tokens"]
    if kind in ("embed", "embed_grad"):
        V, H, dt = case["vocab"], case["hidden"], TYPES[case["dtype"]]
        s["ids"] = _words(T, V, g)
        if kind == "embed":
            s["w"] = torch.empty(V, H, device="cuda", dtype=dt).normal_(0, 0.02, generator=g)
        else:
            s["dy"] = torch.empty(T, H, device="cuda", dtype=dt).normal_(0, 1e-2, generator=g)
    elif kind in ("loss", "loss_grad"):
        V, H = case["vocab"], case["hidden"]
        w = torch.empty(V, H, device="cuda", dtype=torch.bfloat16).normal_(0, 1.3 / math.sqrt(H), generator=g)
        y = _words(T, V, g)
        # what the model has learnt: its hidden state leans towards the next token, from not at all to a sure guess
        lean = torch.rand(T, 1, device="cuda", generator=g) * 12
        x = torch.randn(T, H, device="cuda", generator=g) + lean * w[y].float() / 1.3
        s["x"], s["w"] = x.to(torch.bfloat16), w
        if T > 2:  # prompts and padding are not trained on
            y = torch.where(torch.rand(T, device="cuda", generator=g) < 0.05, torch.full_like(y, IGNORE), y)
        s["y"] = y
        s["weights"] = torch.rand(T, device="cuda", generator=g) + 0.5 if case.get("weighted") else None
    else:
        E, k = case["experts"], case["topk"]
        s["logits"] = (torch.randn(T, E, device="cuda", generator=g) + 0.5 * torch.randn(E, device="cuda", generator=g)).to(TYPES[case["dtype"]])
        s["mask"] = torch.rand(T, device="cuda", generator=g) < 0.85 if case["masked"] else None
        if kind == "route_grad":
            s["dgates"] = torch.randn(T, k, device="cuda", generator=g) * 1e-2
            s["coef"] = 1e-2
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _loss_plain(s, grad):
    """Losses per token; with `grad` the weighted mean and its gradients (weights of tokens without a target are zero)."""
    xf, wf, y = s["x"].float(), s["w"].float(), s["y"]
    valid = (y >= 0) & (y < wf.shape[0])
    at = torch.where(valid, y, torch.zeros_like(y))
    logits = xf @ wf.t()
    top = logits.max(dim=1, keepdim=True).values
    target = logits.gather(1, at[:, None])
    e = torch.exp(logits - top)
    z = e.sum(dim=1, keepdim=True)
    losses = torch.where(valid, (torch.log(z) + (top - target))[:, 0], torch.zeros_like(top[:, 0]))
    if not grad:
        return losses
    weight = valid.float() if s["weights"] is None else valid.float() * s["weights"]
    total = weight.sum()
    share = torch.where(total > 0, weight / total, torch.zeros_like(weight))
    ds = e.mul_(share[:, None] / z)
    ds[torch.arange(len(at), device=at.device), at] -= share
    return (losses * share).sum(), (ds @ wf).to(s["x"].dtype), (ds.t() @ xf).to(s["w"].dtype)


def _route_plain(s):
    l, k = s["logits"].float(), s["topk"]
    ok = (l > -math.inf).any(dim=1)
    if s["mask"] is not None:
        ok = ok & s["mask"]
    top = l.max(dim=1, keepdim=True).values
    e = torch.exp(l - top)
    p = torch.where(ok[:, None], e / e.sum(dim=1, keepdim=True), torch.zeros_like(l))
    order = torch.sort(l, dim=1, descending=True, stable=True)  # equal logits: the lowest expert first
    chosen = ok[:, None] & (order.values[:, :k] > -math.inf)
    idx = torch.where(chosen, order.indices[:, :k], torch.full_like(order.indices[:, :k], -1))
    picked = torch.where(chosen, p.gather(1, order.indices[:, :k]), torch.zeros_like(p[:, :k]))
    whole = picked.sum(dim=1, keepdim=True)
    gates = torch.where(whole > 0, picked / whole, torch.zeros_like(picked))
    slots = (idx[:, :, None] == torch.arange(l.shape[1], device=l.device)) if l.shape[0] * k * l.shape[1] <= 1 << 24 else None
    if slots is not None:
        counts = slots.sum(dim=(0, 1))
    else:
        counts = torch.zeros(l.shape[1] + 1, device=l.device, dtype=torch.int64).index_add_(0, (idx.reshape(-1) + 1), torch.ones_like(idx.reshape(-1)))[1:]
    n = ok.sum().float()
    per = torch.where(n > 0, l.shape[1] / (k * n * n), torch.zeros_like(n))
    balance = per * (counts.float() * p.sum(dim=0)).sum()
    return idx, gates, counts, balance, p, per


def _route_grad_plain(s):
    idx, gates, counts, balance, p, per = _route_plain(s)
    c = s["coef"] * per * counts.float()
    dl = p * (c[None, :] - (p * c[None, :]).sum(dim=1, keepdim=True))
    dg = gates * (s["dgates"] - (gates * s["dgates"]).sum(dim=1, keepdim=True))
    dl.scatter_add_(1, idx.clamp(min=0), torch.where(idx >= 0, dg, torch.zeros_like(dg)))
    return idx.int(), gates, counts.int(), balance, dl.to(s["logits"].dtype)


def _embed_grad_plain(s):
    dw = torch.zeros(s["vocab"], s["hidden"], device=s["dy"].device)
    dw.index_add_(0, s["ids"], s["dy"].float())
    return (dw * s["scale"]).to(s["dy"].dtype)


def run(state):
    s, kind = state, state["kind"]
    if own:
        from cann_hccl_b200.parallel import moe, vocab
        if kind == "embed":
            return vocab.embedding(s["ids"], s["w"], scale=s["scale"])
        if kind == "embed_grad":
            return vocab.embedding_grad(s["ids"], s["dy"], s["vocab"], scale=s["scale"])
        if kind == "loss":
            return vocab.linear_cross_entropy(s["x"], s["w"], s["y"], reduction="none")
        if kind == "loss_grad":
            return vocab.linear_cross_entropy_grad(s["x"], s["w"], s["y"], weights=s["weights"])
        g = moe.gate(s["logits"], s["topk"], mask=s["mask"])
        if kind == "route":
            return g.idx, g.gates, g.counts, g.balance
        return g.idx, g.gates, g.counts, g.balance, moe.gate_grad(s["logits"], g, s["dgates"], balance=s["coef"])
    if kind == "embed":
        return (s["w"][s["ids"]].float() * s["scale"]).to(s["w"].dtype)
    if kind == "embed_grad":
        return _embed_grad_plain(s)
    if kind == "loss":
        return _loss_plain(s, False)
    if kind == "loss_grad":
        return _loss_plain(s, True)
    if kind == "route":
        idx, gates, counts, balance, _, _ = _route_plain(s)
        return idx.int(), gates, counts.int(), balance
    return _route_grad_plain(s)


def work(case):
    kind, T = case["kind"], case["tokens"]
    if kind in ("embed", "embed_grad"):
        V, H, size = case["vocab"], case["hidden"], SIZE[case["dtype"]]
        # lookup: the distinct rows of a Zipf text are read, every token's row is written; gradient: every token's row read, the table written
        if kind == "embed":
            return {"bytes": T * 8 + (T + _distinct(T, V)) * H * size, "flops": T * H}
        return {"bytes": T * 8 + T * H * size + V * H * size, "flops": 2 * T * H}
    if kind in ("loss", "loss_grad"):
        V, H = case["vocab"], case["hidden"]
        if kind == "loss":
            return {"bytes": 2 * H * (T + V) + 12 * T, "flops": 2 * T * V * H}
        return {"bytes": 4 * H * (T + V) + 12 * T, "flops": 6 * T * V * H}
    E, k, size = case["experts"], case["topk"], SIZE[case["dtype"]]
    if kind == "route":
        return {"bytes": T * E * size + T * k * 8 + 4 * E, "flops": 5 * T * E}
    return {"bytes": 2 * T * E * size + T * k * 12 + 4 * E, "flops": 10 * T * E}


def _distinct(T, V):
    """Expected number of distinct ids of _words(T, V): rank r has the share log(1 + 1/r) / log V."""
    total, r = 0.0, 1
    while r < V:
        step = max(1, r // 64)
        p = math.log1p(1 / r) / math.log(V)
        total += min(step, V - r) * -math.expm1(T * math.log1p(-min(p, 1 - 1e-12)))
        r += step
    return int(total)


# ---------------------------------------------------------------------------------------------------------- 64 bits
def _exact_embed(s):
    if s["kind"] == "embed":
        return torch.index_select(s["w"], 0, s["ids"]).double() * s["scale"]
    dw = torch.zeros(s["vocab"], s["hidden"], device="cuda", dtype=torch.float64)
    order = torch.argsort(s["ids"], stable=True)
    for part in order.split(8192):
        dw.index_add_(0, s["ids"][part], s["dy"][part].double(), alpha=s["scale"])
    return dw


def _exact_loss(s, grad):
    x, w, y = s["x"].double(), s["w"].double(), s["y"]
    T, V = len(x), len(w)
    has = (y != IGNORE) & (y >= 0) & (y < V)
    losses = torch.zeros(T, device="cuda", dtype=torch.float64)
    if grad:
        share = has.double() * (1.0 if s["weights"] is None else s["weights"].double())
        share = share / share.sum() if float(share.sum()) else share
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    rows = max(1, (1 << 28) // V)
    for a in range(0, T, rows):
        b = min(T, a + rows)
        logp = torch.log_softmax(torch.mm(x[a:b], w.mT), dim=-1)
        hit = torch.zeros_like(logp)
        hit[has[a:b].nonzero()[:, 0], y[a:b][has[a:b]]] = 1.0
        losses[a:b] = -(logp * hit).sum(-1)
        if grad:
            d = (logp.exp_() - hit) * share[a:b, None]
            dx[a:b] = torch.mm(d, w)
            dw.addmm_(d.mT, x[a:b])
    return ((losses * share).sum(), dx, dw) if grad else losses


def _exact_route(s, grad):
    l, k = s["logits"].double(), s["topk"]
    T, E = l.shape
    keep = torch.ones(T, device="cuda", dtype=torch.bool) if s["mask"] is None else s["mask"].clone()
    keep &= ~torch.isneginf(l).all(-1)
    p = torch.where(keep[:, None], torch.softmax(l, -1), 0.0)
    # k rounds of the first largest logit that is left
    left, picks = l.clone(), []
    for _ in range(k):
        best = left.max(-1, keepdim=True).values
        first = (left == best).to(torch.uint8).argmax(-1, keepdim=True)
        picks.append(torch.where(keep[:, None] & ~torch.isneginf(best), first, -1))
        left.scatter_(1, first, -math.inf)
    idx = torch.cat(picks, 1)
    on = (idx >= 0).double()
    sel = torch.where(idx >= 0, l.gather(1, idx.clamp(min=0)), -math.inf)
    gates = torch.nan_to_num(torch.softmax(sel, -1), nan=0.0) * on
    counts = torch.bincount(idx[idx >= 0], minlength=E)
    n = int(keep.sum())
    f = counts.double() * (E / (k * n * n) if n else 0.0)
    balance = torch.dot(f, p.sum(0))
    if not grad:
        return idx.int(), gates, counts.int(), balance
    f = f * s["coef"]
    dl = p * f - p * (p @ f)[:, None]
    dg = s["dgates"].double()
    part = gates * dg - gates * (gates * dg).sum(-1, keepdim=True)
    for j in range(k):
        dl.scatter_add_(1, idx[:, j:j + 1].clamp(min=0), part[:, j:j + 1] * on[:, j:j + 1])
    return idx.int(), gates, counts.int(), balance, dl


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("embed", "embed_grad"):
        return _exact_embed(s)
    if case["kind"] in ("loss", "loss_grad"):
        return _exact_loss(s, case["kind"] == "loss_grad")
    return _exact_route(s, case["kind"] == "route_grad")
