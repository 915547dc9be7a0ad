"""The selection operators of a language model, as cases to measure: sampling a token from a row
of logits, routing tokens to experts, ordering the assignments by expert, and moving rows to the
experts and back.

Where ``own`` is false, ``run`` computes each operator in its plain form (elementary torch
operations in 32 bits); where it is true, it calls ``batch_topk_b200.torch_api``.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NEG = float("-inf")


# ---- the cases -----------------------------------------------------------------------------

def listed():
    return [
        # one user's chat: every microsecond of the call is felt between two tokens
        dict(name="sample-one-row", op="sample", rows=1, vocab=32000, dtype="fp32",
             filters="topk_topp"),
        # a served batch: every request brings its own settings, some a grammar's mask
        dict(name="sample-served-batch", op="sample", rows=64, vocab=128256, dtype="bf16",
             filters="mixed"),
        # rollouts for reinforcement learning: the whole distribution, nothing cut
        dict(name="sample-rollout", op="sample", rows=200, vocab=151936, dtype="bf16",
             filters="none"),
        # offline generation at a large batch: nucleus sampling over the whole vocabulary
        dict(name="sample-offline-nucleus", op="sample", rows=1024, vocab=151936, dtype="fp16",
             filters="topp"),
        # a decode step of a model with many small experts: sigmoid scores, balance bias, groups
        dict(name="route-decode", op="route", tokens=32, experts=256, k=8, dtype="fp32",
             score="sigmoid", bias=True, groups=8, topk_groups=4, renormalize=True,
             backward=False),
        # a training step's router over 32 sequences of 4096 tokens, forward and backward
        dict(name="route-train", op="route", tokens=131072, experts=256, k=8, dtype="fp32",
             score="softmax", bias=False, groups=1, topk_groups=1, renormalize=False,
             backward=True),
        # the same decode step's assignments, sorted by expert
        dict(name="order-decode", op="order", tokens=32, experts=256, k=8),
        # a long prompt batch of ragged length, some of it padding
        dict(name="order-prefill", op="order", tokens=65521, experts=256, k=8),
        # rows of a small decode batch to their experts
        dict(name="dispatch-decode", op="dispatch", tokens=32, experts=256, k=8, width=4096,
             dtype="bf16", backward=False),
        # a training step: rows out, gradients back
        dict(name="dispatch-train", op="dispatch", tokens=8191, experts=64, k=6, width=2048,
             dtype="bf16", backward=True),
        # experts' rows back to a small decode batch
        dict(name="combine-decode", op="combine", tokens=32, experts=256, k=8, width=4096,
             dtype="bf16", backward=False),
        # a training step: weighted sums, gradients of rows and weights
        dict(name="combine-train", op="combine", tokens=8191, experts=64, k=6, width=2048,
             dtype="bf16", backward=True),
    ]


def _spread(rng, lo, hi):
    """An integer from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "route", "route", "order", "dispatch", "combine"])
    if op == "sample":
        vocab = _spread(rng, 1000, 262144)
        return dict(op=op, rows=_spread(rng, 1, min(1024, 1024 * 151936 // vocab)), vocab=vocab,
                    dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    filters=rng.choice(["none", "topk", "topp", "minp", "topk_topp", "mixed"]))
    k = rng.randint(1, 8)
    if op == "order":
        return dict(op=op, tokens=_spread(rng, 1, 65521), experts=_spread(rng, 8, 512), k=k)
    if op == "route":
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 4, 8])
        experts = max(8, _spread(rng, 8, 512) // groups * groups)
        topk_groups = 1 if groups == 1 else rng.randint(1, groups)
        return dict(op=op, tokens=_spread(rng, 1, 65536), experts=experts,
                    k=min(k, experts // groups * topk_groups),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]), score=score,
                    bias=score == "sigmoid" and rng.random() < 0.5, groups=groups,
                    topk_groups=topk_groups, renormalize=rng.random() < 0.5,
                    backward=rng.random() < 0.5)
    width = _spread(rng, 64, 8192)
    return dict(op=op, tokens=_spread(rng, 1, max(1, 8191 * 6 * 2048 // (k * width))),
                experts=_spread(rng, 8, 256), k=k, width=width,
                dtype=rng.choice(["fp16", "bf16", "fp32"]), backward=rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------

def _logits(case, g, dev):
    """Logits like a language model's: a broad bulk, a head of likely tokens, and a sharpness
    that differs from row to row."""
    n, v = case["rows"], case["vocab"]
    x = torch.randn((n, v), generator=g, device=dev).mul_(2.0)
    head = torch.randint(0, v, (n, 40), generator=g, device=dev)
    lift = 13 + 3 * torch.randn((n, 40), generator=g, device=dev)
    x.scatter_add_(1, head, lift)
    x.mul_(0.7 + 0.6 * torch.rand((n, 1), generator=g, device=dev))
    if case["filters"] == "mixed":  # a grammar leaves one token in ten of every fourth row
        cut = torch.rand((n, v), generator=g, device=dev) < 0.9
        cut &= (torch.arange(n, device=dev) % 4 == 1)[:, None]
        x.masked_fill_(cut, NEG)
    return x.to(DTYPES[case["dtype"]])


def _settings(case, g, dev):
    """temperature, top_k, top_p, min_p: numbers for the batch, or one of each for every row."""
    kind = case["filters"]
    if kind != "mixed":
        return dict(temperature=1.0 if kind == "none" else 0.8,
                    top_k=50 if "topk" in kind else 0,
                    top_p=0.95 if "topp" in kind else 1.0,
                    min_p=0.05 if kind == "minp" else 0.0)
    n = case["rows"]

    def of(values, dtype):
        at = torch.randint(0, len(values), (n,), generator=g, device=dev)
        return torch.tensor(values, device=dev, dtype=dtype)[at]

    return dict(temperature=of([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32),
                top_k=of([0, 0, 1, 20, 50, 200], torch.int32),
                top_p=of([1.0, 0.8, 0.9, 0.95], torch.float32),
                min_p=of([0.0, 0.0, 0.02, 0.1], torch.float32))


def _experts(case, g, dev):
    """k different experts a token, a few experts popular; every 64th token is padding (-1)."""
    t, e = case["tokens"], case["experts"]
    pull = torch.randn((1, e), generator=g, device=dev)
    score = pull - torch.empty((t, e), device=dev).exponential_(generator=g).log_()
    ex = score.topk(min(case["k"], e), dim=1).indices.to(torch.int32)
    ex[63::64] = -1
    return ex


def _plan(experts, num):
    """offsets, order and position of the assignments, sorted by expert."""
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, num, flat)
    ranked, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ranked, torch.arange(num + 1, device=flat.device))
    rank = torch.arange(flat.numel(), device=flat.device)
    position = torch.empty_like(order)
    position[order] = rank
    position = torch.where(flat < 0, -1, position)
    order = torch.where(rank < offsets[num], order, -1)
    return (offsets.to(torch.int32), order.to(torch.int32),
            position.to(torch.int32).view(experts.shape))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    s = dict(case=case, op=op)
    if op == "sample":
        s["logits"] = _logits(case, g, dev)
        noise = torch.empty((case["rows"], case["vocab"]), device=dev)
        s["noise"] = noise.exponential_(generator=g).clamp_(min=1e-20)
        s["settings"] = _settings(case, g, dev)
    elif op == "route":
        t, e = case["tokens"], case["experts"]
        x = torch.randn((t, e), generator=g, device=dev) * 1.5
        s["logits"] = x.to(DTYPES[case["dtype"]]).requires_grad_(case["backward"])
        s["bias"] = torch.randn((e,), generator=g, device=dev) * 0.05 if case["bias"] else None
        s["grad"] = torch.randn((t, case["k"]), generator=g, device=dev)
    else:
        s["experts"] = _experts(case, g, dev)
        if op != "order":
            t, k, w = case["tokens"], s["experts"].shape[1], case["width"]
            dt = DTYPES[case["dtype"]]
            s["plan"] = _plan(s["experts"], case["experts"])
            rows = torch.randn((t * k, w), generator=g, device=dev).to(dt)
            toks = torch.randn((t, w), generator=g, device=dev).to(dt)
            if op == "dispatch":
                s["x"], s["grad"] = toks.requires_grad_(case["backward"]), rows
            else:
                s["rows"], s["grad"] = rows.requires_grad_(case["backward"]), toks
                wt = torch.rand((t, k), generator=g, device=dev)
                s["weights"] = (wt / wt.sum(1, keepdim=True)).requires_grad_(case["backward"])
    return s


# ---- one pass ------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from batch_topk_b200 import torch_api as api

    c, op = s["case"], s["op"]
    if op == "sample":
        tokens, logprobs = api.sample(s["logits"], s["noise"], **s["settings"])
        return dict(tokens=tokens, logprobs=logprobs)
    if op == "route":
        weights, experts = api.route(s["logits"], c["k"], score=c["score"], bias=s["bias"],
                                     groups=c["groups"], topk_groups=c["topk_groups"],
                                     renormalize=c["renormalize"], scale=2.5)
        out = dict(weights=weights, experts=experts)
        if c["backward"]:
            out["d_logits"], = torch.autograd.grad(weights, s["logits"], s["grad"])
        return out
    if op == "order":
        plan = api.expert_order(s["experts"], c["experts"])
        return dict(offsets=plan.offsets, order=plan.order, position=plan.position)
    plan = api.ExpertOrder(*s["plan"])
    if op == "dispatch":
        rows = api.dispatch(s["x"], plan)
        out = dict(rows=rows)
        if c["backward"]:
            out["d_x"], = torch.autograd.grad(rows, s["x"], s["grad"])
        return out
    y = api.combine(s["rows"], plan, s["weights"])
    out = dict(y=y)
    if c["backward"]:
        out["d_rows"], out["d_weights"] = torch.autograd.grad(y, (s["rows"], s["weights"]),
                                                              s["grad"])
    return out


@torch.no_grad()
def _run_plain(s):
    return dict(sample=_sample, route=_route, order=_order, dispatch=_dispatch,
                combine=_combine)[s["op"]](s)


def _sample(s):
    x = s["logits"].float() + 0.0
    x = torch.where(torch.isnan(x), NEG, x)
    n, v = x.shape

    def row(value, dtype):
        return torch.as_tensor(value, dtype=dtype, device=x.device).expand(n)[:, None]

    t = row(s["settings"]["temperature"], torch.float32)
    top_k = row(s["settings"]["top_k"], torch.int64)
    top_p = row(s["settings"]["top_p"], torch.float32)
    min_p = row(s["settings"]["min_p"], torch.float32)
    greedy = ~(t > 0)
    top = x.amax(1, keepdim=True)
    d = torch.where(x == top, 0.0, (x - top) * torch.where(greedy, 1.0, 1.0 / t))
    w = torch.where(top == NEG, 0.0, torch.exp(d))
    # filters, in rank order: value descending, then the lower index
    rank = torch.sort(x, dim=1, descending=True, stable=True).indices
    pos = torch.arange(v, device=x.device)
    in_k = (pos < top_k) | (top_k <= 0)
    ws = torch.where(in_k, w.gather(1, rank), 0.0)
    mass = ws.cumsum(1)
    before = torch.nn.functional.pad(mass[:, :-1], (1, 0))
    in_p = (before < top_p * mass[:, -1:]) | ~(top_p < 1) | (pos == 0)
    kept = torch.zeros_like(in_k).scatter_(1, rank, in_k & in_p) & ~(w < min_p.clamp(max=1.0))
    # the race: the largest weight over noise wins
    score = w / s["noise"]
    score = torch.where(greedy, (x == top).float(), torch.where(score >= 0, score, -1.0))
    score = torch.where(kept & (x > NEG), score, -2.0)
    best = score.amax(1, keepdim=True)
    token = torch.where(score == best, pos, v).amin(1)
    logprob = d.gather(1, token[:, None])[:, 0] - torch.log(w.sum(1))
    none = best[:, 0] == -2.0
    return dict(tokens=torch.where(none, -1, token).to(torch.int32),
                logprobs=torch.where(none, NEG, logprob))


def _route(s):
    c, bias = s["case"], s["bias"]
    x = s["logits"].detach().float() + 0.0
    x = torch.where(torch.isnan(x), NEG, x)
    n, e = x.shape
    if c["score"] == "softmax":
        top = x.amax(1, keepdim=True)
        w = torch.where(top == NEG, 0.0, torch.exp(torch.where(x == top, 0.0, x - top)))
        sc = w / w.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        sc = 1.0 / (1.0 + torch.exp(-x))
    choice = x if bias is None else torch.where(x == NEG, NEG, sc + bias)
    if c["groups"] > 1:
        value = choice if c["score"] == "softmax" else sc if bias is None else choice
        value = torch.where(choice == NEG, NEG, value).view(n, c["groups"], -1)
        two = value.sort(dim=2, descending=True).values[:, :, :2]
        if c["score"] == "softmax":
            of_group = two[:, :, 0]
        else:
            of_group = torch.where(two == NEG, 0.0, two).sum(2)
            of_group = torch.where(two[:, :, 0] == NEG, NEG, of_group)
        order = torch.sort(of_group, dim=1, descending=True, stable=True).indices
        stays = torch.zeros_like(of_group, dtype=torch.bool)
        stays.scatter_(1, order[:, :c["topk_groups"]], True)
        choice = torch.where(stays.repeat_interleave(e // c["groups"], 1), choice, NEG)
    best = torch.sort(choice, dim=1, descending=True, stable=True)
    experts, closed = best.indices[:, :c["k"]], best.values[:, :c["k"]] == NEG
    sel = torch.where(closed, 0.0, sc.gather(1, experts))
    total = sel.sum(1, keepdim=True) + 1e-20 if c["renormalize"] else torch.ones_like(sel[:, :1])
    out = dict(weights=2.5 * sel / total,
               experts=torch.where(closed, -1, experts).to(torch.int32))
    if c["backward"]:
        g = torch.where(closed, 0.0, s["grad"])
        d_sel = 2.5 * g / total
        if c["renormalize"]:
            d_sel = d_sel - (d_sel * sel).sum(1, keepdim=True) / total
        d_sc = torch.zeros_like(sc).scatter_add_(1, experts, torch.where(closed, 0.0, d_sel))
        if c["score"] == "softmax":
            dx = sc * (d_sc - (d_sc * sc).sum(1, keepdim=True))
        else:
            dx = d_sc * sc * (1.0 - sc)
        out["d_logits"] = dx.to(s["logits"].dtype)
    return out


def _order(s):
    offsets, order, position = _plan(s["experts"], s["case"]["experts"])
    return dict(offsets=offsets, order=order, position=position)


def _rows_of(rows, at):
    """rows[at] in 32 bits, nothing where at is -1."""
    got = rows.detach()[at.clamp(min=0).long()].float()
    return torch.where((at < 0)[..., None], 0.0, got)


def _dispatch(s):
    _, order, position = s["plan"]
    src = torch.where(order < 0, -1, order // position.shape[1])
    out = dict(rows=_rows_of(s["x"], src).to(s["x"].dtype))
    if s["case"]["backward"]:
        out["d_x"] = _rows_of(s["grad"], position).sum(1).to(s["x"].dtype)
    return out


def _combine(s):
    _, order, position = s["plan"]
    k, dt = position.shape[1], s["rows"].dtype
    w = s["weights"].detach()
    got = _rows_of(s["rows"], position)
    out = dict(y=(w[..., None] * got).sum(1).to(dt))
    if s["case"]["backward"]:
        at = order.clamp(min=0).long()
        d = w.reshape(-1)[at][:, None] * s["grad"][at // k].float()
        out["d_rows"] = torch.where((order < 0)[:, None], 0.0, d).to(dt)
        out["d_weights"] = (got * s["grad"].float()[:, None, :]).sum(2)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        es = 4 if case["dtype"] == "fp32" else 2
        noise = 4 * n if case["filters"] == "none" else 0  # else the kept tokens' alone: few
        return dict(bytes=n * es + noise + 8 * case["rows"], flops=4 * n)
    t, k = case["tokens"], case["k"]
    if op == "route":
        n, es = t * case["experts"], 4 if case["dtype"] == "fp32" else 2
        back = n * es + 4 * t * k if case["backward"] else 0  # the logits need not be read twice
        return dict(bytes=n * es + 8 * t * k + back, flops=(12 if case["backward"] else 6) * n)
    if op == "order":
        return dict(bytes=12 * t * k + 4 * (case["experts"] + 1), flops=0)
    es = 4 if case["dtype"] == "fp32" else 2
    row = case["width"] * es
    if op == "dispatch":
        one = t * row + t * k * row + 8 * t * k
        return dict(bytes=one * (2 if case["backward"] else 1),
                    flops=t * k * case["width"] if case["backward"] else 0)
    one = t * row + t * k * row + 8 * t * k
    # backward: the rows are read for the weights' gradient and a row's gradient is written
    back = t * row + t * k * row + 8 * t * k if case["backward"] else 0
    return dict(bytes=one + back, flops=(6 if case["backward"] else 2) * t * k * case["width"])


# ---- the definition in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "sample":
            return _exact_sample(case, s)
        if case["op"] == "route":
            return _exact_route(case, s)
        if case["op"] == "order":
            return None  # whole numbers only
        return _exact_rows(case, s)


def _exact_sample(case, s):
    """Row by row: sort, cut, race; the log-probability is that of the uncut distribution."""
    tokens, logprobs = [], []
    values = {a: (b.tolist() if isinstance(b, torch.Tensor) else [b] * case["rows"])
              for a, b in s["settings"].items()}
    for i in range(case["rows"]):
        x, q = s["logits"][i].double(), s["noise"][i].double()
        t, k, p, mp = (values[a][i] for a in ("temperature", "top_k", "top_p", "min_p"))
        t = float(t)
        value, at = torch.sort(x / t if t > 0 else x, descending=True, stable=True)
        lw = torch.log_softmax(value, 0)
        if t > 0:
            n = k if k > 0 else x.numel()
            pr = torch.softmax(value[:n], 0)
            if p < 1:
                pr = torch.where(pr.cumsum(0) - pr < p * pr.sum(), pr, 0.0)
            pr = torch.where(pr >= mp * pr[0], pr, 0.0)
            j = (pr / q[at[:n]]).argmax()
        else:
            j = torch.zeros((), dtype=torch.long, device=x.device)
        tokens.append(at[j])
        logprobs.append(lw[j])
    return dict(tokens=torch.stack(tokens).int(), logprobs=torch.stack(logprobs))


def _exact_route(case, s):
    x = s["logits"].detach().double().requires_grad_(case["backward"])
    with torch.enable_grad():
        sc = x.softmax(1) if case["score"] == "softmax" else x.sigmoid()
        pick = (sc if s["bias"] is None else sc + s["bias"].double()).detach().clone()
        if case["groups"] > 1:
            by = pick.view(case["tokens"], case["groups"], -1)
            few = 1 if case["score"] == "softmax" else min(2, by.shape[2])
            good = by.topk(few, 2).values.sum(2).topk(case["topk_groups"], 1).indices
            shut = torch.ones(by.shape[:2], dtype=torch.bool, device=x.device)
            shut.scatter_(1, good, False)
            pick = by.masked_fill(shut[:, :, None], NEG).view(pick.shape)
        at = torch.sort(pick, dim=1, descending=True, stable=True).indices[:, :case["k"]]
        w = sc.gather(1, at)
        w = 2.5 * (w / w.sum(1, keepdim=True) if case["renormalize"] else w)
        out = dict(weights=w.detach(), experts=at.int())
        if case["backward"]:
            out["d_logits"], = torch.autograd.grad(w, x, s["grad"].double())
    return out


def _exact_rows(case, s):
    """Both ways as sums over the assignments, one of the k at a time."""
    _, _, position = s["plan"]
    t, k = position.shape
    live = (position >= 0).double()
    if case["op"] == "dispatch":
        x = s["x"].detach().double()
        rows = torch.zeros((t * k, case["width"]), dtype=torch.float64, device=x.device)
        dx = torch.zeros_like(x)
        for j in range(k):
            at = position[:, j].long()
            ok = at >= 0
            rows[at[ok]] = x[ok]
            dx[ok] += s["grad"][at[ok]].double()
        return dict(rows=rows, d_x=dx) if case["backward"] else dict(rows=rows)
    rows, w, g = s["rows"].detach(), s["weights"].detach().double(), s["grad"].double()
    y, dw = torch.zeros_like(g), torch.zeros_like(w)
    d_rows = torch.zeros(rows.shape, dtype=torch.float64, device=rows.device)
    for j in range(k):
        at = position[:, j].long().clamp(min=0)
        r = rows[at].double() * live[:, j, None]
        y += w[:, j, None] * r
        dw[:, j] = (r * g).sum(1)
        ok = position[:, j] >= 0
        d_rows[at[ok]] = (w[:, j, None] * g)[ok]
    return dict(y=y, d_rows=d_rows, d_weights=dw) if case["backward"] else dict(y=y)
