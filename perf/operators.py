"""Measured cases of three operator families, each beside its plain form.

* ``vocab_score`` / ``vocab_train``: log-probabilities of given tokens straight from the hidden states and the output
  projection, without logits in memory (``logprobs_from_hidden``), and their gradients.
* ``prefix_decode``: one decode step of attention over a paged cache for sequences that share long prefixes
  (``ops.shared_prefix_attention``), the batch that sampling several answers per prompt makes.
* ``router`` / ``router_train``: expert routing from softmax or sigmoid scores with a selection bias, expert groups,
  renormalised and scaled weights (``grouped_topk_router``), and the gradient of the logits.

``own`` says which side ``run`` takes: the plain form in elementary torch operations, or the framework's calls.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- cases


def _vocab(name, op, tokens, hidden, vocab, temperature=1.0, ignored=0):
    return {"name": name, "op": op, "tokens": tokens, "hidden": hidden, "vocab": vocab, "temperature": temperature, "ignored": ignored}


def _prefix(name, seqs, groups, prefix, tail, heads, kv_heads, dim, page, dtype="bf16"):
    return {"name": name, "op": "prefix_decode", "seqs": seqs, "groups": groups, "prefix": prefix, "tail": tail, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _router(name, op, tokens, experts, top_k, score, groups, topk_groups, group_top, bias, logits, weights, scale=1.0):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "groups": groups,
            "topk_groups": topk_groups, "group_top": group_top, "bias": bias, "logits": logits, "weights": weights, "scale": scale}


def listed():
    return [
        # the log-probabilities of a decode step's tokens, a handful of sequences: the weight matrix is the work
        _vocab("score a few tokens", "vocab_score", 7, 2048, 151936),
        # one short packed batch scored under a sampling temperature, odd vocabulary, prompt tokens without a label
        _vocab("score a ragged batch", "vocab_score", 1000, 1024, 32003, temperature=0.7, ignored=37),
        # the reference-policy pass over a packed batch of answers
        _vocab("score a packed batch", "vocab_score", 16384, 2048, 151936),
        # a small training step: log-probabilities, gradients of the hidden states and of the projection
        _vocab("train on a short batch", "vocab_train", 300, 1024, 32003, ignored=11),
        # the policy update of one micro-batch
        _vocab("train on a micro-batch", "vocab_train", 4096, 2048, 151936),
        # eight answers to one prompt: the smallest group worth sharing
        _prefix("decode one group of 8", 8, 1, 4096, 512, 32, 4, 128, 16),
        # a full decode batch: 16 answers to each of 16 prompts, answers of mixed length
        _prefix("decode 16 groups of 16", 256, 16, 8192, 1024, 32, 4, 128, 16),
        # one long document, many questions
        _prefix("decode 64 on a long prefix", 64, 1, 32768, 700, 32, 8, 128, 16),
        # groups of uneven size, half precision, one query head per kv head
        _prefix("decode uneven groups fp16", 45, 7, 2000, 300, 16, 16, 64, 32, "fp16"),
        # routing of a decode step with balanced, grouped experts
        _router("route a decode step", "router", 64, 256, 8, "sigmoid", 8, 4, 2, True, "fp32", "bf16", 2.5),
        # the same router over a training micro-batch, with its gradient
        _router("train the grouped router", "router_train", 16384, 256, 8, "sigmoid", 8, 4, 2, True, "fp32", "fp32", 2.5),
        # softmax scores, groups by their best expert, logits in 16 bits
        _router("train the softmax router", "router_train", 4099, 160, 6, "softmax", 8, 3, 1, False, "bf16", "bf16", 16.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["vocab_score", "vocab_train", "prefix_decode", "router", "router_train"])
    if family.startswith("vocab"):
        while True:
            tokens, hidden, vocab = _log(rng, 1, 16384), 8 * _log(rng, 16, 512), _log(rng, 500, 160000)
            if rng.random() < 0.5:
                hidden = max(64, hidden // 64 * 64)
            if tokens * hidden * vocab * (4 if family == "vocab_train" else 1) <= 16384 * 2048 * 151936:
                break
        c = _vocab("", family, tokens, hidden, vocab, rng.choice([1.0, 0.7, 1.3]), rng.randrange(0, 1 + tokens // 8))
    elif family == "prefix_decode":
        while True:
            groups = _log(rng, 1, 24)
            seqs = groups * _log(rng, 1, 64) + rng.randrange(0, groups)
            kv_heads = rng.choice([1, 2, 4, 8])
            heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
            dim, page = rng.choice([64, 80, 96, 128, 128, 128]), rng.choice([16, 16, 32, 64, 24])
            prefix, tail = _log(rng, 30, 30000), _log(rng, 1, 3000)
            if seqs <= 320 and seqs * (prefix + tail) * kv_heads * dim <= 256 * 9216 * 4 * 128 and seqs * (prefix + tail) * heads * dim <= 256 * 9216 * 32 * 128:
                break
        c = _prefix("", seqs, groups, prefix, tail, heads, kv_heads, dim, page, rng.choice(["bf16", "bf16", "fp16"]))
    else:
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * rng.randrange(max(2, 8 // groups), 1 + 512 // groups)
        topk_groups = rng.randrange(1, groups + 1)
        # one renormalised weight is constant: it has no gradient
        top_k = rng.randrange(2 if family == "router_train" else 1, 1 + min(16, topk_groups * (experts // groups)))
        c = _router("", family, _log(rng, 1, 16384), experts, top_k, rng.choice(["softmax", "sigmoid"]), groups, topk_groups,
                    rng.choice([1, 2]), rng.random() < 0.6, rng.choice(["fp32", "bf16"]), rng.choice(["fp32", "bf16"]), rng.choice([1.0, 2.5]))
    del c["name"]
    return c


# ----------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"vocab": _prepare_vocab, "prefi": _prepare_prefix, "route": _prepare_router}[case["op"][:5]](case, g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_vocab(c, g):
    T, H, V = c["tokens"], c["hidden"], c["vocab"]
    hidden = _randn(g, T, H).to(torch.bfloat16)  # rows as the last norm leaves them
    weight = (1.8 / math.sqrt(H) * _randn(g, V, H)).to(torch.bfloat16)  # logits with a spread of about two
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    labels[torch.randperm(T, generator=g, device="cuda")[: c["ignored"]]] = -100  # padding: no label
    s = {"case": c, "hidden": hidden, "weight": weight, "labels": labels, "temperature": c["temperature"]}
    if c["op"] == "vocab_train":
        s["d_out"] = _randn(g, T) / T  # advantages over a mean
        s["hidden"].requires_grad_()
        s["weight"].requires_grad_()
    return s


def _prepare_prefix(c, g):
    B, G, page, Hkv, D, dt = c["seqs"], c["groups"], c["page"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    cpu = torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=g, device="cuda")))
    # group sizes: even where they divide, otherwise uneven with at least one sequence each
    if B % G == 0:
        sizes = torch.full((G,), B // G, dtype=torch.int64)
    else:
        sizes = 1 + torch.bincount(torch.randint(0, G, (B - G,), generator=cpu), minlength=G)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    group_of = torch.repeat_interleave(torch.arange(G), sizes)
    # prefix lengths about the case's (within a fifth of it, the longest exactly it); whole pages are shared
    lens = (c["prefix"] * (0.8 + 0.2 * torch.rand(G, generator=cpu))).long().clamp(min=1)
    lens[0] = c["prefix"]
    shared_pages = lens // page
    kv_len = lens[group_of] + torch.randint(1, c["tail"] + 1, (B,), generator=cpu)
    pages = (kv_len + page - 1) // page
    own_pages = pages - shared_pages[group_of]
    total = int(shared_pages.sum() + own_pages.sum())
    ids = torch.randperm(total, generator=cpu).int()
    first_shared = shared_pages.cumsum(0) - shared_pages
    first_own = int(shared_pages.sum()) + own_pages.cumsum(0) - own_pages
    slot = torch.arange(int(pages.max()))[None, :].expand(B, -1)
    shared_here = shared_pages[group_of][:, None]
    src = torch.where(slot < shared_here, first_shared[group_of][:, None] + slot, first_own[:, None] + slot - shared_here)
    table = torch.where(slot < pages[:, None], ids[src.clamp(max=total - 1)], torch.zeros((), dtype=torch.int32))
    cache = lambda: _randn(g, total, page, Hkv, D).to(dt)  # noqa: E731
    return {"case": c, "k": cache(), "v": cache(), "q": _randn(g, B, c["heads"], D).to(dt), "scale": D**-0.5,
            "cu": torch.arange(B + 1, dtype=torch.int32, device="cuda"), "kv_len": kv_len.int().cuda(), "table": table.int().cuda(),
            "groups": offsets.int().cuda(), "prefix": (shared_pages * page).int().cuda(), "max_prefix": int(shared_pages.max()) * page}


def _prepare_router(c, g):
    T, E = c["tokens"], c["experts"]
    logits = _randn(g, T, E).to(DTYPES[c["logits"]])
    s = {"case": c, "logits": logits, "bias": 0.1 * _randn(g, E) if c["bias"] else None}
    if c["op"] == "router_train":
        s["d_weights"] = _randn(g, T, c["top_k"]).to(DTYPES[c["weights"]])
        s["logits"].requires_grad_()
    return s


# ----------------------------------------------------------------------------- one pass


def run(state):
    return {"vocab": _run_vocab, "prefi": _run_prefix, "route": _run_router}[state["case"]["op"][:5]](state)


def _run_vocab(s):
    train = s["case"]["op"] == "vocab_train"
    if own:
        from vexact_amd.batch_invariant_ops.standalone_logprobs import logprobs_from_hidden

        with torch.set_grad_enabled(train):
            lp = logprobs_from_hidden(s["hidden"], s["weight"], s["labels"], temperature=s["temperature"])
            return [lp, *torch.autograd.grad(lp, (s["hidden"], s["weight"]), s["d_out"])] if train else [lp]
    with torch.no_grad():
        h, w = s["hidden"].float(), s["weight"].float()
        x = (h @ w.t()) / s["temperature"]
        top = x.amax(-1, keepdim=True)
        lse = top[:, 0] + torch.log(torch.exp(x - top).sum(-1))
        labelled = s["labels"] >= 0
        at = s["labels"].clamp(min=0)[:, None]
        lp = torch.where(labelled, x.gather(1, at)[:, 0] - lse, math.nan)  # no label: no log-probability
        if not train:
            return [lp]
        d = torch.where(labelled, s["d_out"], 0.0) / s["temperature"]
        dx = torch.exp(x - lse[:, None]) * -d[:, None]
        dx.scatter_add_(1, at, d[:, None])
        return [lp, (dx @ w).to(torch.bfloat16), (dx.t() @ h).to(torch.bfloat16)]


def _run_prefix(s):
    if own:
        from vexact_amd import ops

        return [ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["cu"], s["kv_len"], s["table"], s["groups"], s["prefix"], s["scale"],
                                            max_prefix_len=s["max_prefix"])]
    q, table = s["q"].float(), s["table"].long()
    B, Hq, D = q.shape
    page, Hkv = s["k"].shape[1], s["k"].shape[2]
    # the sequences' keys and values, [sequences, kv heads, keys, dim]
    rows = lambda cache: cache[table].view(B, -1, Hkv, D).transpose(1, 2).float()  # noqa: E731
    x = (q.view(B, Hkv, Hq // Hkv, D) @ rows(s["k"]).transpose(2, 3).contiguous()) * s["scale"]
    x = x.masked_fill(torch.arange(table.shape[1] * page, device=q.device) >= s["kv_len"].view(B, 1, 1, 1), -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    out = (p @ rows(s["v"])) / p.sum(-1, keepdim=True)
    return [out.view(B, Hq, D).to(s["q"].dtype)]


def _run_router(s):
    c = s["case"]
    train = c["op"] == "router_train"
    if own:
        from vexact_amd.batch_invariant_ops.router import grouped_topk_router

        with torch.set_grad_enabled(train):
            w, idx = grouped_topk_router(s["logits"], c["top_k"], score=c["score"], bias=s["bias"], n_groups=c["groups"],
                                         topk_groups=c["topk_groups"], group_top=c["group_top"], scale=c["scale"], out_dtype=DTYPES[c["weights"]])
            return [w, idx, *torch.autograd.grad(w, s["logits"], s["d_weights"])] if train else [w, idx]
    with torch.no_grad():
        # in 64 bits: which of two close scores is the larger must not hang on a rounding
        x = s["logits"].double()
        if c["score"] == "softmax":
            e = torch.exp(x - x.amax(-1, keepdim=True))
            score = e / e.sum(-1, keepdim=True)
        else:
            score = 1 / (1 + torch.exp(-x))
        choice = score if s["bias"] is None else score + s["bias"].double()
        T, E, n = *x.shape, c["groups"]
        if n > 1:
            best = choice.view(T, n, E // n).sort(dim=-1, descending=True).values[..., : c["group_top"]].sum(-1)
            kept = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["topk_groups"]]
            group_ok = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
            choice = choice.masked_fill(~group_ok.repeat_interleave(E // n, 1), -math.inf)
        idx = choice.sort(dim=-1, descending=True, stable=True).indices[:, : c["top_k"]]
        sel = score.gather(1, idx)
        norm = sel / sel.sum(-1, keepdim=True)
        w = (norm * c["scale"]).to(DTYPES[c["weights"]])
        if not train:
            return [w, idx]
        d = s["d_weights"].double() * c["scale"]
        d_sel = (d - (d * norm).sum(-1, keepdim=True)) / sel.sum(-1, keepdim=True)
        d_score = torch.zeros_like(score).scatter_(1, idx, d_sel)
        if c["score"] == "softmax":
            dx = score * (d_score - (d_score * score).sum(-1, keepdim=True))
        else:
            dx = d_score * score * (1 - score)
        return [w, idx, dx.to(s["logits"].dtype)]


# ----------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    if c["op"].startswith("vocab"):
        T, H, V = c["tokens"], c["hidden"], c["vocab"]
        train = c["op"] == "vocab_train"
        # a training step computes the logits at least once and two products of that size beside them
        return {"bytes": (2 * (T * H + V * H)) * (2 if train else 1) + T * (16 if train else 12), "flops": 2 * T * H * V * (3 if train else 1)}
    if c["op"] == "prefix_decode":
        # the mean case of prepare(): prefixes at 0.9 of the longest, tails at half
        kv_row = 2 * c["kv_heads"] * c["dim"] * 2
        keys = c["seqs"] * (0.9 * c["prefix"] + 0.5 * c["tail"])
        return {"bytes": int(kv_row * (c["groups"] * 0.9 * c["prefix"] + c["seqs"] * 0.5 * c["tail"]) + 4 * c["seqs"] * c["heads"] * c["dim"]),
                "flops": int(4 * c["heads"] * c["dim"] * keys)}
    T, E, k = c["tokens"], c["experts"], c["top_k"]
    lb, wb = (4 if c["logits"] == "fp32" else 2), (4 if c["weights"] == "fp32" else 2)
    fwd, bwd = T * (E * lb + k * (wb + 8)) + 4 * E * c["bias"], T * (E * lb + k * wb)
    train = c["op"] == "router_train"
    return {"bytes": fwd + (bwd if train else 0), "flops": 10 * T * E * (2 if train else 1)}


# ----------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"vocab": _exact_vocab, "prefi": _exact_prefix, "route": _exact_router}[case["op"][:5]](s)


def _exact_vocab(s):
    train, w = s["case"]["op"] == "vocab_train", s["weight"].double()
    lps, dhs, dw = [], [], torch.zeros_like(w) if train else None
    for r in range(0, s["hidden"].shape[0], 2048):  # so many rows at a time: 64-bit logits are large
        h, y = s["hidden"][r : r + 2048].double(), s["labels"][r : r + 2048]
        logp = torch.log_softmax(torch.mm(h, w.t()) / s["temperature"], dim=1)
        row = torch.arange(len(y), device=y.device)
        good = (y >= 0) & (y < w.shape[0])
        lp = torch.full((len(y),), math.nan, dtype=torch.float64, device=y.device)
        lp[good] = logp[row[good], y[good]]
        lps.append(lp)
        if train:
            weight_of = (s["d_out"][r : r + 2048].double() / s["temperature"]) * good
            grad = logp.exp_().mul_(-weight_of[:, None])  # d logits = d (onehot - softmax) / temperature
            grad[row[good], y[good]] += weight_of[good]
            dhs.append(torch.mm(grad, w))
            dw.addmm_(grad.t(), h)
    return [torch.cat(lps), torch.cat(dhs), dw] if train else [torch.cat(lps)]


def _exact_prefix(s):
    out = []
    group = s["q"].shape[1] // s["k"].shape[2]
    for i, n in enumerate(s["kv_len"].tolist()):
        at = torch.arange(n, device="cuda")
        page = s["k"].shape[1]
        block, inside = s["table"][i, at // page].long(), at % page
        k, v = s["k"][block, inside].double(), s["v"][block, inside].double()  # [keys, kv heads, dim]
        k, v = (t.repeat_interleave(group, dim=1).transpose(0, 1).contiguous() for t in (k, v))
        prob = torch.softmax(torch.bmm(k, s["q"][i].double()[:, :, None])[:, :, 0] * s["scale"], dim=1)
        out.append(torch.bmm(prob[:, None, :], v)[:, 0])
    return [torch.stack(out)]


def _exact_router(s):
    c, x = s["case"], s["logits"].detach().double()
    score = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
    ranked = score.clone()
    if s["bias"] is not None:
        ranked += s["bias"].double()
    n, size = c["groups"], x.shape[1] // c["groups"]
    tops = torch.stack([ranked[:, i * size : (i + 1) * size].topk(min(c["group_top"], size), dim=1).values.sum(1) for i in range(n)], 1)
    order = torch.argsort(tops, dim=1, descending=True, stable=True)
    place = torch.argsort(order, dim=1)  # a group's place in that order
    if n > 1:
        ranked[(place >= c["topk_groups"]).repeat_interleave(size, dim=1)] = -math.inf
    idx = torch.argsort(ranked, dim=1, descending=True, stable=True)[:, : c["top_k"]]
    row = torch.arange(len(x), device=x.device)[:, None]
    chosen = score[row, idx]
    total = chosen.sum(1, keepdim=True)
    out = [c["scale"] * chosen / total, idx]
    if c["op"] == "router_train":
        d = c["scale"] * s["d_weights"].double()
        # through w_i = s_i / sum s: d s_i = d w_i / sum - sum_j d w_j s_j / sum^2
        d_chosen = d / total - (d * chosen).sum(1, keepdim=True) / total**2
        full = torch.zeros_like(score)
        full[row, idx] = d_chosen
        slope = score * (full - (full * score).sum(1, keepdim=True)) if c["score"] == "softmax" else full * score * (1 - score)
        out.append(slope)
    return out
