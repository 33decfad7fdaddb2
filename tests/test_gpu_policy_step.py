"""One step over sampled answers with the operators it is made of: attention over the prompts' shared prefixes, grouped
routing of the expert block, and the chosen tokens' log-probabilities straight from the last hidden states."""

import pytest
import torch

from vexact_amd import ops
from vexact_amd.batch_invariant_ops.fused_moe import fused_moe_forward
from vexact_amd.batch_invariant_ops.router import grouped_topk_router
from vexact_amd.batch_invariant_ops.standalone_logprobs import logprobs_from_hidden

from .test_gpu_shared_prefix import make
from .util import assert_bitwise

pytestmark = pytest.mark.gpu

Hq, Hkv, D, H, E, I, K, V = 8, 2, 64, 256, 16, 64, 4, 1500


def weights(seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).to(torch.bfloat16)  # noqa: E731
    return dict(q=r(Hq * D, H), o=r(H, Hq * D), norm1=torch.ones(H).to(torch.bfloat16), norm2=torch.ones(H).to(torch.bfloat16), router=r(E, H),
                bias=0.1 * torch.randn(E, generator=g), gate=r(E, I, H), up=r(E, I, H), down=r(E, H, I), head=2 * r(V, H))


def step(w, x, attn, labels):
    """The step on the GPU; returns the log-probabilities and the selected experts."""
    q = ops.matmul(x, w["q"].t()).view(-1, Hq, D)
    a = ops.shared_prefix_attention(**{**attn, "q": q})
    y = ops.matmul(a.view(-1, Hq * D), w["o"].t()) + x
    h = ops.rms_norm(y, w["norm1"])
    route, sel = grouped_topk_router(h @ w["router"].t() if h.requires_grad else ops.matmul(h, w["router"].t()), K, score="sigmoid",
                                     bias=w["bias"], n_groups=4, topk_groups=2, scale=1.5)
    z = y + fused_moe_forward(num_experts=E, routing_weights=route, selected_experts=sel, hidden_states=h, fc1_1_weight=w["gate"],
                              fc1_2_weight=w["up"], fc2_weight=w["down"])
    return logprobs_from_hidden(ops.rms_norm(z, w["norm2"]), w["head"], labels), sel


def reference(w, x, attn, labels, sel):
    w = {n: t.double() for n, t in w.items()}
    x = x.double()
    norm = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    q = (x @ w["q"].t()).view(-1, Hq, D)
    k, v, page = attn["k_cache"].cpu().double(), attn["v_cache"].cpu().double(), attn["k_cache"].shape[1]
    a = torch.zeros_like(q)
    for i, n in enumerate(attn["seqused_k"].tolist()):
        at = torch.arange(n)
        blk = attn["page_table"][i].cpu()[at // page].long()
        for hh in range(Hq):
            kk, vv = k[blk, at % page, hh // (Hq // Hkv)], v[blk, at % page, hh // (Hq // Hkv)]
            a[i, hh] = torch.softmax(kk @ q[i, hh] * attn["softmax_scale"], 0) @ vv
    y = a.view(-1, Hq * D) @ w["o"].t() + x
    h = norm(y)
    s = torch.sigmoid(h @ w["router"].t()).gather(1, sel)
    route = 1.5 * s / s.sum(1, keepdim=True)
    act = torch.nn.functional.silu(torch.einsum("th,tkih->tki", h, w["gate"][sel])) * torch.einsum("th,tkih->tki", h, w["up"][sel])
    z = y + (torch.einsum("tki,tkhi->tkh", act, w["down"][sel]) * route[..., None]).sum(1)
    return torch.log_softmax(norm(z) @ w["head"].t(), 1).gather(1, labels[:, None])[:, 0]


def test_a_step_over_sampled_answers():
    w = weights(1)
    wg = {n: t.cuda() for n, t in w.items()}
    attn = make([4, 3, 1], [600, 300, 90], [7, 1, 270, 40], (Hq, Hkv), (D, D), 16, seed=3)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, H, generator=g).to(torch.bfloat16)
    labels = torch.randint(0, V, (8,), generator=g)
    lp, sel = step(wg, x.cuda(), attn, labels.cuda())
    want = reference(w, x, attn, labels, sel.cpu())
    # a logit is a sum over H of a normalised row (entries about 1) times weights of about 2 / sqrt(H): the some ten bf16
    # roundings between x and that row (2^-8 each, adding like independent ones) move it by about 2 sqrt(10) 2^-8 = 0.025
    # in the root mean square; five times that for the largest of eight
    assert (lp.cpu().double() - want).abs().max() <= 0.125
    # every answer alone (a group of one shares nothing) and a replay of the captured step give the same bits
    for i in range(8):
        one = dict(attn, cu_seqlens_q=attn["cu_seqlens_q"][:2], seqused_k=attn["seqused_k"][i : i + 1], page_table=attn["page_table"][i : i + 1],
                   group_offsets=attn["group_offsets"][:1].new_tensor([0, 1]), prefix_lens=attn["prefix_lens"][:1])
        lp1, sel1 = step(wg, x[i : i + 1].cuda(), one, labels[i : i + 1].cuda())
        assert torch.equal(sel1, sel[i : i + 1])
        assert_bitwise(lp1, lp[i : i + 1], f"answer {i} alone")
    xs = x.cuda()
    labels_g = labels.cuda()
    step(wg, xs, attn, labels_g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = step(wg, xs, attn, labels_g)
    for seed in (5, 6, 7):
        xs.copy_(torch.randn(8, H, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        eager, _ = step(wg, xs, attn, labels_g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert_bitwise(out, eager, f"replay {seed}")


def test_training_on_the_scored_answers():
    """Routing, expert products and the loss on the chosen tokens with gradients through all of them; rows of the prompt
    carry no label."""
    T = 90
    w = weights(4)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    labels = torch.randint(0, V, (T,), generator=g)
    labels[:30] = -100
    adv = torch.randn(T, generator=g)
    names = ("router", "gate", "up", "down", "head")
    wg = {n: t.cuda().requires_grad_(n in names) for n, t in w.items()}
    xg = x.cuda().requires_grad_()

    def loss(x, w, to_logits, route_fn, moe_fn, lp_fn):
        route, sel = route_fn(to_logits(x, w["router"]))
        z = x + moe_fn(x, route, sel, w)
        lp = lp_fn(z, w["head"])
        return (torch.where(labels.to(lp.device) >= 0, lp, 0.0) * adv.to(lp.device)).sum() / T, sel

    out, sel = loss(xg, wg, lambda x, r: x.float() @ r.float().t(),
                    lambda l: grouped_topk_router(l, K, score="sigmoid", bias=wg["bias"], n_groups=4, topk_groups=2, scale=1.5),
                    lambda x, route, sel, w: fused_moe_forward(num_experts=E, routing_weights=route, selected_experts=sel, hidden_states=x,
                                                               fc1_1_weight=w["gate"], fc1_2_weight=w["up"], fc2_weight=w["down"]),
                    lambda z, head: logprobs_from_hidden(z, head, labels.cuda()))
    got = torch.autograd.grad(out, (xg, *(wg[n] for n in names)))
    W = {n: t.double().requires_grad_(n in names) for n, t in w.items()}
    X = x.double().requires_grad_()
    sel = sel.cpu()

    def route64(logits):
        s = torch.sigmoid(logits).gather(1, sel)
        return 1.5 * s / s.sum(1, keepdim=True), sel

    def moe64(x, route, sel, w):
        act = torch.nn.functional.silu(torch.einsum("th,tkih->tki", x, w["gate"][sel])) * torch.einsum("th,tkih->tki", x, w["up"][sel])
        return (torch.einsum("tki,tkhi->tkh", act, w["down"][sel]) * route[..., None]).sum(1)

    ref, _ = loss(X, W, lambda x, r: x @ r.t(), route64, moe64,
                  lambda z, head: torch.log_softmax(z @ head.t(), 1).gather(1, labels.clamp(min=0)[:, None])[:, 0])
    want = torch.autograd.grad(ref, (X, *(W[n] for n in names)))
    # some dozen bf16 roundings (half a step, 2^-8 each) on the way to any of them, adding like independent ones: below
    # sqrt(12) 2^-8 = 0.014 of a gradient's norm, twice that here
    for n, a, b in zip(("x", *names), got, want):
        assert (a.cpu().double() - b).norm() <= 0.028 * b.norm(), n


def test_second_derivatives_are_refused():
    """The gradients are the kernels' in either mode; a gradient of a gradient says that there is none."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(12, 32, generator=g).cuda().requires_grad_()
    h = torch.randn(12, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    w, y = torch.randn(200, 64, generator=g).to(torch.bfloat16).cuda(), torch.randint(0, 200, (12,), generator=g).cuda()
    for f, leaf in ((lambda: grouped_topk_router(x, 4, out_dtype=torch.float32)[0].square().sum(), x), (lambda: logprobs_from_hidden(h, w, y).square().sum(), h)):
        (plain,) = torch.autograd.grad(f(), leaf)
        (again,) = torch.autograd.grad(f(), leaf, create_graph=True)
        assert_bitwise(again.detach(), plain)
        assert not plain.requires_grad and again.requires_grad
        with pytest.raises(RuntimeError, match="once_differentiable"):
            again.float().sum().backward()


@pytest.mark.parametrize("which", ["hidden", "weight", "labels", "logits"])
def test_operands_changed_before_the_backward_are_noticed(which):
    """What the backward would read again must not have changed in place; copies that were made on the way may."""
    g = torch.Generator().manual_seed(6)
    t = dict(hidden=torch.randn(2, 6, 64, generator=g).to(torch.bfloat16).cuda(), weight=torch.randn(200, 64, generator=g).to(torch.bfloat16).cuda(),
             labels=torch.randint(0, 200, (2, 6), generator=g).cuda(), logits=torch.randn(12, 32, generator=g).cuda())
    leaves = {n: t[n].requires_grad_() for n in ("hidden", "weight", "logits")}
    out = grouped_topk_router(t["logits"], 4)[0] if which == "logits" else logprobs_from_hidden(t["hidden"], t["weight"], t["labels"])
    with torch.no_grad():
        t[which].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()
    # the rows of an expanded hidden state are copied for the kernel: the gradient is that of the call
    row = t["hidden"].detach()[0, :1].clone().requires_grad_()
    lp = logprobs_from_hidden(row.expand(6, 64), leaves["weight"].detach(), torch.arange(6).cuda())
    (want,) = torch.autograd.grad(lp.sum(), row, retain_graph=True)
    with torch.no_grad():
        row.zero_()
    assert_bitwise(torch.autograd.grad(lp.sum(), row)[0], want)
