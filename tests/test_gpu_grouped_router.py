"""Grouped, biased routing and its gradient against a plain implementation in 64 bits.

The selected experts have to be equal. Weights: the kernel's arithmetic is in 64 bits, so a weight is off by the one
rounding of its type (half a step: 2^-24 fp32, 2^-8 bf16, beside a second one of 2^-24 on the way to bf16). Gradients:
the same, plus 2^-40 of the largest term of a cancelling difference.
"""

import pytest
import torch

from vexact_amd import ops
from vexact_amd.batch_invariant_ops.fused_moe import fused_moe_forward
from vexact_amd.batch_invariant_ops.router import grouped_topk_router

from .util import assert_bitwise

gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8 + 2.0**-23}


def reference(x, k, score, bias, n, kept, top, renorm, scale, d=None):
    x = x.double()
    s = torch.softmax(x, 1) if score == "softmax" else 1 / (1 + torch.exp(-x))
    c = s if bias is None else s + bias.double()
    c = torch.where(torch.isnan(c), -torch.inf, c)
    T, E = c.shape
    if n > 1:
        best = c.view(T, n, E // n).sort(dim=-1, descending=True).values[..., :top].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True).indices[:, :kept]
        ok = torch.zeros(T, n, dtype=torch.bool).scatter_(1, order, True)
        c = torch.where(ok.repeat_interleave(E // n, 1), c, -torch.inf)
    idx = c.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    sel = s.gather(1, idx)
    tot = sel.sum(1, keepdim=True) if renorm else torch.ones(T, 1, dtype=torch.float64)
    norm = torch.where(tot == 0, 0.0, sel / tot)
    if d is None:
        return norm * scale, idx
    dd = d.double() * scale
    d_sel = (dd - (dd * norm).sum(1, keepdim=True)) / tot if renorm else dd
    d_s = torch.zeros_like(s).scatter_(1, idx, torch.where(tot == 0, 0.0, d_sel))
    dx = s * (d_s - (d_s * s).sum(1, keepdim=True)) if score == "softmax" else d_s * s * (1 - s)
    largest = (dd.abs().sum(1, keepdim=True) / tot) * s  # of the terms that may cancel
    return norm * scale, idx, dx, largest


CASES = [  # T, E, k, score, bias, groups, kept, group_top
    (1, 1, 1, "softmax", False, 1, 1, 2),
    (1, 8, 3, "sigmoid", True, 1, 1, 1),
    (5, 64, 8, "softmax", True, 8, 3, 2),
    (7, 65, 6, "sigmoid", False, 5, 2, 1),
    (130, 128, 8, "softmax", False, 1, 1, 2),
    (64, 160, 6, "softmax", False, 8, 3, 1),
    (333, 256, 8, "sigmoid", True, 8, 4, 2),
    (41, 257, 10, "sigmoid", True, 1, 1, 2),
    (17, 512, 64, "sigmoid", True, 64, 64, 2),
    (16, 512, 16, "softmax", True, 64, 2, 2),
    (9, 6, 6, "softmax", True, 6, 6, 2),  # groups of one expert, every expert selected
]


@gpu
@pytest.mark.parametrize("logits,weights", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("T,E,k,score,bias,n,kept,top", CASES)
def test_forward_and_backward(T, E, k, score, bias, n, kept, top, logits, weights):
    g = torch.Generator().manual_seed(E + T)
    x = (2 * torch.randn(T, E, generator=g)).to(logits)  # bf16 logits bring exact ties
    b = 0.1 * torch.randn(E, generator=g) if bias else None
    d = torch.randn(T, k, generator=g).to(weights)
    for renorm, scale in ((True, 2.5), (False, 1.0)):
        w, idx = ops.router_topk_grouped(x.cuda(), k, score=score, bias=None if b is None else b.cuda(), n_groups=n, topk_groups=kept,
                                         group_top=top, renorm=renorm, scale=scale, out_dtype=weights)
        w_ref, idx_ref, dx_ref, largest = reference(x, k, score, b, n, kept, top, renorm, scale, d)
        assert torch.equal(idx.cpu(), idx_ref)
        assert ((w.cpu().double() - w_ref).abs() <= HALF[weights] * w_ref.abs() + 1e-40).all()
        dx = ops.router_topk_grouped_backward(x.cuda(), idx, d.cuda(), score=score, renorm=renorm, scale=scale)
        assert dx.dtype == logits
        assert ((dx.cpu().double() - dx_ref).abs() <= HALF[logits] * dx_ref.abs() + 2.0**-40 * largest + 1e-40).all()
    w32, idx32 = ops.router_topk_grouped(x.cuda(), k, score=score, bias=None if b is None else b.cuda(), n_groups=n, topk_groups=kept,
                                         group_top=top, renorm=renorm, scale=scale, out_dtype=weights, index_dtype=torch.int32)
    assert idx32.dtype == torch.int32 and torch.equal(idx32.long(), idx)
    assert_bitwise(w32, w)


@gpu
def test_close_scores_are_told_apart_and_ties_go_to_the_lower_index():
    E = 64
    x = torch.zeros(4, E)
    x[1, 40] = 1e-7  # above the others by less than a step of sigmoid's fp32 value
    x[2, 10] = -1e-7
    x[3, 63], x[3, 0] = float("inf"), float("-inf")
    for bias in (None, torch.full((E,), 0.25), torch.tensor([1e-9 * (e == 33) for e in range(E)])):
        for score in ("sigmoid", "softmax"):
            if score == "softmax":
                x = x[:3]
            for n, kept in ((1, 1), (8, 2)):
                b = None if bias is None else bias.float()
                w, idx = ops.router_topk_grouped(x.cuda(), 5, score=score, bias=None if b is None else b.cuda(), n_groups=n, topk_groups=kept)
                assert torch.equal(idx.cpu(), reference(x, 5, score, b, n, kept, 2, True, 1.0)[1]), (score, n)
        x = torch.cat([x, x[:1]])


@gpu
def test_rows_without_anything_to_choose():
    """NaN ranks with -inf, vanished scores give weights of 0, disabled experts come last."""
    E, k = 40, 4
    x = torch.randn(6, E, generator=torch.Generator().manual_seed(1))
    x[1] = float("nan")
    x[2] = -1e30  # every sigmoid is 0
    x[3, 5] = float("nan")
    b = torch.zeros(E)
    b[7:] = float("-inf")
    w, idx = ops.router_topk_grouped(x.cuda(), k, score="sigmoid", bias=b.cuda(), out_dtype=torch.float32)
    w, idx = w.cpu(), idx.cpu()
    assert ((idx >= 0) & (idx < E)).all() and all(len(set(r.tolist())) == k for r in idx)
    assert (idx[[0, 4, 5]] < 7).all() and 5 not in idx[3].tolist()
    assert torch.isnan(w[1]).all() and (w[2] == 0).all() and torch.isfinite(w[[0, 3, 4, 5]]).all()
    dx = ops.router_topk_grouped_backward(x.cuda(), idx.cuda(), torch.ones(6, k).cuda(), score="sigmoid").cpu()
    assert (dx[2] == 0).all() and torch.isfinite(dx[[0, 3, 4, 5]]).sum() == 4 * E - 1  # the one NaN logit
    assert ops.router_topk_grouped(x[:0].cuda(), k)[0].shape == (0, k)


@gpu
def test_strided_logits_rows_alone_and_a_replayed_capture():
    T, E, k = 50, 256, 8
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(T, 2 * E, generator=g).cuda()
    b = (0.1 * torch.randn(E, generator=g)).cuda()
    kw = dict(score="sigmoid", bias=b, n_groups=8, topk_groups=4, scale=2.5)
    w, idx = ops.router_topk_grouped(wide[:, 3 : 3 + E], k, **kw)
    w2, idx2 = ops.router_topk_grouped(wide[:, 3 : 3 + E].contiguous(), k, **kw)
    assert_bitwise(w, w2)
    assert torch.equal(idx, idx2)
    for i in (0, 17, 49):
        wi, ii = ops.router_topk_grouped(wide[i : i + 1, 3 : 3 + E], k, **kw)
        assert_bitwise(wi, w[i : i + 1])
        assert torch.equal(ii, idx[i : i + 1])
    x = wide[:, :E].contiguous()
    d = torch.randn(T, k, generator=g).cuda()

    def step():
        w, i = ops.router_topk_grouped(x, k, **kw)
        return w, i, ops.router_topk_grouped_backward(x, i, d, score="sigmoid", scale=2.5)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6, 7):
        x.copy_(torch.randn(T, E, generator=torch.Generator().manual_seed(seed)))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert_bitwise(a, c)


@gpu
@pytest.mark.parametrize("E,n", [(8, 4), (512, 64)])
def test_group_score_that_is_no_number(E, n):
    """The best two of group 0 are +inf and -inf: their sum is NaN, which ranks with -inf, so the group goes last."""
    size = E // n
    bias = torch.zeros(E)
    bias[:size] = -torch.inf
    bias[1] = torch.inf
    x = torch.randn(5, E, generator=torch.Generator().manual_seed(8))
    _, idx = ops.router_topk_grouped(x.cuda(), 2, score="sigmoid", bias=bias.cuda(), n_groups=n, topk_groups=2)
    s = torch.sigmoid(x.double()).view(5, n, size)
    best = s[:, 1:].sort(dim=-1, descending=True).values[..., :2].sum(-1).sort(dim=-1, descending=True).indices[:, :2] + 1
    ok = torch.zeros(5, n, dtype=torch.bool).scatter_(1, best, True).repeat_interleave(size, 1)
    want = torch.where(ok, s.view(5, E), -torch.inf).sort(dim=-1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(idx.cpu(), want)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_backward_of_an_expert_selected_twice(score, renorm):
    """A selection of the caller's own may name an expert more than once: its gradients add up."""
    T, E, k = 9, 96, 6
    g = torch.Generator().manual_seed(9)
    x, d = torch.randn(T, E, generator=g), torch.randn(T, k, generator=g)
    idx = torch.randint(0, 4, (T, k), generator=g) * 30  # six of four experts
    got = ops.router_topk_grouped_backward(x.cuda(), idx.cuda(), d.cuda(), score=score, renorm=renorm, scale=1.5).cpu().double()
    X = x.double().requires_grad_()
    s = torch.softmax(X, 1) if score == "softmax" else torch.sigmoid(X)
    sel = s.gather(1, idx)
    w = 1.5 * sel / sel.sum(1, keepdim=True) if renorm else 1.5 * sel
    (want,) = torch.autograd.grad(w, X, d.double())
    # one rounding to fp32, and 2^-40 of the terms that may cancel: at most 2 k scale max |d|, as s <= 1 and 1 / S times
    # a selected score <= 1
    assert (got - want).abs().le(2.0**-24 * want.abs() + 2.0**-40 * 2 * k * 1.5 * d.abs().max()).all()


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(score):
    T, E, k, eps = 6, 32, 4, 2.0**-9
    x = (torch.randn(T, E, generator=torch.Generator().manual_seed(3)) * 64).round() / 64
    xg = x.cuda().requires_grad_()
    w, idx = grouped_topk_router(xg, k, score=score, n_groups=4, topk_groups=2, scale=2.0, out_dtype=torch.float32)
    d = torch.randn(T, k, generator=torch.Generator().manual_seed(4))
    (g,) = torch.autograd.grad(w, xg, d.cuda())
    # the selection held fixed, the weights as the kernel computes them at x +- eps: a smooth function of the logits
    step = torch.randn(T, E, generator=torch.Generator().manual_seed(5)).sign() * eps

    def value(z):
        s = torch.softmax(z.double(), 1) if score == "softmax" else torch.sigmoid(z.double())
        sel = s.gather(1, idx.cpu())
        return (2.0 * sel / sel.sum(1, keepdim=True) * d.double()).sum(1)

    diff = (value(x + step) - value(x - step)) / 2
    # the remainder: a sixth of the third derivative along the step, below 2 (4 eps)^3 sum |d|
    assert ((g.cpu().double() * step.double()).sum(1) - diff).abs().le(2 * (4 * eps) ** 3 * d.double().abs().sum(1) + 2.0**-22 * eps * E).all()


@gpu
def test_routes_the_expert_products():
    """The router's outputs as the expert block takes them, with gradients through both."""
    T, H, I, E, k = 48, 128, 64, 16, 4
    g = torch.Generator().manual_seed(7)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    wr = (torch.randn(E, H, generator=g) / H**0.5).cuda().requires_grad_()
    gate, up, down = (0.1 * torch.randn(E, a, b, generator=g) for a, b in ((I, H), (I, H), (H, I)))
    gate, up, down = (t.to(torch.bfloat16).cuda().requires_grad_() for t in (gate, up, down))
    bias = (0.1 * torch.randn(E, generator=g)).cuda()
    logits = x.float() @ wr.t()
    weights, selected = grouped_topk_router(logits, k, score="sigmoid", bias=bias, n_groups=4, topk_groups=2, scale=2.0)
    y = fused_moe_forward(num_experts=E, routing_weights=weights, selected_experts=selected, hidden_states=x, fc1_1_weight=gate,
                          fc1_2_weight=up, fc2_weight=down)
    dy = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    grads = torch.autograd.grad(y, (wr, x, down), dy)
    # the same in 64 bits on the CPU, with the selection given
    X, WR, G, U, D = (t.detach().cpu().double().requires_grad_() for t in (x, wr, gate, up, down))
    s = torch.sigmoid(X @ WR.t()).gather(1, selected.cpu())
    w = 2.0 * s / s.sum(1, keepdim=True)
    a = torch.einsum("th,tkih->tki", X, G[selected.cpu()])
    h = torch.nn.functional.silu(a) * torch.einsum("th,tkih->tki", X, U[selected.cpu()])
    Y = (torch.einsum("tki,tkhi->tkh", h, D[selected.cpu()]) * w[..., None]).sum(1)
    ref = torch.autograd.grad(Y, (WR, X, D), dy.cpu().double())
    # a chain of at most eight bf16 roundings (half a step each, 2^-8) between input and output
    assert (y.cpu().double() - Y).norm() <= 8 * 2.0**-8 * Y.norm()
    for got, want in zip(grads, ref):
        assert (got.cpu().double() - want).norm() <= 8 * 2.0**-8 * want.norm()


def test_refusals():
    with pytest.raises(ValueError, match="CUDA tensor"):
        grouped_topk_router(torch.zeros(2, 8), 2)


@gpu
def test_refusals_on_the_gpu():
    x = torch.zeros(2, 8).cuda()
    for call, what in (
        (lambda: ops.router_topk_grouped(x, 9), "at most"), (lambda: ops.router_topk_grouped(x, 0), "top_k"),
        (lambda: ops.router_topk_grouped(x.half(), 2), "float32 or bfloat16"), (lambda: ops.router_topk_grouped(x, 2, score="tanh"), "score"),
        (lambda: ops.router_topk_grouped(x, 2, n_groups=3), "equal groups"), (lambda: ops.router_topk_grouped(x, 2, n_groups=4, topk_groups=5), "equal groups"),
        (lambda: ops.router_topk_grouped(x, 3, n_groups=4, topk_groups=1), "do not hold"), (lambda: ops.router_topk_grouped(x, 2, group_top=3), "group_top"),
        (lambda: ops.router_topk_grouped(x, 2, bias=torch.zeros(7).cuda()), "bias"), (lambda: ops.router_topk_grouped(x, 2, bias=torch.zeros(8)), "bias"),
        (lambda: ops.router_topk_grouped(torch.zeros(2, 513).cuda(), 2), "512"), (lambda: ops.router_topk_grouped(x, 2, out_dtype=torch.float16), "dtypes"),
        (lambda: ops.router_topk_grouped_backward(x, torch.zeros(3, 2, dtype=torch.int64).cuda(), torch.zeros(3, 2).cuda()), "top_k"),
    ):
        with pytest.raises(ValueError, match=what):
            call()


def test_c_abi_refusals():
    from vexact_amd import _lib

    a, lib = 4096, _lib.load()

    def fwd(**kw):
        v = {"x": a, "w": a, "i": a, "T": 4, "E": 16, "k": 2, "n": 1, "kept": 1, "top": 2, **kw}
        return lib.vx_router_grouped(v["x"], None, v["w"], v["i"], v["T"], v["E"], v["k"], 16, 0, v["n"], v["kept"], v["top"], 1, 1.0, 0, 0, 1, None)

    assert fwd(T=0) == 0
    assert fwd(x=None) == fwd(w=None) == fwd(i=None) == fwd(T=-1) == fwd(E=0) == fwd(k=0) == fwd(k=17) == fwd(n=3) == fwd(n=0) == -1
    assert fwd(n=4, kept=5) == fwd(n=8, kept=0) == fwd(n=8, kept=1, k=3) == fwd(top=3) == -1
    assert fwd(E=520) == fwd(E=128, k=65) == fwd(E=128, n=128, kept=8) == -2
    bwd = lambda **kw: lib.vx_router_grouped_bwd(*[{"x": a, "i": a, "d": a, "o": a, **kw}[n] for n in "xido"], kw.get("T", 0), kw.get("E", 16), 2, 16, 16, 0, 1, 1.0, 0, 0, None)  # noqa: E731
    assert bwd() == 0 and bwd(x=None) == bwd(o=None) == bwd(T=-1) == -1 and bwd(E=600) == -2
