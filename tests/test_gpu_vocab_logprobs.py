"""Log-probabilities from hidden states and their gradients against a plain implementation in 64 bits.

Tolerances. Forward: a logit is a sum of H products accumulated in fp32; its rounding errors add like independent ones,
so 8 sqrt(H) 2^-24 sum_k |h_k w_k| covers a logit, and twice that a log-probability (its own logit and the lse, which
moves by at most the largest logit error), beside a few fp32 steps of the result. Gradients: every entry of the logits'
derivative is rounded to bf16 once (half a step, 2^-8 relative), which moves an output by at most 2^-8 sum |dx| |w|;
the result is rounded to bf16 once more (2^-8 of itself); 2^-11 of the same sum covers the fp32 part (a probability's
relative error is that of its exponent's argument, below 2^-13 here) and the accumulation.
"""

import pytest
import torch

from vexact_amd import ops
from vexact_amd.batch_invariant_ops.standalone_logprobs import logprobs_from_hidden

from .util import assert_bitwise

gpu = pytest.mark.gpu


def make(T, V, H, seed=0, ignored=0, spread=1.8):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g).to(torch.bfloat16)
    w = (spread / H**0.5 * torch.randn(V, H, generator=g)).to(torch.bfloat16)
    y = torch.randint(0, V, (T,), generator=g)
    y[torch.randperm(T, generator=g)[:ignored]] = -100
    return h, w, y


def reference(h, w, y, temperature=1.0, d=None):
    h64, w64 = h.double(), w.double()
    x = h64 @ w64.t() / temperature
    lse = torch.logsumexp(x, 1)
    ok = (y >= 0) & (y < w.shape[0])
    at = y.clamp(0, w.shape[0] - 1)
    lp = torch.where(ok, x.gather(1, at[:, None])[:, 0] - lse, torch.nan)
    if d is None:
        return lp, lse
    dd = torch.where(ok, d.double(), 0.0) / temperature
    dx = -torch.exp(x - lse[:, None]) * dd[:, None]
    dx[torch.arange(len(y)), at] += dd
    return lp, lse, dx, dx @ w64, dx.t() @ h64


def check_forward(h, w, y, out, lse, temperature=1.0):
    lp_ref, lse_ref = reference(h, w, y, temperature)
    mass = (h.double().abs() @ w.double().abs().t()).max() / temperature
    tol = 16 * h.shape[1] ** 0.5 * 2.0**-24 * mass + 4 * 2.0**-24 * lse_ref.abs().max() + 2.0**-20
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(lp_ref))
    ok = ~torch.isnan(lp_ref)
    assert (out.cpu().double() - lp_ref)[ok].abs().max() <= tol if ok.any() else True
    assert (lse.cpu().double() - lse_ref).abs().max() <= tol


# rows on both sides of the kernels' tile heights; vocabularies that end inside a strip, a tile and a segment; depths
# that are and are not a multiple of the wide kernel's step
SHAPES = [(1, 1, 8), (1, 5, 64), (3, 64, 64), (7, 257, 72), (64, 1000, 128), (65, 1000, 128), (100, 1024, 136), (129, 8192, 64),
          (300, 8193, 192), (257, 20011, 128), (513, 16449, 256), (30, 20011, 520),
          (300, 30001, 64), (700, 16449, 512)]


@gpu
@pytest.mark.parametrize("T,V,H", SHAPES)
def test_forward(T, V, H):
    h, w, y = make(T, V, H, seed=T, ignored=T // 5)
    if T > 2:
        y[0], y[1] = V - 1, V  # the last token, and one past it
    out, lse = ops.vocab_logprobs(h.cuda(), w.cuda(), y.cuda(), 0.7)
    check_forward(h, w, y, out, lse, 0.7)


@gpu
@pytest.mark.parametrize("T,V,H", SHAPES)
def test_backward(T, V, H):
    h, w, y = make(T, V, H, seed=T + 1, ignored=T // 5)
    d = torch.randn(T, generator=torch.Generator().manual_seed(3))
    hg, wg, yg = h.cuda(), w.cuda(), y.cuda()
    _, lse = ops.vocab_logprobs(hg, wg, yg, 1.3)
    dh, dw = ops.vocab_logprobs_backward(hg, wg, yg, lse, d.cuda(), 1.3)
    _, _, dx, dh_ref, dw_ref = reference(h, w, y, 1.3, d)
    slack = 2.0**-8 + 2.0**-11
    tol_h = slack * (dx.abs() @ w.double().abs()) + 2.0**-8 * dh_ref.abs() + 1e-30
    tol_w = slack * (dx.abs().t() @ h.double().abs()) + 2.0**-8 * dw_ref.abs() + 1e-30
    assert ((dh.cpu().double() - dh_ref).abs() <= tol_h).all()
    assert ((dw.cpu().double() - dw_ref).abs() <= tol_w).all()
    # one gradient alone is the same
    assert_bitwise(ops.vocab_logprobs_backward(hg, wg, yg, lse, d.cuda(), 1.3, need_weight=False)[0], dh, "d_hidden alone")
    assert_bitwise(ops.vocab_logprobs_backward(hg, wg, yg, lse, d.cuda(), 1.3, need_hidden=False)[1], dw, "d_weight alone")


@gpu
@pytest.mark.parametrize("V,H", [(20011, 128), (30001, 128), (1000, 72)])
def test_rows_do_not_depend_on_the_batch(V, H):
    h, w, y = (t.cuda() for t in make(600, V, H, seed=5))
    out, lse = ops.vocab_logprobs(h, w, y)
    d = torch.randn(600, generator=torch.Generator().manual_seed(1)).cuda()
    dh, _ = ops.vocab_logprobs_backward(h, w, y, lse, d)
    for a, b in ((0, 1), (17, 24), (100, 164), (100, 165), (300, 600)):
        o2, l2 = ops.vocab_logprobs(h[a:b], w, y[a:b])
        assert_bitwise(o2, out[a:b], f"rows {a}..{b}")
        assert_bitwise(l2, lse[a:b], f"lse of rows {a}..{b}")
        dh2, _ = ops.vocab_logprobs_backward(h[a:b], w, y[a:b], l2, d[a:b], need_weight=False)
        assert_bitwise(dh2, dh[a:b], f"d_hidden of rows {a}..{b}")


@gpu
def test_pieces_of_the_vocabulary_change_nothing():
    """Enough rows for several pieces: the gradient of the first rows is that of a one-piece call."""
    V, H, T = 40000, 128, 12000
    h, w, y = (t.cuda() for t in make(T, V, H, seed=6))
    out, lse = ops.vocab_logprobs(h, w, y)
    d = torch.randn(T, generator=torch.Generator().manual_seed(2)).cuda()
    dh, dw = ops.vocab_logprobs_backward(h, w, y, lse, d)
    few = ops.vocab_logprobs_backward(h[:200], w, y[:200], lse[:200], d[:200], need_weight=False)[0]
    assert_bitwise(dh[:200], few, "first rows")
    # the weight gradient of all rows against products of the logits' derivative in 32 bits
    x = h.float() @ w.float().t()
    dx = -torch.exp(x - lse[:, None]) * d[:, None]
    dx.scatter_add_(1, y[:, None], d[:, None])
    ref, mass = dx.t() @ h.float(), dx.abs().t() @ h.float().abs()
    assert ((dw.float() - ref).abs() <= (2.0**-8 + 2.0**-10) * mass + 2.0**-8 * ref.abs()).all()


@gpu
def test_strided_operands_and_special_rows():
    T, V, H = 70, 500, 128
    h, w, y = make(T, V, H, seed=8)
    hb, wb = torch.zeros(T, H + 24, dtype=torch.bfloat16).cuda(), torch.zeros(V, 2 * H, dtype=torch.bfloat16).cuda()
    hb[:, 8 : 8 + H], wb[:, H:] = h.cuda(), w.cuda()
    base, lse = ops.vocab_logprobs(h.cuda(), w.cuda(), y.cuda())
    for hv, wv in ((hb[:, 8 : 8 + H], wb[:, H:]), (h.cuda().t().contiguous().t(), w.cuda()), (h.cuda(), w.cuda().t().contiguous().t())):
        out, l2 = ops.vocab_logprobs(hv, wv, y.cuda())
        assert_bitwise(out, base)
        assert_bitwise(l2, lse)
        d = torch.ones(T).cuda()
        for a, b in zip(ops.vocab_logprobs_backward(hv, wv, y.cuda(), l2, d), ops.vocab_logprobs_backward(h.cuda(), w.cuda(), y.cuda(), lse, d)):
            assert_bitwise(a, b)
    # a row with a NaN is NaN, its neighbours are not touched; a huge row does not overflow
    h2 = h.clone()
    h2[3, 5] = float("nan")
    h2[4] *= 1000
    out, l2 = ops.vocab_logprobs(h2.cuda(), w.cuda(), y.cuda())
    keep = [i for i in range(T) if i not in (3, 4)]
    assert torch.isnan(out[3]) and torch.isnan(l2[3]) and torch.isfinite(out[4])
    assert_bitwise(out[keep], base[keep])
    # no rows at all; rows without any label: no gradient, whatever d_out holds
    assert ops.vocab_logprobs(h[:0].cuda(), w.cuda(), y[:0].cuda())[0].shape == (0,)
    dh, dw = ops.vocab_logprobs_backward(h[:0].cuda(), w.cuda(), y[:0].cuda(), l2[:0], torch.ones(0).cuda())
    assert dh.shape == (0, H) and not dw.any()
    none = torch.full((T,), -1).cuda()
    assert torch.isnan(ops.vocab_logprobs(h.cuda(), w.cuda(), none)[0]).all()
    dh, dw = ops.vocab_logprobs_backward(h.cuda(), w.cuda(), none, lse, torch.full((T,), float("nan")).cuda())
    assert not dh.any() and not dw.any()
    # padding rows may hold anything: nothing of it reaches d_weight or the other rows
    y2, h3 = y.clone(), h.clone()
    y2[[2, 5, 69]] = torch.tensor([-100, -1, V])
    h3[2], h3[5], h3[69] = float("nan"), float("inf"), float("-inf")
    clean = h.clone()
    clean[[2, 5, 69]] = 0
    got, want = [], []
    for hh, dst in ((h3, got), (clean, want)):
        _, ls = ops.vocab_logprobs(hh.cuda(), w.cuda(), y2.cuda())
        dst.extend(ops.vocab_logprobs_backward(hh.cuda(), w.cuda(), y2.cuda(), ls, torch.ones(T).cuda()))
    assert torch.isfinite(got[1]).all() and not got[0][[2, 5, 69]].any()
    for a, b in zip(got, want):
        assert_bitwise(a, b, "padding rows")


@gpu
def test_rows_far_apart():
    """Rows further apart than the kernels' 32-bit offsets of a piece allow: the values of copies that lie close."""
    T, V, H, pitch = 5, 70, 64, (1 << 18) + 8
    h, w, y = (t.cuda() for t in make(T, V, H, seed=21))
    far = lambda t: torch.zeros(len(t), pitch, dtype=t.dtype, device="cuda")[:, :H].copy_(t)  # noqa: E731
    hf, wf = far(h), far(w)
    assert hf.stride(0) == wf.stride(0) == pitch
    d = torch.linspace(-1, 1, T).cuda()
    near, apart = ops.vocab_logprobs(h, w, y), ops.vocab_logprobs(hf, wf, y)
    for a, b in zip(near + ops.vocab_logprobs_backward(h, w, y, near[1], d), apart + ops.vocab_logprobs_backward(hf, wf, y, near[1], d)):
        assert_bitwise(a, b)


@gpu
def test_weights_beyond_four_gib():
    """Byte offsets past 32 bits, in the forward's column ranges and the backward's pieces."""
    T, V, H = 70, 270000, 8192
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(V, H, generator=g, device="cuda", dtype=torch.bfloat16) * 0.02
    h = torch.randn(T, H, generator=g, device="cuda", dtype=torch.bfloat16)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[:3] = torch.tensor([V - 1, 0, V - 300])
    x = torch.cat([h.float() @ part.float().t() for part in w.split(30000)], 1)
    lse_ref = torch.logsumexp(x.double(), 1)
    lp_ref = x.gather(1, y[:, None])[:, 0].double() - lse_ref
    # fp32 sums of 8192 products on both sides: sqrt(8192) 2^-24 of the root sum of squares of the products (about 1.8) is
    # 1e-5; ten times that for the largest of the rows
    for rows in (5, T):
        out, lse = ops.vocab_logprobs(h[:rows], w, y[:rows])
        assert (out.double() - lp_ref[:rows]).abs().max() <= 1e-4 and (lse.double() - lse_ref[:rows]).abs().max() <= 1e-4
    d = torch.randn(T, generator=g, device="cuda")
    dh, dw = ops.vocab_logprobs_backward(h, w, y, lse, d)
    dx = -torch.exp(x - lse_ref[:, None].float()) * d[:, None]
    dx.scatter_add_(1, y[:, None], d[:, None])
    dh_ref = sum(dx[:, i : i + 30000] @ w[i : i + 30000].float() for i in range(0, V, 30000))
    assert (dh.float() - dh_ref).norm() <= 2.0**-7 * dh_ref.norm()
    for i in (0, V - 300, V - 1):
        ref = dx[:, i] @ h.float()
        assert (dw[i].float() - ref).norm() <= 2.0**-7 * ref.norm()


@gpu
def test_autograd_shapes_and_differences():
    B, S, V, H = 2, 40, 700, 64
    h, w, y = make(B * S, V, H, seed=9)
    hg, wg, yg = h.view(B, S, H).cuda().requires_grad_(), w.cuda().requires_grad_(), y.view(B, S).cuda()
    out = logprobs_from_hidden(hg, wg, yg, temperature=0.9)
    assert out.shape == (B, S) and out.dtype == torch.float32
    d = torch.randn(B, S, generator=torch.Generator().manual_seed(4)).cuda()
    (out * d).sum().backward()
    assert hg.grad.shape == hg.shape and wg.grad.shape == wg.shape and hg.grad.dtype == torch.bfloat16
    ref = reference(h, w, y, 0.9, d.cpu().reshape(-1))
    assert (hg.grad.cpu().double().view(-1, H) - ref[3]).norm() <= 2.0**-7 * ref[3].norm()
    assert (wg.grad.cpu().double() - ref[4]).norm() <= 2.0**-7 * ref[4].norm()
    with torch.no_grad():
        assert_bitwise(logprobs_from_hidden(hg, wg, yg, temperature=0.9), out.detach(), "without autograd")
    # central differences along a direction of exactly representable steps, in the function's own outputs: the remainder
    # is a sixth of the third derivative, at most (range of the logits' change)^3 per row
    grid = (h.float() * 8).round() / 8  # multiples of 1/8: +- 1/64 stays exact below 2, which is enforced
    grid = grid.clamp(-1.75, 1.75)
    step = torch.randn(B * S, H, generator=torch.Generator().manual_seed(7)).sign() / 64
    f = lambda z: ops.vocab_logprobs(z.to(torch.bfloat16).cuda(), wg.detach(), yg.reshape(-1), 0.9)  # noqa: E731
    mid, lse = f(grid)
    dh, _ = ops.vocab_logprobs_backward(grid.to(torch.bfloat16).cuda(), wg.detach(), yg.reshape(-1), lse, torch.ones(B * S).cuda(), 0.9, need_weight=False)
    slope = (dh.cpu().double() * step.double()).sum(1)
    diff = (f(grid + step)[0] - f(grid - step)[0]).cpu().double() / 2
    moved = (step.double() @ w.double().t()) / 0.9
    spread = moved.max(1).values - moved.min(1).values
    dx_mass = 2 / 0.9 * (w.double().abs().max() * step.abs().sum(1).double())  # sum |dx| <= 2 / temperature
    tol = spread**3 / 6 + 2.0**-7 * dx_mass + 2.0**-18
    assert ((slope - diff).abs() <= tol).all()
    assert (slope - diff).norm() <= 0.1 * slope.norm()


@gpu
def test_frozen_projection_and_second_stream():
    T, V, H = 130, 3001, 128
    h, w, y = make(T, V, H, seed=11)
    hg = h.cuda().requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    wg, yg = w.cuda(), y.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        out = logprobs_from_hidden(hg, wg, yg)
        (g,) = torch.autograd.grad(out.sum(), hg)
    torch.cuda.current_stream().wait_stream(stream)
    _, lse = ops.vocab_logprobs(hg.detach(), wg, yg)
    assert_bitwise(g, ops.vocab_logprobs_backward(hg.detach(), wg, yg, lse, torch.ones(T).cuda(), need_weight=False)[0])


@gpu
def test_captured_forward_and_backward_replay():
    T, V, H = 140, 9000, 128
    h, w, y = (t.cuda() for t in make(T, V, H, seed=12))
    d = torch.randn(T, generator=torch.Generator().manual_seed(5)).cuda()

    def step():
        out, lse = ops.vocab_logprobs(h, w, y)
        return (out, *ops.vocab_logprobs_backward(h, w, y, lse, d))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (21, 22, 23):
        h2, _, y2 = make(T, V, H, seed=seed)
        h.copy_(h2)
        y.copy_(y2)
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert_bitwise(a, b, f"replay on inputs {seed}")


def test_refusals():
    h, w, y = make(4, 10, 16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.vocab_logprobs(h, w, y)
    with pytest.raises(ValueError, match="shape of hidden's rows"):
        logprobs_from_hidden(h, w, y[:3])


@gpu
def test_refusals_on_the_gpu():
    h, w, y = (t.cuda() for t in make(4, 10, 16))
    for args, what in (((h.half(), w.half(), y), "bfloat16"), ((h, w[:, :8], y), "need hidden"), ((h, w, y[:3]), "one per row"),
                       ((h, w, y.float()), "integers"), ((h[:, :12], w[:, :12], y), "multiple of 8"), ((h, w[:0], y), "V positive"),
                       ((h, w.cpu(), y), "one device")):
        with pytest.raises(ValueError, match=what):
            ops.vocab_logprobs(*args)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.vocab_logprobs(h, w, y, bad)
    with pytest.raises(ValueError, match="one entry per row"):
        ops.vocab_logprobs_backward(h, w, y, torch.zeros(3).cuda(), torch.zeros(4).cuda())


def test_c_abi_refusals():
    """Bad arguments come back as status codes before anything is launched (no GPU needed)."""
    from vexact_amd import _lib

    lib = _lib.load()
    a = 4096  # an aligned non-null address that is never read
    ok = dict(h=a, w=a, y=a, o=a, l=a, T=4, V=10, H=16, ldh=16, ldw=16, ws=a, n=1 << 20)

    def fwd(**kw):
        v = {**ok, **kw}
        return lib.vx_vocab_logprobs(v["h"], v["w"], v["y"], v["o"], v["l"], v["T"], v["V"], v["H"], v["ldh"], v["ldw"], 1.0, v["ws"], v["n"], None)

    assert fwd(T=0) == 0
    assert fwd(h=None) == fwd(w=None) == fwd(y=None) == fwd(o=None, l=None) == fwd(T=-1) == fwd(V=0) == fwd(H=0) == -1
    assert fwd(H=12) == fwd(ldh=12) == fwd(ldw=20) == fwd(h=a + 2) == -2
    assert fwd(ws=None) == fwd(n=16) == fwd(ws=a + 4) == -3

    def bwd(**kw):
        v = {**ok, "dh": a, "dw": a, "g": a, "ldd": 16, **kw}
        return lib.vx_vocab_logprobs_bwd(v["h"], v["w"], v["y"], v["l"], v["g"], v["dh"], v["dw"], v["T"], v["V"], v["H"], v["ldh"], v["ldw"],
                                         v["ldd"], v["ldd"], 1.0, v["ws"], v["n"], None)

    assert bwd(T=0) == bwd(g=None) == bwd(l=None) == bwd(dh=None, dw=None) == -1
    assert bwd(H=12) == bwd(ldd=18) == bwd(dh=a + 4) == bwd(T=1 << 28, n=1 << 60) == -2
    assert bwd(ws=None) == bwd(n=16) == -3


def test_c_abi_refuses_rows_too_far_apart():
    """A row pitch that no split of the rows or of the vocabulary brings within 32-bit offsets is refused."""
    from vexact_amd import _lib

    lib, a = _lib.load(), 4096
    for H, ldh, ldw in ((16, 1 << 23, 16), (16, 16, 1 << 23), (16, 1 << 40, 16), (16, 16, 1 << 40), (1 << 23, 1 << 23, 1 << 23), (16, -16, 16), (16, 16, -16)):
        assert lib.vx_vocab_logprobs(a, a, a, a, a, 4, 10, H, ldh, ldw, 1.0, a, 1 << 40, None) == -2
        assert lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, 4, 10, H, ldh, ldw, H, H, 1.0, a, 1 << 60, None) == -2


def _entries(h, ldh, w, ldw, y, d, T, V, H):
    """The C entry points, with row pitches that no tensor of the front end has: (out, lse, d_hidden, d_weight)."""
    from vexact_amd import _lib

    lib = _lib.load()
    f = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    out, lse, dh, dw = f(T), f(T), f(T, H, dtype=torch.bfloat16), f(V, H, dtype=torch.bfloat16)
    ws = f(max(lib.vx_vocab_logprobs_workspace_bytes(T, V), lib.vx_vocab_logprobs_bwd_workspace_bytes(T, V, H)), dtype=torch.uint8)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.vx_vocab_logprobs(h.data_ptr(), w.data_ptr(), y.data_ptr(), out.data_ptr(), lse.data_ptr(), T, V, H, ldh, ldw, 1.0,
                                     ws.data_ptr(), ws.numel(), stream), "forward")
    _lib.check(lib.vx_vocab_logprobs_bwd(h.data_ptr(), w.data_ptr(), y.data_ptr(), lse.data_ptr(), d.data_ptr(), dh.data_ptr(), dw.data_ptr(),
                                         T, V, H, ldh, ldw, H, H, 1.0, ws.data_ptr(), ws.numel(), stream), "backward")
    return out, lse, dh, dw


@gpu
@pytest.mark.parametrize("T,V,H", [(5, 70, 64), (300, 9000, 128), (70, 300, 72)])
def test_one_row_for_all(T, V, H):
    """A row pitch of zero, of the hidden states and of the weights: the values of copies of that row."""
    h, w, y = (t.cuda() for t in make(T, V, H, seed=31))
    d = torch.linspace(-1, 1, T).cuda()
    h1, w1 = h[:1].expand(T, H).contiguous(), w[:1].expand(V, H).contiguous()
    for got, want in ((_entries(h, 0, w, H, y, d, T, V, H), _entries(h1, H, w, H, y, d, T, V, H)),
                      (_entries(h, H, w, 0, y, d, T, V, H), _entries(h, H, w1, H, y, d, T, V, H))):
        for a, b in zip(got, want):
            assert_bitwise(a, b)


def test_c_abi_zero_row_pitch():
    """The plan of the backward's pieces does not divide by a row pitch of zero (no GPU needed: the workspace is too small)."""
    from vexact_amd import _lib

    lib, a = _lib.load(), 4096
    for ldh, ldw in ((16, 0), (0, 16), (0, 0), (16, 8)):
        assert lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, 4, 10, 16, ldh, ldw, 16, 16, 1.0, a, 16, None) == -3
    # what the workspace function promises is enough whatever the pitch, also where a row's length splits the vocabulary
    T, V, H = 4, 1 << 20, 1 << 17
    n = lib.vx_vocab_logprobs_bwd_workspace_bytes(T, V, H)
    for ldw in (0, 8, H, H + 8):
        assert lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, T, V, H, H, ldw, H, H, 1.0, a + 8, n, None) == -3  # misaligned, after the plan
        assert lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, T, V, H, H, ldw, H, H, 1.0, a, n // 2, None) == -3


@gpu
def test_temperatures():
    """Those whose reciprocal fp32 does not hold are refused; at the largest allowed the distribution is uniform, whether or not
    the vocabulary ends inside a tile; at a small one the largest logit takes it all."""
    for V in (500, 512, 64):
        h, w, y = make(70, V, 64, seed=33)
        for bad in (float("inf"), 2.0**127, 2.0**-128, 1e-45, 5e-324, -float("inf")):
            with pytest.raises(ValueError, match="temperature"):
                ops.vocab_logprobs(h.cuda(), w.cuda(), y.cuda(), bad)
            with pytest.raises(ValueError, match="temperature"):
                logprobs_from_hidden(h.cuda().requires_grad_(), w.cuda(), y.cuda(), bad)
        for rows in (7, 70):
            out, lse = ops.vocab_logprobs(h[:rows].cuda(), w.cuda(), y[:rows].cuda(), 2.0**126)
            # logits below 2^-120, exponentials of 1, an exact sum: one step of a base-2 logarithm in [8, 16) (2^-20, times
            # log 2), half a step of its product with log 2 (2^-22) and that constant's own rounding (2^-21) are left
            want = torch.log(torch.tensor(float(V), dtype=torch.float64))
            assert ((lse.cpu().double() - want).abs() <= 2.0**-19).all() and ((out.cpu().double() + want).abs() <= 2.0**-19).all()
            best = (h[:rows].double() @ w.double().t()).topk(2, 1)
            sure = best.values[:, 0] - best.values[:, 1] > 1e-3  # times 2^20: nothing is left of the others
            out, _ = ops.vocab_logprobs(h[:rows].cuda(), w.cuda(), best.indices[:, 0].cuda(), 2.0**-20)
            # 0 up to the rounding of the scaled maximum
            assert sure.any() and (out.cpu().double().abs() <= 2.0**-23 * 2.0**20 * best.values[:, 0].abs())[sure].all()


def test_c_abi_refuses_scales_out_of_range():
    from vexact_amd import _lib

    lib, a = _lib.load(), 4096
    for scale in (0.0, -1.0, float("inf"), float("nan"), 1e-39, 2.0**127 * 1.5):
        assert lib.vx_vocab_logprobs(a, a, a, a, a, 4, 10, 16, 16, 16, scale, a, 16, None) == -1
        assert lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, 4, 10, 16, 16, 16, 16, 16, scale, a, 16, None) == -1
    for scale in (2.0**-126, 2.0**127):
        assert lib.vx_vocab_logprobs(a, a, a, a, a, 4, 10, 16, 16, 16, scale, a, 16, None) == -3


# d_hidden by 256 x 256 tiles (what more than 1152 workgroups of 64 or 96 rows x 64 columns x 8192 tokens come to, per round of
# 256 tiles): segments that end inside a step of 64 tokens, a last segment of 10 tokens, one segment that is shorter than a step,
# a depth that ends inside a tile, several pieces of several segments
WIDE = [(3000, 20011, 1024), (3001, 8202, 1536), (6000, 50, 1536), (3000, 20011, 1000), (12000, 40001, 512)]


@gpu
@pytest.mark.parametrize("T,V,H", WIDE)
def test_backward_of_large_batches(T, V, H):
    h, w, y = (t.cuda() for t in make(T, V, H, seed=T + 7, ignored=T // 7))
    d = torch.randn(T, generator=torch.Generator().manual_seed(3)).cuda()
    _, lse = ops.vocab_logprobs(h, w, y, 1.3)
    dh, dw = ops.vocab_logprobs_backward(h, w, y, lse, d, 1.3)
    _, _, dx, dh_ref, dw_ref = reference(h, w, y, 1.3, d)
    slack = 2.0**-8 + 2.0**-11
    assert ((dh.double() - dh_ref).abs() <= slack * (dx.abs() @ w.double().abs()) + 2.0**-8 * dh_ref.abs() + 1e-30).all()
    assert ((dw.double() - dw_ref).abs() <= slack * (dx.abs().t() @ h.double().abs()) + 2.0**-8 * dw_ref.abs() + 1e-30).all()
    assert not dh[(y < 0)].any()
    again = ops.vocab_logprobs_backward(h, w, y, lse, d, 1.3)
    assert_bitwise(again[0], dh, "d_hidden again")
    assert_bitwise(again[1], dw, "d_weight again")
    # small batches take other kernels (tiles of 64 and 96 rows): the same bits
    for a, b in ((0, 1), (250, 350), (T - 257, T)):
        few = ops.vocab_logprobs_backward(h[a:b], w, y[a:b], lse[a:b], d[a:b], 1.3, need_weight=False)[0]
        assert_bitwise(few, dh[a:b], f"d_hidden of rows {a}..{b}")


@gpu
@pytest.mark.parametrize("T", [16500, 33000])
def test_rows_in_several_launches(T):
    """Rows 256 KB apart, more than 4 GiB of them: the logits of a launch reach as far as its 32-bit offsets."""
    V, H, pitch = 300, 64, 1 << 17
    h, w, y = (t.cuda() for t in make(T, V, H, seed=41, ignored=9))
    far = torch.empty(T, pitch, dtype=h.dtype, device="cuda")[:, :H].copy_(h)
    assert far.stride(0) == pitch and T * pitch * 2 > 1 << 32
    d = torch.linspace(-1, 1, T).cuda()
    near, apart = ops.vocab_logprobs(h, w, y), ops.vocab_logprobs(far, w, y)
    for a, b in zip(near + ops.vocab_logprobs_backward(h, w, y, near[1], d), apart + ops.vocab_logprobs_backward(far, w, y, near[1], d)):
        assert_bitwise(a, b)


def test_c_abi_backward_limits():
    """The workspace function says which sizes the backward takes, and the backward agrees."""
    from vexact_amd import _lib

    lib, a = _lib.load(), 4096

    def bwd(T, V, H):  # a workspace that is too small is noticed after the sizes
        return lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, T, V, H, H, H, H, H, 1.0, a, 16, None)

    for T, V, H in ((262142, 8129, 64), (262142, 151936, 2048), (264000, 8128, 64), (4, 10, 262112), (33554303, 64, 8)):
        assert lib.vx_vocab_logprobs_bwd_workspace_bytes(T, V, H) > 0 and bwd(T, V, H) == -3, (T, V, H)
    for T, V, H in ((262143, 8129, 64), (262143, 151936, 2048), (4, 10, 262120), (33554304, 64, 8), (33554303, 64, 1 << 17), (1 << 40, 64, 8)):
        assert lib.vx_vocab_logprobs_bwd_workspace_bytes(T, V, H) == 0 and bwd(T, V, H) == -2, (T, V, H)


def test_c_abi_backward_grid_limit():
    """Four elements of d_hidden per thread, fewer than 2^32 threads in a launch."""
    from vexact_amd import _lib

    lib, a = _lib.load(), 4096
    for T, H, rc in ((262142, 65536, -3), (262142, 65544, -2), (100000, 1 << 17, -3), (100000, 200000, -2)):
        assert (lib.vx_vocab_logprobs_bwd_workspace_bytes(T, 9000, H) > 0) == (rc == -3), (T, H)
        assert lib.vx_vocab_logprobs_bwd(a, a, a, a, a, a, a, T, 9000, H, H, H, H, H, 1.0, a, 16, None) == rc, (T, H)


@gpu
def test_most_rows():
    """As many rows as the backward takes, offsets up to 2^32; one more is refused by the differentiable forward already."""
    T, V, H = 262142, 8200, 256
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn(T, H, generator=g, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(V, H, generator=g, device="cuda", dtype=torch.bfloat16) * 0.1
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    d = torch.randn(T, generator=g, device="cuda")
    out, lse = ops.vocab_logprobs(h, w, y)
    dh, dw = ops.vocab_logprobs_backward(h, w, y, lse, d)
    for a, b in ((0, 100), (131000, 131100), (T - 100, T)):
        few, lse_few = ops.vocab_logprobs(h[a:b], w, y[a:b])
        assert_bitwise(few, out[a:b])
        assert_bitwise(ops.vocab_logprobs_backward(h[a:b], w, y[a:b], lse_few, d[a:b], need_weight=False)[0], dh[a:b], f"d_hidden of {a}..{b}")
    for v in (0, 4097, 8191, V - 1):
        dx = -torch.exp(h.double() @ w[v].double() - lse.double()) * d.double() + torch.where(y == v, d.double(), 0.0)
        ref, mass = dx @ h.double(), dx.abs() @ h.double().abs()
        # a half step of each derivative and of the result; 8 sqrt(T) 2^-24 = 2^-12 of the mass for the fp32 sum and 2^-13
        # for the exponent's argument
        assert ((dw[v].double() - ref).abs() <= (2.0**-8 + 2.0**-11) * mass + 2.0**-8 * ref.abs()).all()
    h = torch.zeros(262143, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w, y = torch.zeros(8192, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(262143, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="for the backward"):
        logprobs_from_hidden(h, w, y)
    with torch.no_grad():  # the forward alone takes it
        assert ((logprobs_from_hidden(h, w, y) + torch.log(torch.tensor(8192.0))).abs() <= 2.0**-18).all()
    with pytest.raises(ValueError, match="for the backward"):
        ops.vocab_logprobs_backward(h, w, y, torch.zeros(262143, device="cuda"), torch.zeros(262143, device="cuda"))
