"""Decode attention over shared prefixes: the bits of the paged attention on the same block tables, and the value of a
plain implementation in 64 bits.

Tolerance against 64 bits: the probabilities are rounded to the element type (half a step h: 2^-8 bf16, 2^-11 fp16) in
the weighted sum and in its denominator, which moves an output by at most 2 h sum p |v| <= 2 h max |v|, the result by
another h of itself, and the scores' fp32 arithmetic by far less than h.
"""

import pytest
import torch

from vexact_amd import ops

from .util import assert_bitwise

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make(groups, prefixes, tails, heads, dims, page, dtype=torch.bfloat16, seed=0, head_major=False):
    """groups: sequences per group; prefixes: shared keys per group; tails: own keys per sequence (cycled)."""
    Hq, Hkv = heads
    Dk, Dv = dims
    g = torch.Generator().manual_seed(seed)
    B = sum(groups)
    lens, tables, nxt = [], [], 0
    for n, pre in zip(groups, prefixes):
        shared = list(range(nxt, nxt + pre // page))
        nxt += len(shared)
        for _ in range(n):
            length = pre + tails[len(lens) % len(tails)]
            own = -(-length // page) - len(shared) if length else 0
            tables.append((shared + list(range(nxt, nxt + own))) if length else [])
            nxt += max(own, 0)
            lens.append(length)
    width = max(1, max(len(t) for t in tables)) + 1
    perm = torch.randperm(max(nxt, 1), generator=g)
    table = torch.full((B, width), 1 << 30, dtype=torch.int32)  # entries that nothing may follow
    for i, t in enumerate(tables):
        table[i, : len(t)] = perm[torch.tensor(t, dtype=torch.long)].int() if t else table[i, :0]
    if head_major:
        k = torch.randn(max(nxt, 1), Hkv, page, Dk, generator=g).to(dtype).cuda().permute(0, 2, 1, 3)
        v = torch.randn(max(nxt, 1), Hkv, page, Dv, generator=g).to(dtype).cuda().permute(0, 2, 1, 3)
    else:
        k = torch.randn(max(nxt, 1), page, Hkv, Dk, generator=g).to(dtype).cuda()
        v = torch.randn(max(nxt, 1), page, Hkv, Dv, generator=g).to(dtype).cuda()
    q = torch.randn(B, Hq, Dk, generator=g).to(dtype).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    offs = [0]
    for n in groups:
        offs.append(offs[-1] + n)
    return dict(q=q, k_cache=k, v_cache=v, cu_seqlens_q=i32(list(range(B + 1))), seqused_k=i32(lens), page_table=table.cuda(),
                group_offsets=i32(offs), prefix_lens=i32([p // page * page for p in prefixes]), softmax_scale=Dk**-0.5)


def paged(a, **kw):
    names = ("q", "k_cache", "v_cache", "cu_seqlens_q", "seqused_k", "page_table", "softmax_scale")
    return ops.paged_attention(**{n: a[n] for n in names}, max_seqlen_q=1, **kw)


def plain(a):
    q, k, v = a["q"].cpu().double(), a["k_cache"].cpu().double(), a["v_cache"].cpu().double()
    page, Hkv = k.shape[1], k.shape[2]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[-1], dtype=torch.float64)
    for i, n in enumerate(a["seqused_k"].tolist()):
        if n == 0:
            continue
        at = torch.arange(n)
        block = a["page_table"][i].cpu()[at // page].long()
        ki, vi = k[block, at % page], v[block, at % page]
        for h in range(q.shape[1]):
            kh = h * Hkv // q.shape[1]
            out[i, h] = torch.softmax(ki[:, kh] @ q[i, h] * a["softmax_scale"], 0) @ vi[:, kh]
    return out


CASES = [  # groups, prefixes, tails, (Hq, Hkv), (Dk, Dv), page
    ([1], [0], [1], (1, 1), (128, 128), 16),
    ([2], [256], [1, 256], (8, 2), (128, 128), 16),
    ([8], [1000], [1, 17, 300, 40], (32, 4), (128, 128), 16),
    ([3, 1, 5, 2], [600, 700, 255, 2049], [1, 600, 33], (16, 2), (128, 128), 32),
    ([7], [1300], [5, 900], (10, 2), (64, 64), 16),  # five heads per kv head: rows of a sequence in two tiles
    ([20], [515], [1, 3], (3, 1), (128, 128), 16),
    ([5, 4], [800, 530], [9, 260], (32, 1), (128, 128), 64),  # two query tiles per sequence
    ([4], [777], [50, 4], (4, 4), (128, 128), 24),  # pages that are no power of two
    ([4, 3], [513, 300], [11], (8, 4), (80, 96), 16),  # padded head sizes
    ([3], [600], [20], (4, 2), (192, 128), 16),
    ([3], [600], [700], (4, 2), (256, 256), 16),
    ([2], [520], [3], (24, 1), (256, 256), 16),
    ([2, 3, 2, 2], [70, 130, 200, 63], [1, 60, 200], (8, 2), (128, 128), 16),  # less than a chunk shared, by whole blocks
    ([6, 2], [447, 448], [1, 65, 1000], (16, 4), (64, 64), 16),
    ([3], [600], [20, 1], (6, 2), (36, 20), 16),  # rows that 16-byte accesses cannot address
    ([2, 2], [300, 256], [1], (4, 2), (64, 64), 1),  # pages of one key
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups,prefixes,tails,heads,dims,page", CASES)
def test_bits_and_value(groups, prefixes, tails, heads, dims, page, dtype):
    a = make(groups, prefixes, tails, heads, dims, page, dtype, seed=sum(groups))
    out = ops.shared_prefix_attention(**a)
    assert_bitwise(out, paged(a, decode_kernel="split"), "paged attention")
    ref = plain(a)
    tol = HALF[dtype] * (2 * float(a["v_cache"].abs().max()) + ref.abs()) + 1e-6
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    bound = int(a["prefix_lens"].max())
    assert_bitwise(ops.shared_prefix_attention(**a, max_prefix_len=bound), out, "tight bound")
    assert_bitwise(ops.shared_prefix_attention(**a, max_prefix_len=bound // 2), out, "prefixes shared up to half")
    assert_bitwise(ops.shared_prefix_attention(**a, max_prefix_len=0), out, "nothing shared")


@gpu
def test_long_tails_and_many_groups():
    """Own chunks beyond one round of the workgroups that share them, and more groups than a wavefront has lanes."""
    a = make([2, 1], [300, 100], [9000, 70, 4000], (4, 1), (128, 128), 16, seed=8)
    assert_bitwise(ops.shared_prefix_attention(**a), paged(a, decode_kernel="split"))
    a = make([1 + i % 3 for i in range(150)], [256 + 16 * (i % 40) for i in range(150)], [3, 90], (4, 2), (64, 64), 16, seed=9)
    assert_bitwise(ops.shared_prefix_attention(**a), paged(a, decode_kernel="split"))
    a = make([130], [700], [3, 90], (2, 1), (128, 128), 16, seed=10)  # more sequences than lanes
    assert_bitwise(ops.shared_prefix_attention(**a), paged(a, decode_kernel="split"))


@gpu
def test_pages_beyond_four_gib():
    """Cache offsets past 32 bits: only the last pages of a 4.6 GB cache are in use."""
    a = make([3, 2], [700, 300], [5, 270], (8, 2), (128, 128), 16, seed=11)
    n = a["k_cache"].shape[0]
    blocks = (1 << 32) // (16 * 2 * 128 * 2) + 2 * n
    for name in ("k_cache", "v_cache"):
        big = torch.empty(blocks, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
        big[-n:] = a[name]
        a[name] = big
    used = a["page_table"] < (1 << 30)
    a["page_table"][used] += blocks - n
    assert_bitwise(ops.shared_prefix_attention(**a), paged(a, decode_kernel="split"))


@gpu
def test_rows_of_a_page_far_apart():
    """A cache whose outermost dimension is the place in a page: neighbouring keys lie 290 MB apart, a page spans 4.6 GB."""
    a = make([5], [1040], [40, 3], (8, 2), (128, 128), 16, seed=10)
    want = paged(a, decode_kernel="split")
    n = a["k_cache"].shape[0]
    for name in ("k_cache", "v_cache"):
        far = torch.empty(16, 570000, 2, 128, dtype=torch.bfloat16, device="cuda").permute(1, 0, 2, 3)
        far[:n] = a[name]
        a[name] = far
    assert 15 * 2 * a["k_cache"].stride(1) > 1 << 32
    assert_bitwise(ops.shared_prefix_attention(**a), want)


@gpu
def test_no_groups_and_a_given_workspace():
    a = make([2, 1], [300, 0], [40, 3, 700], (8, 2), (128, 128), 16, seed=11)
    a["group_offsets"], a["prefix_lens"] = a["group_offsets"][:1].contiguous(), a["prefix_lens"][:0]
    want = paged(a, decode_kernel="split")
    assert_bitwise(ops.shared_prefix_attention(**a), want)
    for n in (1 << 22, 16):  # enough, and too small: then it is not used
        ws = torch.full((n,), float("nan"), device="cuda")
        assert_bitwise(ops.shared_prefix_attention(**a, workspace=ws), want)
        assert torch.isnan(ws).all() == (n == 16)
    for ws in (torch.empty(1 << 22), torch.empty(1 << 22, 2, device="cuda")[:, 0]):
        with pytest.raises(ValueError, match="workspace must be"):
            ops.shared_prefix_attention(**a, workspace=ws)


@gpu
def test_the_first_columns_of_a_wide_table():
    """A view of the columns that are in use gives the same bits, and asks for a workspace of its own width."""
    a = make([4, 3], [600, 300], [40, 7, 300], (8, 2), (128, 128), 16, seed=15)
    want, width = paged(a, decode_kernel="split"), a["page_table"].shape[1]
    wide = torch.full((7, 8192), 1 << 30, dtype=torch.int32).cuda()
    wide[:, :width] = a["page_table"]
    assert_bitwise(ops.shared_prefix_attention(**{**a, "page_table": wide}, max_prefix_len=600), want)
    a["page_table"] = wide[:, :width]
    assert not a["page_table"].is_contiguous()
    ws = torch.zeros(4 << 20, dtype=torch.uint8, device="cuda")
    assert_bitwise(ops.shared_prefix_attention(**a, max_prefix_len=600, workspace=ws), want)
    assert ws.any()


@gpu
def test_a_full_decode_batch():
    a = make([16] * 16, [1024 + 96 * i for i in range(16)], list(range(1, 600, 37)), (32, 4), (128, 128), 16, seed=3, head_major=True)
    assert_bitwise(ops.shared_prefix_attention(**a), paged(a))


@gpu
def test_padded_batches():
    """Slots without a query token or without keys, sequences outside every group, rows behind the last sequence."""
    a = make([4, 3, 2], [600, 300, 520], [40, 7, 300], (8, 2), (128, 128), 16, seed=4)
    B = a["q"].shape[0]
    a["q"] = torch.cat([a["q"], torch.randn(3, 8, 128).to(torch.bfloat16).cuda()])
    a["group_offsets"] = a["group_offsets"][:3].contiguous()  # the last two sequences belong to no group
    a["prefix_lens"] = a["prefix_lens"][:2].contiguous()
    used = a["seqused_k"].clone()
    used[0] = 0  # the first sequence of a group is an empty slot: its block table must not be followed
    a["seqused_k"] = used
    a["page_table"][0] = 1 << 30
    cu = list(range(B + 1))
    for i in range(6, B + 1):
        cu[i] -= 1  # sequence 5 has no query token
    a["cu_seqlens_q"] = torch.tensor(cu, dtype=torch.int32).cuda()
    sentinel = torch.full((B + 3, 8, 128), 7.0, dtype=torch.bfloat16).cuda()
    out = ops.shared_prefix_attention(**a, out=sentinel.clone())
    want = paged(a, decode_kernel="split", out=sentinel.clone())
    want[0] = 0
    assert_bitwise(out, want)
    assert (out[B - 1 :] == 7).all() and (out[0] == 0).all()
    # a prefix length beyond every sequence is cut to the keys that exist
    a["prefix_lens"] = torch.tensor([1 << 20, 1 << 20], dtype=torch.int32).cuda()
    b = make([4], [600], [0, 0, 0, 0], (8, 2), (128, 128), 16, seed=5)
    b["prefix_lens"] = torch.tensor([1 << 20], dtype=torch.int32).cuda()
    b["page_table"][:] = b["page_table"][:1]  # one document, four questions: every page shared
    assert_bitwise(ops.shared_prefix_attention(**b), paged(b, decode_kernel="split"))


@gpu
@pytest.mark.parametrize("heads,dims,page", [((8, 2), (128, 128), 16), ((6, 2), (64, 64), 16), ((4, 4), (80, 80), 24)])
def test_an_ended_sequence_inside_a_group(heads, dims, page):
    """A slot without a query token keeps the length of the sequence that ended in it, the longest of its group, and a block
    table whose (valid) pages hold other keys by now. The others' prefix is read from one of their own tables, and is
    shared no further than one of them reaches."""
    a = make([4, 3], [960, 960], [120, 300, 40], heads, dims, page, seed=13)
    table, used = a["page_table"].clone(), a["seqused_k"].clone()
    pages = torch.arange(a["k_cache"].shape[0] - 1, -1, -1, dtype=torch.int32).cuda()
    gone = (1, 4)
    for s in gone:
        n = int((table[s] < (1 << 30)).sum())
        assert not torch.equal(table[s, :n], pages[:n])
        table[s, :n] = pages[:n]
        used[s] = n * page
    used[5], used[6] = 700, 530  # of the second group nobody else reaches the prefix's end
    assert int(used[:4].argmax()) == 1 and int(used[4:].argmax()) == 0
    cu = [0]
    for s in range(7):
        cu.append(cu[-1] + (s not in gone))
    a.update(page_table=table, seqused_k=used, cu_seqlens_q=torch.tensor(cu, dtype=torch.int32).cuda(), q=a["q"][: cu[-1]].contiguous())
    out = ops.shared_prefix_attention(**a)
    assert_bitwise(out, paged(a, decode_kernel="split"))


@gpu
@pytest.mark.parametrize("heads,dims,page", [((8, 2), (128, 128), 16), ((6, 2), (64, 64), 16), ((4, 4), (80, 80), 24)])
def test_what_lies_behind_a_short_sequence_inside_the_prefix(heads, dims, page):
    """Sequences that end inside their group's prefix read nothing of the keys behind their end, which for them may hold
    anything, though others of the group do: infinite keys, NaN and infinite values."""
    a = make([3, 2], [960, 960], [120], heads, dims, page, seed=9)
    lens = [1080, 300, 256, 1080, 1]
    a["seqused_k"] = torch.tensor(lens, dtype=torch.int32).cuda()
    table = a["page_table"].cpu()
    for seq, key, kv, value in ((0, 300, "k_cache", float("inf")), (0, 305, "v_cache", float("nan")), (3, 2, "v_cache", float("inf")),
                                (3, 200, "v_cache", float("nan"))):
        a[kv][int(table[seq, key // page]), key % page] = value
    out, want = ops.shared_prefix_attention(**a), paged(a, decode_kernel="split")
    for i in (1, 2, 4):
        assert torch.isfinite(want[i]).all()
        assert_bitwise(out[i], want[i])
    for i in (0, 3):
        assert torch.isnan(out[i]).all() and torch.isnan(want[i]).all()


@gpu
def test_extreme_scores_and_strides():
    a = make([6], [1040], [30, 1], (8, 2), (128, 128), 16, seed=6)
    a["q"] = torch.cat([a["q"], a["q"]], dim=1)[:, :8]  # token stride of 16 heads
    a["q"][0] *= 300
    a["k_cache"][:, :, 0] *= 20
    out = torch.zeros(6, 10, 128, dtype=torch.bfloat16).cuda()
    got = ops.shared_prefix_attention(**a, out=out[:, 1:9])
    assert_bitwise(got.contiguous(), paged(a, decode_kernel="split"))
    assert not out[:, 0].any() and not out[:, 9].any() and torch.isfinite(out).all()


@gpu
def test_other_stream_and_replayed_capture():
    a = make([8, 8], [1100, 640], [50, 300, 7], (32, 4), (128, 128), 16, seed=7)
    want = paged(a)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = ops.shared_prefix_attention(**a, max_prefix_len=1100)
    s.synchronize()
    assert_bitwise(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.shared_prefix_attention(**a, max_prefix_len=1100)
    for step in range(3):  # the sequences grow by a token, the groups' prefixes shrink
        a["seqused_k"] -= 1
        a["q"].copy_(torch.randn(a["q"].shape, generator=torch.Generator().manual_seed(step)).to(torch.bfloat16))
        a["prefix_lens"] -= 128 * step
        eager = paged(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert_bitwise(out, eager, f"replay {step}")


@gpu
def test_attention_wrapper_with_prefix_groups():
    """Through the interface a model calls: a step with prefix groups in the context gives the bits of one without."""
    from types import SimpleNamespace

    from vexact_amd.batch_invariant_ops import flash_attention_forward
    from vexact_amd.batch_invariant_ops.kv_cache_context import PrefixGroups, clear_kv_cache_context, set_kv_cache_context

    a = make([5, 2], [600, 300], [40, 7, 300], (8, 2), (128, 128), 16, seed=12)
    B = a["q"].shape[0]
    a["page_table"][a["page_table"] == 1 << 30] = -1  # padded as the step metadata pads it
    q = a["q"].transpose(0, 1).unsqueeze(0)  # [1, heads, tokens, dim]
    new = torch.randn(1, 2, B, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    last = (a["seqused_k"] - 1).long()
    slots = (a["page_table"].gather(1, (last // 16)[:, None])[:, 0] * 16 + last % 16).int()
    outs = []
    for groups in (None, PrefixGroups(a["group_offsets"], a["prefix_lens"], 600)):
        set_kv_cache_context(is_paged_attn=True, key_cache={0: a["k_cache"]}, value_cache={0: a["v_cache"]}, block_tables=a["page_table"],
                             context_lens=a["seqused_k"], slot_mapping=slots, query_start_loc=a["cu_seqlens_q"], max_seqlen_q=1, prefix_groups=groups)
        try:
            with torch.no_grad():
                outs.append(flash_attention_forward(SimpleNamespace(layer_idx=0), q, new, new, None, 128**-0.5)[0])
        finally:
            clear_kv_cache_context()
    assert outs[0].shape == (B, 8, 128)
    assert_bitwise(outs[1], outs[0])


@gpu
@pytest.mark.parametrize("form", ["fp32", "strided metadata", "default scale", "tensor scale", "under autograd"])
def test_prefix_groups_refuse_nothing_that_runs_without_them(form):
    """A context with prefix groups gives what the same context without them gives: the same bits, or the same error."""
    from types import SimpleNamespace

    from vexact_amd.batch_invariant_ops import flash_attention_forward
    from vexact_amd.batch_invariant_ops.kv_cache_context import PrefixGroups, clear_kv_cache_context, set_kv_cache_context

    a = make([3, 2], [300, 600], [40, 7], (8, 2), (64, 64), 16, seed=14)
    table, used, cu = a["page_table"], a["seqused_k"], a["cu_seqlens_q"]
    q, k, v, scale = a["q"], a["k_cache"], a["v_cache"], 0.1
    if form == "fp32":
        q, k, v = q.float(), k.float(), v.float()
    elif form == "strided metadata":
        used, cu = torch.stack([used, used], 1)[:, 0], torch.stack([cu, cu], 1)[:, 1]
        table = table.t().contiguous().t()
        assert table.stride(-1) != 1 and used.stride(0) == cu.stride(0) == 2
    elif form != "under autograd":
        scale = None if form == "default scale" else torch.tensor(0.1)
    results = []
    for groups in (None, PrefixGroups(a["group_offsets"], a["prefix_lens"], 600)):
        set_kv_cache_context(is_paged_attn=True, key_cache={0: k}, value_cache={0: v}, block_tables=table, context_lens=used,
                             slot_mapping=None, query_start_loc=cu, max_seqlen_q=1, prefix_groups=groups)
        try:
            with torch.set_grad_enabled(form == "under autograd"):
                results.append(flash_attention_forward(SimpleNamespace(layer_idx=0), q.transpose(0, 1).unsqueeze(0), None, None, None, scale)[0])
        except ValueError as e:
            results.append(str(e))
        finally:
            clear_kv_cache_context()
    if form == "tensor scale":
        assert results[0] == results[1] and "softmax_scale" in results[0]
    else:
        assert_bitwise(results[1], results[0])


@gpu
def test_prefix_groups_with_buffers_of_more_rows_than_sequences():
    """Block tables and query offsets longer than the step has sequences, and a value cache of more pages, as without groups."""
    from types import SimpleNamespace

    from vexact_amd.batch_invariant_ops import flash_attention_forward
    from vexact_amd.batch_invariant_ops.kv_cache_context import PrefixGroups, clear_kv_cache_context, set_kv_cache_context

    a = make([3, 2], [300, 600], [40, 7], (8, 2), (64, 64), 16, seed=16)
    table = torch.cat([a["page_table"], torch.full_like(a["page_table"], -1)])
    cu = torch.cat([a["cu_seqlens_q"], a["cu_seqlens_q"][-1:].expand(6)])
    for v in (a["v_cache"], torch.cat([a["v_cache"], a["v_cache"]])):
        outs = []
        for groups in (None, PrefixGroups(a["group_offsets"], a["prefix_lens"], 600)):
            set_kv_cache_context(is_paged_attn=True, key_cache={0: a["k_cache"]}, value_cache={0: v}, block_tables=table,
                                 context_lens=a["seqused_k"], slot_mapping=None, query_start_loc=cu, max_seqlen_q=1, prefix_groups=groups)
            try:
                with torch.no_grad():
                    outs.append(flash_attention_forward(SimpleNamespace(layer_idx=0), a["q"].transpose(0, 1).unsqueeze(0), None, None, None, 0.1)[0])
            finally:
                clear_kv_cache_context()
        assert_bitwise(outs[1], outs[0])


def test_refusals():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.shared_prefix_attention(z(1, 1, 8), z(1, 1, 1, 8), z(1, 1, 1, 8), z(2), z(1), z(1, 1), z(2), z(1), 1.0)


@gpu
def test_refusals_on_the_gpu():
    a = make([2], [300], [5], (4, 2), (64, 64), 16)
    for change, what in (
        ({"q": a["q"].float()}, "one dtype"), ({"group_offsets": a["group_offsets"][:1]}, "groups need"), ({"seqused_k": a["seqused_k"].long()}, "int32"),
        ({"page_table": a["page_table"][:1]}, "groups need"), ({"prefix_lens": a["prefix_lens"].cpu()}, "int32 tensor on"),
        ({"q": a["q"][:, :3]}, "does not fit"), ({"q": a["q"][..., :32]}, "does not fit"),
        ({"max_prefix_len": -1}, "negative"), ({"out": torch.zeros(1, 4, 64, dtype=torch.bfloat16).cuda()}, "out must be"),
        ({"q": a["q"][:, :, ::2].repeat(1, 1, 2)[:, :, ::1].transpose(1, 2).contiguous().transpose(1, 2)}, "contiguous in the head"),
    ):
        with pytest.raises(ValueError, match=what):
            ops.shared_prefix_attention(**{**a, **change})
    f = {n: t.float() if t.is_floating_point() else t for n, t in a.items() if torch.is_tensor(t)}
    with pytest.raises(ValueError, match="bfloat16 and float16"):
        ops.shared_prefix_attention(**f, softmax_scale=1.0)


def test_c_abi_refusals():
    from vexact_amd import _lib

    lib, p = _lib.load(), 4096

    def call(**kw):
        v = dict(q=p, k=p, v=p, o=p, cu=p, used=p, bt=p, go=p, pl=p, B=4, G=2, Hq=8, Hkv=2, Dk=128, Dv=128, pages=64, page=16, maxp=512, dt=0, ws=p, n=1 << 30)
        v.update(kw)
        return lib.vx_shared_prefix_attention(
            v["q"], v["k"], v["v"], v["o"], v["cu"], v["used"], v["bt"], v["go"], v["pl"], v["B"], v["G"], v["Hq"], v["Hkv"], v["Dk"], v["Dv"],
            1024, 128, 4096, 256, 128, 4096, 256, 128, 1024, 128, v["pages"], v["pages"], v["page"], 1.0, v["maxp"], v["dt"], v["ws"], v["n"], None)

    assert call(B=0) == 0
    for bad in (dict(q=None), dict(k=None), dict(o=None), dict(cu=None), dict(used=None), dict(bt=None), dict(go=None), dict(pl=None), dict(B=-1),
                dict(G=-1), dict(Hq=7), dict(Dk=0), dict(page=0), dict(pages=0), dict(maxp=-1), dict(q=p + 1)):
        assert call(**bad) == -1, bad
    for bad in (dict(dt=2), dict(Dk=257), dict(Dv=300), dict(Hq=66, Hkv=2), dict(B=70000), dict(G=1 << 28)):
        assert call(**bad) == -2, bad
    for bad in (dict(ws=None), dict(n=1000), dict(ws=p + 8)):
        assert call(**bad) == -3, bad
    # 4 sequences x 4 heads / 16 + 2 groups = 3 tiles x 2 kv heads x 2 chunks of 16 rows, and 4 x 2 x 3 own chunks of 4 rows
    assert lib.vx_shared_prefix_workspace_bytes(4, 2, 8, 2, 128, 512, 700) == (3 * 2 * 2 * 16 + 4 * 2 * 3 * 4) * 130 * 4
    assert lib.vx_shared_prefix_workspace_bytes(4, 2, 8, 2, 128, 255, 256) == 4 * 2 * 4 * 130 * 4
    assert lib.vx_shared_prefix_workspace_bytes(4, 2, 3, 1, 1, 0, 1) == 4 * 20 * 4  # rounded up to 16 bytes


def test_c_abi_refuses_sizes_whose_products_wrap():
    """Counts whose product passes 64 bits (to 0, or below it) are refused like those of a smaller product."""
    from vexact_amd import _lib

    lib, p = _lib.load(), 4096

    def call(G, H, pages, B=1):
        return lib.vx_shared_prefix_attention(p, p, p, p, p, p, p, p, p, B, G, H, H, 128, 256, 1024, 128, 4096, 256, 128, 4096, 256, 128,
                                              1024, 128, pages, pages, 16, 1.0, 1 << 62, 0, p + 8, 1 << 62, None)

    assert call(2, 8, 64) == -3  # supported: the workspace is refused, for its alignment
    for G, H, pages, B in ((1 << 30, 1 << 15, (1 << 27) - 128, 1), ((1 << 31) - 1, 65535, (1 << 27) - 17, 1), (1 << 62, 8, 64, 1), (0, 32767, (1 << 27) - 17, 65535),
                           (2, 8, 1 << 60, 1), (2, 8, (1 << 60) + 4, 1)):
        assert call(G, H, pages, B) == -2, (G, H, pages, B)
        assert lib.vx_shared_prefix_workspace_bytes(B, G, H, H, 256, min(pages, 1 << 59) * 16, min(pages, 1 << 59) * 16) == 0
