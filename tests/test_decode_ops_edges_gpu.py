"""The decode-step operators at the edges of what their callers may do: hidden
pages that hold anything, wide tables, rows of a page with gaps, plans in
place, captured calls, and the sizes at which a launch takes another form."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import decode_kernel as dk
from decode_kernel import capi
from test_decode_ops_gpu import (CODES, HALF, attention_case, check_append, check_attention, encode, gen, ints, plan_reference, random_pools, raw,
                                 run_attention, slots_of)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Plan
# ---------------------------------------------------------------------------


def test_plan_with_drafts_taken_back_loses_no_page():
    """Steps of five tokens of which some are taken back: the pages that a lower length leaves go to the ring's end."""
    requests, bs, width, blocks = 40, 16, 12, 300
    g = gen(1)
    held = torch.zeros(requests, dtype=torch.int32, device="cuda")
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(blocks, dtype=torch.int32, device="cuda")
    ring = ints([0, blocks, 0, 0], torch.int64)
    column = torch.arange(width, device="cuda")
    most = 0
    for step in range(60):
        fresh = torch.full((requests,), 5, dtype=torch.int32)
        fresh[torch.rand(requests, generator=g) < 0.03] = -1
        plan = dk.cache_plan(held, fresh.cuda(), table, free, ring, bs, 5 * requests)
        held, ring = plan.lengths, plan.ring
        assert ring[2:].tolist() == [0, 0]
        # Up to 21 tokens back, past a page's border now and then.
        back = torch.where(torch.rand(requests, generator=g) < 0.1, 21, torch.randint(0, 5, (requests,), generator=g)).int().cuda()
        kept = (held - back).clamp(min=0).clamp(max=width * bs - 10)
        left = table[(column >= -(-kept // bs)[:, None]) & (column < -(-held // bs)[:, None])]
        free[(ring[1] + torch.arange(len(left), device="cuda")) % len(free)] = left
        ring[1] += len(left)
        most = max(most, len(left))
        held = kept
        mine = table[column < -(-held // bs)[:, None]].tolist()
        head, tail = ring[:2].tolist()
        spare = free[torch.arange(head, tail, device="cuda") % blocks].tolist()
        assert sorted(mine + spare) == list(range(blocks)), step
    assert most > 0 and held.max() > 4 * bs


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("requests,bs,longest,new", [(300, 16, 900, 1300), (2048, 48, 200, 400)])
def test_plan_of_many_slots(requests, bs, longest, new, inplace):
    """Hundreds of thousands of slots, which threads take eight at a time; empty, ended, refused and too wide requests among them."""
    g = gen(requests)
    held = torch.randint(0, longest, (requests,), generator=g).tolist()
    fresh = torch.randint(0, new, (requests,), generator=g).tolist()
    width = -(-(longest + new) // bs) + 1
    for r in range(0, requests, 7):
        fresh[r] = (0, -1, 1, width * bs + 5)[r // 7 % 4]
    need = sum(-(-(h + max(n, 0)) // bs) - -(-h // bs) for h, n in zip(held, fresh) if h + max(n, 0) <= width * bs)
    order = torch.randperm(2 * requests * width + need + 64, generator=g)
    table, free = order[:requests * width].view(requests, width).tolist(), order[requests * width:].tolist()
    ring = [len(free) - 50, len(free) - 50 + need - 40, 0, 0]  # wraps, and the last requests find too few pages
    total = sum(max(n, 0) for n in fresh)
    assert total > 160000
    for tokens in (total, total + 13, total - 3):
        want = plan_reference(held, fresh, table, free, ring, bs, tokens)
        assert want[3][2] > 0 and want[3][3] > 0
        dt, df, dr, dh = ints(table), ints(free), ints(ring, torch.int64), ints(held)
        out = dk.CachePlan(dh, torch.empty(requests + 1, dtype=torch.int32, device="cuda"), torch.empty(tokens, dtype=torch.int64, device="cuda"), dr)
        p = dk.cache_plan(dh, ints(fresh), dt, df, dr, bs, tokens, out=out if inplace else None)
        got = [p.lengths.tolist(), p.starts.tolist(), p.slots.tolist(), p.ring.tolist(), dt.tolist(), df.tolist()]
        for name, a, b in zip(("lengths", "starts", "slots", "ring", "table", "free"), got, want):
            assert a == b, name


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kv,dim,bs,fresh", [
    (2, 64, 16, None), (2, 64, 48, None), (2, 64, 16, [3, 1, 9, 2]), (1, 64, 16, [20, 1, 30, 2]), (2, 128, 16, None), (1, 256, 48, [3, 1, 9, 2]),
])
def test_attention_ignores_hidden_pages_scales(code, kv, dim, bs, fresh):
    """Pages that lie wholly before a request's window may hold anything, their scales too."""
    lengths, window = [100, 70, 500, 49], 50
    case = attention_case(lengths, fresh, 4 * kv, kv, dim, bs, code, "fp16", seed=dim + bs)
    q, k, v, ks, vs, table, lengths, starts = case
    clean = run_attention(case, window=window)
    kb, vb, ks, vs = k.clone().view(torch.uint8), v.clone().view(torch.uint8), ks.clone(), vs.clone()
    hidden = 0
    for r, n in enumerate(lengths):
        low = n - (fresh[r] if fresh else 1) + 1 - window  # the first token that the first query sees
        for page in table[r, :max(0, low) // bs].tolist():
            kb[page] = vb[page] = 0x7F  # NaN in e4m3
            ks[page] = vs[page] = float("nan")
            hidden += 1
    assert hidden
    dirty = run_attention((q, kb.view(k.dtype), vb.view(v.dtype), ks, vs, table, lengths, starts), window=window)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("hq,kv,dim", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("window", [0, 2, 2 ** 31 - 100, 2 ** 31 - 1])
def test_attention_of_more_queries_than_tokens_and_the_largest_windows(hq, kv, dim, window):
    """Queries that stand before a request's first token see none; a window of any size hides no more than it says."""
    check_attention(attention_case([2, 40, 3, 0, 0, 70], [5, 3, 9, 2, 3, 1], hq, kv, dim, 16, "int8", "fp16", seed=dim), window=window)


@pytest.mark.parametrize("hq,kv,dim,window", [(8, 2, 128, 0), (4, 4, 64, 30), (16, 1, 128, 0)])
def test_attention_of_fewer_rows_than_starts(hq, kv, dim, window):
    """Rows that q lacks are left out; the others keep their places before the request's last token."""
    for lengths, fresh, rows in (([130], [100], 97), ([130, 60], [100, 20], 60), ([9, 130, 60], [1, 100, 20], 104)):
        case = attention_case(lengths, fresh, hq, kv, dim, 16, "int8", "fp16", seed=rows)
        whole, lse = run_attention(case, window=window)
        some, some_lse = run_attention((case[0][:rows].contiguous(), *case[1:]), window=window)
        # Another split of the same sums: fp16 weights and outputs.
        torch.testing.assert_close(some, whole[:rows], rtol=2.0 ** -9, atol=2.0 ** -9 * float(whole.abs().max()))
        torch.testing.assert_close(some_lse, lse[:rows], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dim,fresh", [(128, None), (64, None), (128, 5), (256, None)])
def test_attention_of_many_small_weights_behind_a_large_one(dim, fresh):
    """The first token has all the weight and no V; what the others leave, each 2^-25.3 of it, is the output."""
    requests, kv, n = 300, 8, 1024  # more segments than warps: one warp adds up a whole one
    k = torch.zeros(n // 64, kv, 64, dim, dtype=torch.int8)
    v = torch.full_like(k, 100)
    k[0, :, 0, 0], v[0, :, 0] = 127, 0
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), *(torch.ones(n // 64, kv, device="cuda") for _ in range(2)))
    each = fresh or 1
    q = torch.zeros(requests * each, kv, dim, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1
    starts = ints([each * r for r in range(requests + 1)]) if fresh else None
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda").expand(requests, -1).contiguous()
    out = dk.cache_attention(q, cache, table, ints([n] * requests), starts, scale=25.3 * math.log(2) / 127).double().cpu()
    others = torch.arange(n - each, n, dtype=torch.float64).repeat(requests) * 2.0 ** -25.3
    want = (100 * others / (1 + others))[:, None, None]
    # A weight is 2^-18.3 of fp16's 1 and rounded to a multiple of 2^-24; the score's and the output's own rounding.
    assert ((out - want).abs() <= (2.0 ** -6.7 + 2.0 ** -10) * want).all()


@pytest.mark.parametrize("dim,hq,kv,fresh", [(64, 8, 2, None), (128, 8, 2, None), (128, 8, 2, [3, 1, 9]), (256, 4, 2, None)])
def test_attention_of_queries_with_one_large_channel(dim, hq, kv, fresh):
    """A channel of bf16 queries 2^22 times the others, in which the keys hold nothing: the others make the scores."""
    q, k, v, ks, vs, table, lengths, starts = attention_case([70, 130, 400], fresh, hq, kv, dim, 32, "int8", "bf16", seed=dim)
    q[..., 5] = 2.0 ** 22
    k[..., 5] = 0
    check_attention((q, k, v, ks, vs, table, lengths, starts))
    q[..., 5] = 0
    for size in (2.0 ** 123, 2.0 ** -120):  # near the ends of bf16's range
        check_attention((q * size, k, v, ks, vs, table, lengths, starts), scale=dim ** -0.5 / size)


def test_attention_over_a_wide_table():
    """A table for 131072 tokens and 16384 rows in q, of which short requests use a few."""
    lengths, fresh = [300, 290, 17, 1000], [256, 1, 17, 100]
    q, k, v, ks, vs, table, lengths, starts = attention_case(lengths, fresh, 64, 8, 128, 64, "int8", "bf16", seed=3)
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    wide = torch.full((4, 2048), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    many = torch.zeros(16384, 64, 128, dtype=torch.bfloat16, device="cuda")
    many[:starts[-1]] = q.cuda()
    want = dk.cache_attention(q.cuda(), cache, table.cuda(), ints(lengths), ints(starts))
    got = dk.cache_attention(many, cache, wide, ints(lengths), ints(starts))[:starts[-1]]
    torch.testing.assert_close(got.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -9 * float(want.abs().max()))


@pytest.mark.parametrize("fresh", [None, [3, 20]])
@pytest.mark.parametrize("dim,code,dtype", [(64, "e4m3", "fp16"), (128, "int8", "bf16")])
def test_attention_takes_kv_heads_in_several_launches(dim, code, dtype, fresh):
    """The widest table leaves a launch's line of units room for a few KV heads only."""
    case = attention_case([700, 33], fresh, 80, 40, dim, 256, code, dtype, seed=dim)
    q, k, v, ks, vs, table, lengths, starts = case
    wide = torch.full((2, (1 << 30) // 256), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    check_attention((q, k, v, ks, vs, wide, lengths, starts))


@pytest.mark.parametrize("dim,hq,kv,code,dtype", [(128, 8, 2, "int8", "bf16"), (64, 3, 3, "e4m3", "fp16"), (256, 4, 2, "int8", "fp16")])
def test_attention_of_prompts(dim, hq, kv, code, dtype):
    """A prompt of a thousand tokens, one behind kept tokens, and single tokens beside them."""
    lengths, fresh = [1000, 1, 900, 333, 77], [1000, 1, 300, 1, 1]
    for window in (0, 130):
        check_attention(attention_case(lengths, fresh, hq, kv, dim, 64, code, dtype, seed=window + dim), window=window)


def c_attention(q, cache, table, lengths, out, workspace):
    """dk_cache_attention of one query a request on the current stream."""
    k, v = cache.k, cache.v
    c = capi.Cache8(k=k.data_ptr(), v=v.data_ptr(), k_scale=cache.k_scale.data_ptr(), v_scale=cache.v_scale.data_ptr(), blocks=cache.blocks,
                    block_size=cache.block_size, kv_heads=cache.kv_heads, head_dim=cache.head_dim, code=capi.DK_INT8, k_block_stride=k.stride(0),
                    k_head_stride=k.stride(1), k_token_stride=k.stride(2), v_block_stride=v.stride(0), v_head_stride=v.stride(1), v_token_stride=v.stride(2))
    a = capi.CacheAttentionArgs(cache=c, q=q.data_ptr(), out=out.data_ptr(), lse=None, dtype=capi.DK_FP16, q_token_stride=q.stride(0),
                                q_head_stride=q.stride(1), block_table=table.data_ptr(), max_blocks=table.shape[1], table_stride=table.stride(0),
                                lengths=lengths.data_ptr(), starts=None, requests=len(lengths), tokens=len(q), q_heads=q.shape[1],
                                scale=q.shape[2] ** -0.5, causal=1, window=0)
    return capi.load().dk_cache_attention(ctypes.byref(a), workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dim,hq,kv", [(64, 8, 2), (128, 32, 8), (128, 32, 1), (256, 4, 2)])
def test_attention_workspace_needs_only_its_counters_zero(dim, hq, kv):
    # Long requests, so that warps and CTAs leave parts of segments in the workspace.
    q, k, v, ks, vs, table, lengths, _ = attention_case([9000, 40, 2500, 700], None, hq, kv, dim, 64, "int8", "fp16", seed=dim)
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    q, table, lengths = q.cuda(), table.cuda(), ints(lengths)
    want = dk.cache_attention(q, cache, table, lengths)
    workspace = torch.full((capi.load().dk_cache_attention_workspace_bytes(dim),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN
    counters = capi.load().dk_cache_attention_counter_bytes()
    assert 0 < counters <= 1 << 16
    workspace[:counters] = 0
    for _ in range(3):
        out = torch.full_like(want, float("nan"))
        assert c_attention(q, cache, table, lengths, out, workspace) == capi.DK_OK
        assert torch.equal(out, want)
        assert not workspace[:counters].any()


def test_attention_captured_zeroes_only_its_counters():
    runtime = pytest.importorskip("cuda.bindings.runtime")
    q, k, v, ks, vs, table, lengths, _ = attention_case([3000], None, 8, 2, 128, 64, "int8", "fp16")
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    args = (q.cuda(), cache, table.cuda(), ints(lengths))
    want = dk.cache_attention(*args)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        dk.cache_attention(*args, out=out)
    count = runtime.cudaGraphGetNodes(graph.raw_cuda_graph(), 0)[2]
    nodes = runtime.cudaGraphGetNodes(graph.raw_cuda_graph(), count)[1][:count]
    types = [runtime.cudaGraphNodeGetType(n)[1] for n in nodes]
    kind = runtime.cudaGraphNodeType
    assert sorted(types, key=int) == sorted([kind.cudaGraphNodeTypeKernel, kind.cudaGraphNodeTypeMemset], key=int)
    zeroed = runtime.cudaGraphMemsetNodeGetParams(nodes[types.index(kind.cudaGraphNodeTypeMemset)])[1]
    assert zeroed.width * zeroed.height * zeroed.elementSize == capi.load().dk_cache_attention_counter_bytes()
    graph.instantiate()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_attention_workspaces_are_shared_by_head_sizes_and_given_back():
    cases = []
    for dim, hq, kv in ((64, 8, 2), (256, 4, 2), (128, 32, 8)):
        q, k, v, ks, vs, table, lengths, _ = attention_case([5000, 40], None, hq, kv, dim, 64, "int8", "fp16", seed=dim)
        args = (q.cuda(), dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda()), table.cuda(), ints(lengths))
        cases.append((args, dk.cache_attention(*args)))
    torch.cuda.synchronize()
    dk.release_workspaces()
    most = capi.load().dk_cache_attention_workspace_bytes(128)
    assert most >= capi.load().dk_cache_attention_workspace_bytes(256)
    kept = torch.cuda.memory_allocated()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        with torch.cuda.stream(s):
            for args, want in cases * 2:
                assert torch.equal(dk.cache_attention(*args), want)
    torch.cuda.synchronize()
    assert 3 * most <= torch.cuda.memory_allocated() - kept < 3 * most + (8 << 20)
    # Given back between calls that are still on their way.
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            outs += [(dk.cache_attention(*args), want) for args, want in cases]
        dk.release_workspaces()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o, want in outs)
    del outs
    assert torch.cuda.memory_allocated() - kept < 4 << 20


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------


def pages_reference(pool, scale, x, slots, code):
    """dk_cache_append's rule in fp32 on the CPU, page by page: a page's tokens have one maximum and one scale."""
    bs, q = pool.shape[2], CODES[code][1]
    pool, scale, x = pool.clone(), scale.clone(), x.float()
    there = (slots >= 0) & (slots < pool.shape[0] * bs)
    for page in (slots[there] // bs).unique().tolist():
        mine = there & (slots // bs == page)
        rows, y = slots[mine] % bs, x[mine]
        amax = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y)).amax(dim=(0, 2))
        new = amax.clamp(min=2.0 ** -60) / torch.full_like(amax, q)
        first = int(rows.min())
        if first:
            old = scale[page].clone()
            new = torch.maximum(old, new)
            for h in (new > old).nonzero().flatten().tolist():
                pool[page, h, :first] = encode(pool[page, h, :first].float() * (old[h] / new[h]), code)
        scale[page] = new
        raw_pool = pool.view(torch.uint8)  # indexed writes of e4m3
        raw_pool[page][:, rows] = encode(y * (torch.ones_like(new) / new)[None, :, None], code).transpose(0, 1).contiguous().view(torch.uint8)
    return pool, scale


def check_pages(k, v, slots, pools, code):
    dev = [t.cuda() for t in pools]
    dk.cache_append(k.cuda(), v.cuda(), slots.cuda(), dk.PagedCache8.from_tensors(*dev))
    for i, x in ((0, k), (1, v)):
        want, scale = pages_reference(pools[i], pools[2 + i], x, slots, code)
        assert torch.equal(dev[2 + i].cpu(), scale), "scales"
        assert torch.equal(raw(dev[i].cpu()), raw(want)), "codes"


def rows_with_gaps(pages, bs, most, g, whole=0.2):
    """Slots of `pages` pages: in most pages some rows, rising; in a share of them neighbouring rows only."""
    out = []
    for page in torch.randperm(pages, generator=g).tolist():
        n = int(torch.randint(1, min(most, bs) + 1, (1,), generator=g))
        if torch.rand(1, generator=g) < whole:
            at = int(torch.randint(0, bs - n + 1, (1,), generator=g))
            rows = torch.arange(at, at + n)
        else:
            rows = torch.randperm(bs, generator=g)[:n].sort().values
        out.append(page * bs + rows)
        if torch.rand(1, generator=g) < 0.1:
            out.append(torch.tensor([-1]))
    return torch.cat(out)


@pytest.mark.parametrize("dtype,code", [("fp16", "int8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("dim,heads,bs,pages,most", [
    (128, 2, 16, 3, 3), (128, 8, 64, 9, 64), (64, 3, 48, 40, 48), (256, 2, 256, 3, 250), (64, 12, 16, 300, 9), (128, 8, 64, 150, 40),
])
def test_append_rows_with_gaps(dtype, code, dim, heads, bs, pages, most):
    """Rows of a page may rise with gaps: they are one run with one scale, whichever windows and warps they fall to."""
    g = gen(dim + pages)
    slots = rows_with_gaps(pages, bs, most, g)
    pools = random_pools(pages, heads, bs, dim, code, g)
    k, v = ((torch.randn(len(slots), heads, dim, generator=g) * torch.rand(len(slots), heads, 1, generator=g) * 5).to(HALF[dtype][0]) for _ in range(2))
    k[::7, :, 3] = float("inf")
    v[::5, :, 1] = float("nan")
    check_pages(k, v, slots, pools, code)


@pytest.mark.parametrize("dtype,code", [("fp16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("dim,heads,bs,tokens", [
    # Token-heads of K and V in the hundreds of thousands: a CTA takes two, then four heads' K or V, fewer in the last one.
    (64, 5, 48, 20000), (64, 5, 256, 40000), (128, 9, 64, 12000), (128, 7, 16, 30000), (256, 3, 256, 33000), (256, 3, 48, 65000),
    # Long runs in windows of 16 and of 64 tokens.
    (128, 8, 64, 1000), (64, 3, 256, 4000), (128, 8, 64, 2500), (256, 2, 48, 9000),
])
def test_append_in_wide_windows(dtype, code, dim, heads, bs, tokens):
    """Every form that the number of tokens and heads chooses, with pages begun before, short and long runs and values that are not finite."""
    g = gen(dim + tokens)
    held, new, left = [], [], tokens
    while left > 0:
        n = min(left, int(torch.randint(1, 7 * bs, (1,), generator=g)))
        held.append(int(torch.randint(0, 2 * bs, (1,), generator=g)))
        new.append(n)
        left -= n
    slots, pages = slots_of(held, new, bs, g)
    slots = torch.where(torch.rand(len(slots), generator=g) < 0.001, torch.where(slots % bs == 0, -1, slots), slots)  # rows that begin a page left out
    pools = random_pools(pages, heads, bs, dim, code, g)
    k, v = ((torch.randn(tokens, heads, dim, generator=g) * torch.rand(tokens, heads, 1, generator=g) * 5).to(HALF[dtype][0]) for _ in range(2))
    k[::501, :, 3], v[::701, 0, 7], v[::333, -1, 1] = float("inf"), float("-inf"), float("nan")
    check_append(k, v, slots, pools, code)
