"""The decode-step operators on the GPU against plain implementations in 64
bits (whole numbers: in integers): plan, append, attention and block norm, at
the sizes, masks, strides and values where they can go wrong."""

from __future__ import annotations

import math

import pytest
import torch

import decode_kernel as dk

pytestmark = pytest.mark.gpu

CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
HALF = {"fp16": (torch.float16, 2.0 ** -11), "bf16": (torch.bfloat16, 2.0 ** -8)}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


# ---------------------------------------------------------------------------
# Plan
# ---------------------------------------------------------------------------


def plan_reference(held, fresh, table, free, ring, bs, tokens):
    """The rule of dk_cache_plan, one request after the other."""
    table, free = [list(r) for r in table], list(free)
    cap, width = len(free), len(table[0]) if table else 1
    head, tail = ring[0], ring[1]
    asked = taken = missing = wide = 0
    lengths, starts, slots, back = [], [0], [], []
    for r, (c, n) in enumerate(zip(held, fresh)):
        c = max(c, 0)
        have = -(-c // bs)
        if n < 0:
            back += table[r][:min(have, width)]
            lengths.append(0)
            starts.append(starts[-1])
            continue
        starts.append(starts[-1] + n)
        want = -(-(c + n) // bs)
        ok = True
        if n and want > width:
            wide += 1
            ok = False
        elif n and want > have:
            asked += want - have
            if asked > tail - head:
                missing += want - have
                ok = False
            else:
                for j in range(want - have):
                    table[r][have + j] = free[(head + asked - (want - have) + j) % cap]
                taken = asked
        lengths.append(c + n if ok else c)
        slots += [table[r][(c + i) // bs] * bs + (c + i) % bs if ok else -1 for i in range(n)]
    for j, page in enumerate(back):
        free[(tail + j) % cap] = page
    slots = (slots + [-1] * tokens)[:tokens]
    return lengths, starts, slots, [head + taken, tail + len(back), missing, wide], table, free


def plan_case(requests, bs, seed, longest=200, width=None, spare=10, ended=0.2, head=5):
    g = gen(seed)
    held = torch.randint(0, longest, (requests,), generator=g)
    fresh = torch.randint(0, 40, (requests,), generator=g)
    fresh[torch.rand(requests, generator=g) < 0.3] = 1
    fresh[torch.rand(requests, generator=g) < ended] = -1
    held[torch.rand(requests, generator=g) < 0.1] = 0
    width = width or -(-(longest + 40) // bs) + 1
    need = int(sum(max(0, -(-(h + max(n, 0)) // bs) - -(-h // bs)) for h, n in zip(held.tolist(), fresh.tolist())))
    cap = requests * width + need + 64
    order = torch.randperm(cap + requests * width, generator=g)
    table = order[cap:].view(requests, width)
    return held.tolist(), fresh.tolist(), table.tolist(), order[:cap].tolist(), [head, head + need + spare, 0, 0]


def check_plan(held, fresh, table, free, ring, bs, tokens):
    want = plan_reference(held, fresh, table, free, ring, bs, tokens)
    dt = ints(table).view(len(held), -1)
    df, dr = ints(free), ints(ring, torch.int64)
    p = dk.cache_plan(ints(held), ints(fresh), dt, df, dr, bs, tokens)
    got = [p.lengths.tolist(), p.starts.tolist(), p.slots.tolist(), p.ring.tolist(), dt.tolist(), df.tolist()]
    for name, a, b in zip(("lengths", "starts", "slots", "ring", "table", "free"), got, want):
        assert a == b, name


@pytest.mark.parametrize("requests,bs", [(1, 16), (2, 256), (33, 16), (64, 48), (511, 64), (513, 16), (1500, 32), (8192, 16)])
def test_plan_matches_the_rule(requests, bs):
    held, fresh, table, free, ring = plan_case(requests, bs, seed=requests)
    total = sum(max(n, 0) for n in fresh)
    for tokens in {total, total + 13, max(0, total - 3)}:
        check_plan(held, fresh, table, free, ring, bs, tokens)


def test_plan_of_long_prompts_and_of_a_wrapped_ring():
    g = gen(3)
    held, fresh = [0, 5000, 17], [70001, 1, 0]
    bs, width = 16, 4400
    table = torch.randint(0, 10 ** 6, (3, width), generator=g).tolist()
    free = torch.randperm(9000, generator=g).tolist()
    check_plan(held, fresh, table, free, [8000 + 9000 * 10 ** 6, 8000 + 9000 * 10 ** 6 + 8990, 0, 0], bs, sum(fresh))


def test_plan_refuses_requests_that_do_not_fit():
    # The ring has pages for the first two requests only; a request that needs none is still served.
    check_plan([0, 0, 0, 8], [16, 20, 40, 3], [[90] * 4, [91] * 4, [92] * 4, [93] * 4], list(range(50, 60)), [0, 4, 0, 0], 16, 80)
    # Too wide for the table: refused, and its pages go to no one.
    check_plan([0, 60, 0], [100, 10, 16], [[90] * 4, [91] * 4, [92] * 4], list(range(50, 60)), [7, 15, 0, 0], 16, 130)
    check_plan([0], [1], [[9]], [4], [0, 0, 0, 0], 16, 1)


def test_plan_without_requests_or_tokens():
    p = dk.cache_plan(ints([]), ints([]), torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([1]), ints([0, 1, 0, 0], torch.int64), 16, 5)
    assert p.starts.tolist() == [0] and p.slots.tolist() == [-1] * 5 and p.ring.tolist() == [0, 1, 0, 0]
    check_plan([3, 5], [0, -1], [[1], [2]], [7, 8, 9], [1, 2, 0, 0], 16, 0)


def test_plan_in_place_over_steps_in_a_graph():
    bs, requests, width = 16, 700, 6
    held, ring = torch.zeros(requests, dtype=torch.int32, device="cuda"), ints([0, 4200, 0, 0], torch.int64)
    free = torch.arange(4200, dtype=torch.int32, device="cuda")
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    fresh = torch.ones(requests, dtype=torch.int32, device="cuda")
    out = dk.CachePlan(held, torch.empty(requests + 1, dtype=torch.int32, device="cuda"),
                       torch.empty(requests, dtype=torch.int64, device="cuda"), ring)
    step = lambda: dk.cache_plan(held, fresh, table, free, ring, bs, requests, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(40):
        graph.replay()
    assert held.tolist() == [41] * requests
    assert ring.tolist() == [3 * requests, 4200, 0, 0]
    pages = table[:, :3].flatten().tolist()
    assert sorted(pages) == list(range(3 * requests))
    assert out.slots.tolist() == [table[r, 2].item() * bs + 8 for r in range(requests)]
    fresh.fill_(-1)
    graph.replay()
    assert held.tolist() == [0] * requests and ring.tolist() == [3 * requests, 4200 + 3 * requests, 0, 0]


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------


def encode(x, code):
    dtype, q = CODES[code]
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-q, q)
    return (x.round() if code == "int8" else x).to(dtype)


def append_reference(pool, scale, x, slots, code):
    """dk_cache_append's rule in fp32 on the CPU, one run after the other."""
    bs, q = pool.shape[2], CODES[code][1]
    pool, scale, x = pool.clone(), scale.clone(), x.float()
    t = 0
    slots = slots.tolist()
    while t < len(slots):
        if slots[t] < 0 or slots[t] // bs >= pool.shape[0]:
            t += 1
            continue
        page, row, n = slots[t] // bs, slots[t] % bs, 1
        while t + n < len(slots) and row + n < bs and slots[t + n] == slots[t] + n:
            n += 1
        mine = x[t:t + n]
        amax = torch.where(mine.isfinite(), mine.abs(), torch.zeros_like(mine)).amax(dim=(0, 2))
        new = amax.clamp(min=2.0 ** -60) / torch.full_like(amax, q)
        if row:
            old = scale[page].clone()
            new = torch.maximum(old, new)
            for h in (new > old).nonzero().flatten().tolist():
                again = encode(pool[page, h, :row].float() * (old[h] / new[h]), code)
                pool[page, h, :row] = again
        scale[page] = new
        by = torch.ones_like(new) / new
        pool[page, :, row:row + n] = encode(mine * by[None, :, None], code).transpose(0, 1)
        t += n
    return pool, scale


def raw(x):
    return x.contiguous().view(torch.uint8)


def check_append(k, v, slots, pools, code, dk_args=None):
    """pools: (k, v, k_scale, v_scale) on the CPU.  Codes and scales agree to the bit."""
    dev = [x.cuda() for x in pools]
    cache = dk.PagedCache8.from_tensors(*dev)
    a, b, c = dk_args or (k.cuda(), v.cuda(), slots.cuda())
    dk.cache_append(a, b, c, cache)
    for i, x in ((0, k), (1, v)):
        want, scale = append_reference(pools[i], pools[2 + i], x, slots, code)
        assert torch.equal(dev[2 + i].cpu(), scale), "scales"
        assert torch.equal(raw(dev[i].cpu()), raw(want)), "codes"
    return cache


def random_pools(pages, heads, bs, dim, code, g):
    dtype, q = CODES[code]
    make = lambda: encode(torch.randn(pages, heads, bs, dim, generator=g) * q / 3.6, code)  # noqa: E731
    scale = lambda: torch.rand(pages, heads, generator=g) * 4 / q + 0.5 / q  # noqa: E731
    return make(), make(), scale(), scale()


def slots_of(held, new, bs, g, spare=3):
    total = sum(-(-(h + n) // bs) for h, n in zip(held, new))
    order = torch.randperm(total + spare, generator=g).tolist()
    out = []
    for h, n in zip(held, new):
        mine = [order.pop() for _ in range(-(-(h + n) // bs))]
        out += [mine[(h + i) // bs] * bs + (h + i) % bs for i in range(n)]
    return torch.tensor(out, dtype=torch.int64), total + spare


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,heads,bs,held,new", [
    (128, 8, 64, [0, 1, 63, 64, 100], [1, 1, 1, 1, 1]),
    (128, 2, 16, [0, 3, 15, 16], [1, 40, 2, 33]),
    (64, 3, 48, [47, 0, 5], [1, 97, 9]),
    (256, 1, 256, [0, 200, 255], [513, 30, 1]),
    (64, 12, 256, [0], [300]),
    (128, 1, 32, [7], [8]),
    (128, 1, 32, [7], [9]),
])
def test_append_matches_the_rule_to_the_bit(dtype, code, dim, heads, bs, held, new):
    g = gen(dim + bs + len(held))
    slots, pages = slots_of(held, new, bs, g)
    pools = random_pools(pages, heads, bs, dim, code, g)
    k = (torch.randn(len(slots), heads, dim, generator=g) * torch.rand(len(slots), heads, 1, generator=g) * 5).to(HALF[dtype][0])
    v = torch.randn(len(slots), heads, dim, generator=g).to(HALF[dtype][0])
    check_append(k, v, slots, pools, code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_many_tokens(code):
    # Enough tokens for the wide windows; runs that begin and end anywhere in them.
    g = gen(11)
    held, new = [int(x) for x in torch.randint(0, 90, (300,), generator=g)], [int(x) for x in torch.randint(1, 60, (300,), generator=g)]
    slots, pages = slots_of(held, new, 16, g)
    pools = random_pools(pages, 8, 16, 64, code, g)
    k, v = (torch.randn(len(slots), 8, 64, generator=g).half() for _ in range(2))
    check_append(k, v, slots, pools, code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_odd_values(code):
    g = gen(2)
    x = torch.randn(40, 2, 64, generator=g).half()
    x[0, 0, 3] = float("nan")
    x[1, 0, 5], x[1, 1, 6] = float("inf"), float("-inf")
    x[2] = 0
    x[20:36] = 0                      # a page of zeros
    x[36:38] = float("nan")           # a page of nothing finite
    x[39] = 2.0 ** -24                # the smallest fp16
    slots = torch.tensor(list(range(4, 16)) + list(range(32, 40)) + list(range(16, 32)) + [48, 49, 50, 64])
    pools = random_pools(6, 2, 16, 64, code, g)
    check_append(x, x.flip(2), slots, pools, code)


def test_append_skips_and_strides():
    g = gen(4)
    T, heads, dim, bs = 37, 4, 128, 32
    slots = torch.arange(T) + 5
    slots[26] = -7                          # the last row of a page and the first of the next: the rows of
    slots[27] = -1                          # a page stay neighbours
    slots[-1] = 10 ** 9                     # past the pool
    qkv = torch.randn(T, (8 + 2 * heads) * dim, generator=g).half()
    k, v = qkv[:, 8 * dim:12 * dim].view(T, heads, dim), qkv[:, 12 * dim:].view(T, heads, dim)
    pools = random_pools(3, heads, bs, dim, "int8", g)
    d = qkv.cuda()
    check_append(k, v, slots, pools, "int8", (d[:, 8 * dim:12 * dim].view(T, heads, dim), d[:, 12 * dim:].view(T, heads, dim), slots.cuda()))
    # A view that the kernel's loads cannot take (odd offset) and one that is transposed.
    flat = torch.randn(T * heads * dim + 1, generator=g).half()
    k2 = flat[1:].view(T, heads, dim)
    v2 = torch.randn(heads, T, dim, generator=g).half()
    check_append(k2, v2.transpose(0, 1), slots, pools, "int8", (flat.cuda()[1:].view(T, heads, dim), v2.cuda().transpose(0, 1), slots.cuda()))
    # Pools laid out [blocks, block_size, heads, dim] and scaled like the others.
    dev = [pools[0].transpose(1, 2).contiguous().cuda().transpose(1, 2), pools[1].cuda(), pools[2].cuda(), pools[3].cuda()]
    dk.cache_append(k.cuda(), v.cuda(), slots.cuda(), dk.PagedCache8.from_tensors(*dev))
    want, scale = append_reference(pools[0], pools[2], k, slots, "int8")
    assert torch.equal(dev[0].cpu(), want) and torch.equal(dev[2].cpu(), scale)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_token_by_token_stays_near_the_values(code):
    # Each growth of the scale rounds a code once more: by half a code of the
    # scale of that time (int8), or by 2^-4 of itself (e4m3), so a value is off
    # by no more than half the last scale for each growth, or that share of itself.
    g = gen(9)
    bs, heads, dim = 64, 2, 128
    x = torch.randn(bs, heads, dim, generator=g).half() * torch.linspace(0.2, 3, bs)[:, None, None].half()
    cache = dk.PagedCache8(2, bs, heads, dim, dtype=CODES[code][0])
    growths = torch.zeros(heads)
    last = None
    for t in range(bs):
        dk.cache_append(x[t:t + 1].cuda(), x[t:t + 1].cuda(), ints([bs + t], torch.int64), cache)
        now = cache.k_scale[1].cpu()
        growths += (last is None) | (now > (last if last is not None else now))
        last = now
    got = cache.k[1].float().cpu() * cache.k_scale[1].cpu()[:, None, None]
    want = x.float().transpose(0, 1)
    if code == "int8":
        bound = 0.5 * growths * last * 1.0001
        assert ((got - want).abs() <= bound[:, None, None]).all()
    else:
        # 2^-4 of itself a rounding; below the normal range half of 2^-9 of the scale.
        bound = growths[:, None, None] * (want.abs() * 1.07 * 2.0 ** -4 + last[:, None, None] * 2.0 ** -10)
        assert ((got - want).abs() <= bound).all()
    assert torch.equal(cache.k[0].view(torch.uint8).cpu(), torch.zeros(heads, bs, dim, dtype=torch.uint8))


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


def attention_reference(q, k, v, ks, vs, table, lengths, starts, scale, causal, window):
    """(out, sum_j p_j |v_j|, largest |v_j|, lse) in 64 bits."""
    T, hq, dim = q.shape
    bs, kv = k.shape[2], k.shape[1]
    out, mag, big = (torch.zeros(T, hq, dim, dtype=torch.float64) for _ in range(3))
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64)
    for r, n in enumerate(lengths):
        first, last = (starts[r], starts[r + 1]) if starts is not None else (r, r + 1)
        nq = last - first
        if n == 0 or nq == 0:
            continue
        pages = table[r, :-(-n // bs)].long()
        K = (k[pages].double() * ks[pages].double()[..., None, None]).transpose(0, 1).reshape(kv, -1, dim)[:, :n]
        V = (v[pages].double() * vs[pages].double()[..., None, None]).transpose(0, 1).reshape(kv, -1, dim)[:, :n]
        K, V = (x.repeat_interleave(hq // kv, 0) for x in (K, V))
        s = torch.einsum("qhd,htd->qht", q[first:last].double(), K) * scale
        place = torch.arange(n - nq, n)[:, None]
        j = torch.arange(n)[None, :]
        seen = (j <= place) if causal else torch.ones(nq, n, dtype=torch.bool)
        if window:
            seen = seen & (j > place - window)
        s = s.masked_fill(~seen[:, None, :], -math.inf)
        some = seen.any(1)
        p = torch.softmax(s, -1)
        p[~some] = 0
        out[first:last] = torch.einsum("qht,htd->qhd", p, V)
        mag[first:last] = torch.einsum("qht,htd->qhd", p, V.abs())
        big[first:last] = V.abs().amax()
        lse[first:last] = torch.logsumexp(s, -1)
    return out, mag, big, lse


def attention_case(lengths, fresh, hq, kv, dim, bs, code, dtype, seed=0, spare=2, spread=1.0, layout="heads"):
    g = gen(seed)
    per = [-(-n // bs) for n in lengths]
    pages = sum(per) + spare
    k, v, ks, vs = random_pools(pages, kv, bs, dim, code, g)
    ks, vs = ks * torch.exp(spread * torch.randn(ks.shape, generator=g)), vs * torch.exp(spread * torch.randn(vs.shape, generator=g))
    order = torch.randperm(pages, generator=g)[:sum(per)].to(torch.int32)
    table = torch.full((len(lengths), max(per + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(per):
        table[r, :n] = order[at:at + n]
        at += n
    starts = None
    if fresh is not None:
        starts = [0]
        for n in fresh:
            starts.append(starts[-1] + n)
    T = starts[-1] if starts else len(lengths)
    q = torch.randn(T, hq, dim, generator=g).to(HALF[dtype][0])
    return q, k, v, ks, vs, table, lengths, starts


def run_attention(case, causal=True, window=0, scale=None, lse=True, cache=None):
    q, k, v, ks, vs, table, lengths, starts = case
    cache = cache or dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    return dk.cache_attention(q.cuda(), cache, table.cuda(), ints(lengths), ints(starts) if starts is not None else None,
                              scale=scale, causal=causal, window=window, lse=lse)


def tolerance(out, mag, big, n, unit):
    """Rounding of the result; of the weights to fp16 (2^-11 each, or 2^-25 of
    the largest where they are below fp16's normal range, for each of n tokens);
    as much again for the fp32 scores and sums (2^-24 over 256 terms)."""
    return unit * out.abs() + 2.0 ** -10 * mag + n * 2.0 ** -25 * big + 1e-7


def check_attention(case, causal=True, window=0, scale=None, **kw):
    q, k, v, ks, vs, table, lengths, starts = case
    unit = HALF["fp16" if q.dtype == torch.float16 else "bf16"][1]
    s = scale if scale is not None else q.shape[2] ** -0.5
    want, mag, big, lse = attention_reference(q, k, v, ks, vs, table, lengths, starts, s, causal, window)
    out, got_lse = run_attention(case, causal, window, scale, **kw)
    out = out.double().cpu()
    assert out.isfinite().all()
    bad = (out - want).abs() > tolerance(want, mag, big, max(lengths + [1]), unit)
    assert not bad.any(), (bad.nonzero()[:4], (out - want).abs().max())
    none = lse.isinf()
    assert torch.equal(got_lse.cpu().isinf(), none)
    assert (out[none] == 0).all()
    # The log of a sum of weights that are each 2^-18 right, and the scores' own fp32 rounding.
    assert ((got_lse.double().cpu() - lse)[~none].abs() <= 2e-5 + 2e-6 * lse[~none].abs()).all()


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 400]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("hq,kv,dim,bs", [(8, 2, 128, 64), (8, 8, 64, 16), (32, 2, 128, 48), (4, 1, 256, 32), (7, 1, 64, 256), (12, 4, 256, 16), (24, 2, 64, 32)])
def test_attention_single_queries(dtype, code, hq, kv, dim, bs):
    check_attention(attention_case(EDGES, None, hq, kv, dim, bs, code, dtype, seed=hq + dim))


@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("hq,kv,dim,bs", [(8, 2, 128, 64), (6, 6, 64, 16), (16, 2, 256, 32), (5, 1, 128, 16)])
def test_attention_several_queries(code, dtype, hq, kv, dim, bs):
    lengths, fresh = [1, 5, 16, 17, 40, 70, 200, 0, 333, 64], [1, 5, 3, 17, 0, 64, 7, 0, 100, 1]
    for window in (0, 1, 20):
        check_attention(attention_case(lengths, fresh, hq, kv, dim, bs, code, dtype, seed=window + dim), window=window)
    check_attention(attention_case(lengths, fresh, hq, kv, dim, bs, code, dtype, seed=5), causal=False)


@pytest.mark.parametrize("hq,kv,dim", [(8, 4, 128), (8, 2, 128), (6, 1, 128), (16, 2, 128), (3, 1, 64), (12, 2, 64), (2, 1, 256), (4, 1, 256)])
@pytest.mark.parametrize("code,dtype", [("int8", "fp16"), ("e4m3", "bf16")])
def test_attention_drafts(hq, kv, dim, code, dtype):
    # Five queries for each request: 10 to 40 rows for a KV head, one to several tiles of each width.
    lengths = [5, 6, 16, 20, 21, 133, 1000, 5]
    check_attention(attention_case(lengths, [5] * 8, hq, kv, dim, 32, code, dtype, seed=hq))
    check_attention(attention_case(lengths, [5] * 8, hq, kv, dim, 16, code, dtype, seed=hq), window=9)
    check_attention(attention_case([9000, 3000], [5, 5], hq, kv, dim, 64, code, dtype, seed=hq))


def test_attention_shapes_share_a_workspace():
    # Kernels of several row tiles take turns on one stream's workspace; what one writes must not reach another's counters.
    one = attention_case([5000, 7000, 30], None, 8, 2, 128, 64, "int8", "fp16")
    many = attention_case([5000, 7000, 30], [5, 5, 5], 8, 2, 128, 64, "int8", "fp16")
    more = attention_case([5000, 7000], [40, 9], 8, 2, 128, 64, "int8", "fp16")
    want = [run_attention(c)[0] for c in (one, many, more)]
    for _ in range(5):
        for c, w in zip((one, many, more), want):
            assert torch.equal(run_attention(c)[0], w)
    check_attention(one), check_attention(many), check_attention(more)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100])
def test_attention_window(window):
    check_attention(attention_case(EDGES, None, 8, 2, 128, 16, "int8", "fp16", seed=window), window=window)


@pytest.mark.parametrize("hq,kv,dim", [(8, 1, 128), (2, 2, 64), (4, 2, 256), (16, 1, 128)])
def test_attention_long_context_split_over_the_gpu(hq, kv, dim):
    check_attention(attention_case([20011], None, hq, kv, dim, 64, "int8", "fp16", seed=dim))
    check_attention(attention_case([3, 9000, 0, 77, 4097], None, hq, kv, dim, 32, "e4m3", "bf16", seed=dim))


def test_attention_many_requests():
    g = gen(21)
    lengths = torch.randint(0, 50, (9000,), generator=g).tolist()  # more than one launch's requests
    check_attention(attention_case(lengths, None, 2, 1, 64, 16, "int8", "fp16"))


def test_attention_many_requests_of_several_queries():
    g = gen(22)
    fresh = torch.randint(0, 4, (2500,), generator=g).tolist()
    lengths = [n + int(x) for n, x in zip(fresh, torch.randint(0, 40, (2500,), generator=g).tolist())]
    check_attention(attention_case(lengths, fresh, 4, 2, 64, 16, "e4m3", "fp16"), window=11)


def test_attention_and_append_of_nothing():
    q, k, v, ks, vs, table, _, _ = attention_case([20], None, 8, 2, 128, 16, "int8", "fp16")
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    o, l = dk.cache_attention(q.cuda()[:0], cache, table.cuda()[:0], ints([]), lse=True)
    assert o.shape == (0, 8, 128) and l.shape == (0, 8)
    o = dk.cache_attention(q.cuda()[:0], cache, table.cuda(), ints([20]), ints([0, 0]))
    assert o.shape == (0, 8, 128)
    dk.cache_append(q.cuda()[:0, :2], q.cuda()[:0, :2], ints([], torch.int64), cache)
    assert torch.equal(cache.k.cpu(), k)
    # Rows of q beyond the last request's are left alone.
    out = torch.full((3, 8, 128), 7.0, dtype=torch.float16, device="cuda")
    dk.cache_attention(q.cuda().expand(3, 8, 128), cache, table.cuda(), ints([20]), ints([1, 2]), out=out)
    assert (out[0] == 7).all() and (out[2] == 7).all() and not (out[1] == 7).any()


def test_attention_scale_and_large_scores():
    case = attention_case([300, 40], None, 8, 2, 128, 64, "int8", "bf16", spread=0.3)
    check_attention(case, scale=0.02)
    big = (case[0] * 2.0 ** 60,) + case[1:]         # bf16 queries past fp16's range
    check_attention(big, scale=2.0 ** -60 * 128 ** -0.5)
    small = (case[0] * 2.0 ** -90,) + case[1:]
    check_attention(small, scale=2.0 ** 90 * 128 ** -0.5)
    check_attention(case, scale=0.0)


def test_attention_page_scales_of_any_size():
    q, k, v, ks, vs, table, lengths, starts = attention_case([700], None, 8, 2, 128, 16, "int8", "fp16", spread=0.0)
    vs = vs * 2.0 ** torch.linspace(-40, 12, vs.numel()).view_as(vs)
    check_attention((q, k, v, ks, vs, table, lengths, starts))
    ks = torch.zeros_like(ks)                        # every score 0
    check_attention((q, k, v, ks, torch.zeros_like(vs), table, lengths, starts))


@pytest.mark.parametrize("window", [0, 50])
def test_attention_ignores_what_is_masked(window):
    """Bytes past a request's tokens, pages of no one and entries past the table's need may hold anything."""
    case = attention_case([70, 1, 0, 100], None, 8, 2, 128, 32, "e4m3", "fp16", seed=8)
    q, k, v, ks, vs, table, lengths, starts = case
    clean = run_attention(case, window=window)[0]
    nan = 0x7F
    kd, vd = k.clone().view(torch.uint8), v.clone().view(torch.uint8)
    used = set()
    for r, n in enumerate(lengths):
        for b in range(-(-n // 32)):
            page = int(table[r, b])
            used.add(page)
            rows = torch.arange(b * 32, b * 32 + 32)
            hidden = (rows >= n) | ((rows < n - window) if window else torch.zeros(32, dtype=torch.bool))
            kd[page][:, hidden] = nan
            vd[page][:, hidden] = nan
    for page in range(k.shape[0]):
        if page not in used:
            kd[page], vd[page], ks[page], vs[page] = nan, nan, float("nan"), float("nan")
    table = table.clone()
    table[:, -1] = 2 ** 31 - 1
    dirty = run_attention((q, kd.view(k.dtype), vd.view(v.dtype), ks, vs, table, lengths, starts), window=window)[0]
    assert torch.equal(clean, dirty)


def test_attention_hides_tokens_of_entries_outside_the_pool():
    q, k, v, ks, vs, table, lengths, starts = attention_case([64], None, 8, 2, 128, 16, "int8", "fp16")
    for bad in (-1, 10 ** 6):
        t = table.clone()
        t[0, 1] = bad
        out = run_attention((q, k, v, ks, vs, t, lengths, starts))[0]
        keep = torch.tensor([[table[0, 0], table[0, 2], table[0, 3]]], dtype=torch.int32)
        want = run_attention((q, k, v, ks, vs, keep, [48], starts))[0]
        torch.testing.assert_close(out, want, rtol=2.0 ** -10, atol=1e-4)
        t[:] = bad
        assert (run_attention((q, k, v, ks, vs, t, lengths, starts))[0] == 0).all()


def test_attention_strides_and_out():
    case = attention_case([70, 130, 5], None, 8, 2, 128, 32, "int8", "fp16")
    q, k, v, ks, vs, table, lengths, starts = case
    want = run_attention(case, lse=False)
    t = lambda x: x.transpose(1, 2).contiguous().cuda().transpose(1, 2)  # noqa: E731  [blocks, block_size, heads, dim]
    both = torch.stack([k, v], 1).cuda()  # [blocks, 2, heads, block_size, dim]
    for kk, vv in ((t(k), t(v)), (both[:, 0], both[:, 1]), (t(k), both[:, 1])):
        cache = dk.PagedCache8.from_tensors(kk, vv, ks.cuda(), vs.cuda())
        assert torch.equal(run_attention(case, lse=False, cache=cache), want)
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    wide = torch.zeros(3, 20, 128, dtype=torch.float16, device="cuda")
    wide[:, 4:12] = q.cuda()
    wide_table = torch.full((3, 40), 77, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table.cuda()
    out = torch.full_like(want, float("nan"))
    got = dk.cache_attention(wide[:, 4:12], cache, wide_table[:, :table.shape[1]], ints(lengths), out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    odd = torch.zeros(3 * 8 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 8, 128)
    odd.copy_(q)
    assert torch.equal(dk.cache_attention(odd, cache, table.cuda(), ints(lengths)), want)
    assert torch.equal(dk.cache_attention(q.cuda().transpose(0, 1).contiguous().transpose(0, 1), cache, table.cuda(), ints(lengths)), want)


def test_attention_offsets_past_32_bits():
    blocks, bs, kv, dim = 2 ** 31 // (256 * 128) + 40, 256, 1, 128
    cache = dk.PagedCache8(blocks, bs, kv, dim)
    assert cache.k.numel() > 2 ** 31
    g = gen(1)
    pages = [blocks - 1, blocks - 3]
    k, v, ks, vs = random_pools(2, kv, bs, dim, "int8", g)
    q = torch.randn(1, 8, dim, generator=g).half()
    x = torch.randn(2, kv, dim, generator=g).half()
    for i, p in enumerate(pages):
        cache.k[p], cache.v[p], cache.k_scale[p], cache.v_scale[p] = k[i].cuda(), v[i].cuda(), ks[i].cuda(), vs[i].cuda()
    slots = torch.tensor([pages[1] * bs + 254, pages[1] * bs + 255])
    dk.cache_append(x.cuda(), x.cuda(), slots.cuda(), cache)
    small = [t[[blocks - 1, blocks - 3]].cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    want, scale = append_reference(k, ks, x, torch.tensor([bs + 254, bs + 255]), "int8")
    assert torch.equal(small[0], want) and torch.equal(small[2], scale)
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    want, mag, big, _ = attention_reference(q, *small, table, [512], None, 128 ** -0.5, True, 0)
    out = dk.cache_attention(q.cuda(), cache, ints([pages]), ints([512])).double().cpu()
    assert ((out - want).abs() <= tolerance(want, mag, big, 512, 2.0 ** -11)).all()


def test_attention_repeats_its_bits_on_any_stream_and_in_graphs():
    case = attention_case([5000, 3, 777, 0, 20000], None, 32, 8, 128, 64, "int8", "fp16")
    q, k, v, ks, vs, table, lengths, starts = case
    cache = dk.PagedCache8.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    args = (q.cuda(), cache, table.cuda(), ints(lengths))
    want = dk.cache_attention(*args)
    for _ in range(20):
        assert torch.equal(dk.cache_attention(*args), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams * 5:
        with torch.cuda.stream(s):
            outs.append(dk.cache_attention(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        dk.cache_attention(*args, out=out)
    for _ in range(3):  # a graph's replay beside calls of the stream that it was captured on
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        again = dk.cache_attention(*args)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)


def test_attention_and_cache_refuse():
    case = attention_case([20], None, 8, 2, 128, 16, "int8", "fp16")
    q, k, v, ks, vs, table, lengths, starts = [x.cuda() if isinstance(x, torch.Tensor) else x for x in case]
    cache = dk.PagedCache8.from_tensors(k, v, ks, vs)
    n = ints(lengths)
    for bad, msg in [
        (lambda: dk.cache_attention(q.float(), cache, table, n), "fp16 or bf16"),
        (lambda: dk.cache_attention(q[:, :7], cache, table, n), "multiple of kv_heads"),
        (lambda: dk.cache_attention(q[..., :64], cache, table, n), "head_dim"),
        (lambda: dk.cache_attention(q.cpu(), cache, table, n), "CUDA"),
        (lambda: dk.cache_attention(q, cache, table.long(), n), "block_table"),
        (lambda: dk.cache_attention(q, cache, table, n.long()), "lengths"),
        (lambda: dk.cache_attention(q, cache, table, n, n), "starts"),
        (lambda: dk.cache_attention(q.expand(2, 8, 128), cache, table, n), "one token for each request"),
        (lambda: dk.cache_attention(q, cache, table, n, window=3, causal=False), "window"),
        (lambda: dk.cache_attention(q, cache, table, n, out=q.bfloat16()), "out must be"),
        (lambda: dk.PagedCache8.from_tensors(k.float(), v.float(), ks, vs), "int8"),
        (lambda: dk.PagedCache8.from_tensors(k, v.view(torch.float8_e4m3fn), ks, vs), "both"),
        (lambda: dk.PagedCache8.from_tensors(k, v, ks.half(), vs), "fp32"),
        (lambda: dk.PagedCache8.from_tensors(k, v, ks[:, :1], vs), "blocks, kv_heads"),
        (lambda: dk.PagedCache8(2, 24, 1, 128), "block_size"),
        (lambda: dk.PagedCache8(2, 16, 1, 96), "head_dim"),
        (lambda: dk.cache_append(q[:, :2].float(), q[:, :2].float(), ints([0], torch.int64), cache), "fp16 or bf16"),
        (lambda: dk.cache_append(q[:, :3], q[:, :3], ints([0], torch.int64), cache), "kv_heads"),
        (lambda: dk.cache_append(q[:, :2], q[:, :2].bfloat16(), ints([0], torch.int64), cache), "shape and type"),
        (lambda: dk.cache_append(q[:, :2], q[:, :2], ints([0]), cache), "slots"),
        (lambda: dk.cache_plan(n, n, table, n, ints([0, 1, 0], torch.int64), 16, 1), "ring"),
        (lambda: dk.cache_plan(n, n.long(), table, n, ints([0, 1, 0, 0], torch.int64), 16, 1), "fresh"),
        (lambda: dk.cache_plan(n, n, table, n, ints([0, 1, 0, 0], torch.int64), 20, 1), "block_size"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            bad()


# ---------------------------------------------------------------------------
# Block norm
# ---------------------------------------------------------------------------


def norm_reference(r, y, kind, pw, pb, gate, act, a, b, w, c, eps):
    def one(x, weight, bias):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
        return x if bias is None else x + bias.double()

    r = a * r.double()
    if y is not None:
        u = y.double()
        if pw is not None:
            u = one(u, pw, pb)
        if gate is not None:
            g = gate.double()
            u = u * {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z * torch.sigmoid(z)}[act](g)
        r = r + b * u
    return r, None if w is None else one(r, w, c)


def check_norm(rows, dim, dtype="fp16", residual=None, kind="rms", post=False, gate=None, act="none", y=True, pre=True, bias=False,
               seed=0, lead=None, inplace=False, mean=0.0):
    g = gen(seed)
    t, unit = HALF[dtype]
    rt = {"fp32": torch.float32, None: t}[residual]
    shape = (*(lead if lead is not None else (rows,)), dim)
    new = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    r = (new(*shape) * 2 + mean).to(rt)
    yy = (new(*shape) + mean).to(t) if y else None
    weight = lambda: (1 + 0.3 * new(dim)).to(t)  # noqa: E731
    pw, pb = (weight(), new(dim).to(t) if bias else None) if post else (None, None)
    w, c = (weight(), new(dim).to(t) if bias else None) if pre else (None, None)
    gt = {"channel": (dim,), "row": (*shape[:-1], 1), "full": shape}[gate] if gate else None
    gt = new(*gt).to(t) if gt else None
    want_r, want_h = norm_reference(r, yy, kind, pw, pb, gt, act, 0.9, 1.3, w, c, 1e-5)
    cu = lambda x: None if x is None else x.cuda()  # noqa: E731
    rd = r.cuda()
    got_r, got_h = dk.block_norm(rd, cu(yy), kind=kind, post_weight=cu(pw), post_bias=cu(pb), gate=cu(gt), gate_act=act, residual_scale=0.9,
                                 block_scale=1.3, pre_weight=cu(w), pre_bias=cu(c), eps=1e-5, inplace=inplace)
    assert (got_r.data_ptr() == rd.data_ptr()) == inplace
    # The output's rounding, and fp32's: sums of dim terms (their rounding grows as sqrt(dim) at most log2(dim)
    # deep a tree, bounded here by 64 units), relative to the terms that are added.
    f32 = 64 * 2.0 ** -24
    ur = unit if rt == t else 2.0 ** -24
    add = (0.9 * r.double()).abs() + (want_r - 0.9 * r.double()).abs()
    if pb is not None:
        add = add + 1.3 * pb.double().abs() * (gt.double().abs() if gt is not None else 1)
    spread = 1 + (abs(mean) if kind == "layer" else 0)
    assert ((got_r.double().cpu() - want_r).abs() <= ur * want_r.abs() + f32 * add * spread + 1e-7).all()
    if w is None:
        assert got_h is None
        return
    terms = (want_h - (c.double() if c is not None else 0)).abs() + (c.double().abs() if c is not None else 0)
    size = add.amax(-1, keepdim=True) / want_r.double().std(-1, correction=0, keepdim=True).clamp(min=1e-3) if dim > 1 else 1.0
    assert ((got_h.double().cpu() - want_h).abs() <= unit * want_h.abs() + f32 * (terms + size * w.double().abs()) * spread + 1e-7).all()


@pytest.mark.parametrize("dim", [1, 7, 64, 65, 127, 256, 264, 511, 520, 1024, 2040, 2049, 4096, 5001, 8192, 8200, 11008, 16384, 20001, 32768])
def test_norm_sizes(dim):
    check_norm(3, dim, kind="rms", post=True, gate="full", act="silu", seed=dim)
    if dim > 1:
        check_norm(2, dim, dtype="bf16", kind="layer", post=True, bias=True, gate="channel", act="sigmoid", residual="fp32", seed=dim)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("residual", [None, "fp32"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("form", [
    dict(y=False), dict(pre=False), dict(), dict(post=True), dict(gate="channel"), dict(gate="row", act="sigmoid"),
    dict(gate="full", act="silu", post=True), dict(post=True, bias=True, pre=False, gate="row"),
])
def test_norm_forms(dtype, residual, kind, form):
    check_norm(5, 320, dtype, residual, kind, **form)
    check_norm(5, 321, dtype, residual, kind, **form)


def test_norm_leading_dims_rows_and_inplace():
    for lead in ((), (1,), (2, 3), (301,)):
        check_norm(0, 256, lead=lead, post=True, gate="full", act="sigmoid")
        check_norm(0, 256, lead=lead, inplace=True)
    check_norm(1000, 128, gate="row", inplace=True, residual="fp32")
    check_norm(4, 4096, kind="layer", post=True, bias=True, mean=30.0)


@pytest.mark.parametrize("dim", [2056, 4104, 5120, 5128, 6152, 7168, 8000, 8192, 16000])
def test_norm_many_rows(dim):
    # Enough rows for the shapes that keep every SM busy.
    check_norm(333, dim, kind="layer", post=True, gate="row", act="silu", seed=dim)
    check_norm(333, dim, dtype="bf16", residual="fp32", post=True, seed=dim)


def test_norm_strided_rows():
    g = gen(5)
    big = torch.randn(9, 3 * 512 + 8, generator=g).half().cuda()
    for lo in (0, 8, 3):  # 3: rows that are not on a 16-byte boundary
        r, y, z = big[:, lo:lo + 512], big[:, 512:1024], big[:, 1024:1536]
        w = torch.ones(512, dtype=torch.float16, device="cuda")
        got = dk.block_norm(r, y, gate=z, pre_weight=w)
        want = dk.block_norm(r.contiguous(), y.contiguous(), gate=z.contiguous(), pre_weight=w)
        tol = dict(rtol=2.0 ** -10, atol=2.0 ** -12)  # another order of the same sum may round the other way
        assert torch.equal(got[0], want[0])
        torch.testing.assert_close(got[1], want[1], **tol)
    keep = big.clone()
    r2, h2 = dk.block_norm(big[:, 8:520], keep[:, 512:1024], pre_weight=w, inplace=True)
    assert r2.data_ptr() == big[:, 8:520].data_ptr()
    assert torch.equal(big[:, :8], keep[:, :8]) and torch.equal(big[:, 520:], keep[:, 520:])
    assert torch.equal(big[:, 8:520], dk.block_norm(keep[:, 8:520], keep[:, 512:1024])[0])


@pytest.mark.parametrize("residual", [torch.float16, torch.float32])
@pytest.mark.parametrize("dim,width", [(65, 73), (65, 70), (1001, 1009), (1001, 1002), (7, 7), (2049, 2049), (9001, 9009)])
def test_norm_rows_off_the_boundary(residual, dim, width):
    """Rows that begin anywhere: alike (strides equal to multiples of 8) and not; weights on odd places too."""
    g = gen(dim + width)
    rows = 37
    r = torch.randn(rows, width, generator=g).to(residual)
    y = torch.randn(rows, dim, generator=g).half()
    gate = torch.randn(rows, dim, generator=g).half()
    w = torch.randn(4 * dim + 1, generator=g).half()
    pw, pb, hw, hb = (w[i * dim + 1:(i + 1) * dim + 1] for i in range(4))
    d = w.cuda()
    dpw, dpb, dhw, dhb = (d[i * dim + 1:(i + 1) * dim + 1] for i in range(4))
    keep = r.cuda()
    for kind in ("rms", "layer"):
        want_r, want_h = norm_reference(r[:, :dim], y, kind, pw, pb, gate, "sigmoid", 0.9, 1.3, hw, hb, 1e-5)
        for inplace in (False, True):
            rd = keep.clone()
            got_r, got_h = dk.block_norm(rd[:, :dim], y.cuda(), kind=kind, post_weight=dpw, post_bias=dpb, gate=gate.cuda(), gate_act="sigmoid",
                                         residual_scale=0.9, block_scale=1.3, pre_weight=dhw, pre_bias=dhb, eps=1e-5, inplace=inplace)
            assert torch.equal(rd[:, dim:], keep[:, dim:])
            unit = 2.0 ** -11 if residual == torch.float16 else 2.0 ** -24
            f32 = 64 * 2.0 ** -24
            size = r[:, :dim].double().abs() + want_r.abs() + 4 * pb.double().abs()
            assert ((got_r.double().cpu() - want_r).abs() <= unit * want_r.abs() + f32 * (size + 4)).all()
            assert ((got_h.double().cpu() - want_h).abs() <= 2.0 ** -11 * want_h.abs() + f32 * (want_h.abs() + 16 * hw.double().abs() + hb.double().abs()) + 1e-7).all()


def test_norm_of_nothing_zeros_and_odd_values():
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    e = torch.empty(0, 64, dtype=torch.float16, device="cuda")
    r, h = dk.block_norm(e, e, pre_weight=w)
    assert r.shape == h.shape == (0, 64)
    r, h = dk.block_norm(e, e, post_weight=w, gate=e, pre_weight=w)
    assert r.shape == h.shape == (0, 64)
    z = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    assert (dk.block_norm(z, z, pre_weight=w)[1] == 0).all()
    z[1, 5] = float("nan")
    h = dk.block_norm(z, z, pre_weight=w)[1]
    assert (h[0] == 0).all() and h[1].isnan().all()
    gate = torch.tensor([[60000.0], [-60000.0]], dtype=torch.float16, device="cuda").expand(2, 64)
    one = torch.ones(2, 64, dtype=torch.float16, device="cuda")
    for act in ("sigmoid", "silu"):
        r = dk.block_norm(torch.zeros_like(one), one, gate=gate, gate_act=act)[0]
        assert (r[0] == (1 if act == "sigmoid" else 60000)).all() and (r[1] == 0).all()


def test_norm_refuses():
    x = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    w = x[0]
    for bad, msg in [
        (lambda: dk.block_norm(x), "nothing to do"),
        (lambda: dk.block_norm(x, gate=x, pre_weight=w), "belong to y"),
        (lambda: dk.block_norm(x, x, post_bias=w), "post_weight"),
        (lambda: dk.block_norm(x, x, pre_bias=w), "pre_weight"),
        (lambda: dk.block_norm(x.bfloat16(), x, pre_weight=w), "residual must have"),
        (lambda: dk.block_norm(x, x.float(), pre_weight=w), "fp16 or bf16"),
        (lambda: dk.block_norm(x, x[:1], pre_weight=w), "shape"),
        (lambda: dk.block_norm(x, x, gate=x[:, :3], pre_weight=w), "gate must be"),
        (lambda: dk.block_norm(x, x, pre_weight=w[:32]), "pre_weight must be"),
        (lambda: dk.block_norm(x, x, pre_weight=w.float()), "pre_weight must be"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            bad()
