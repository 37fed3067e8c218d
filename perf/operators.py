"""The serving operators around the W4A16 products: what is measured, and their plain forms.

Four operators of one decode step over a paged cache that is held in 8 bits:

  plan       block tables, slot maps and lengths of a step, from the requests' lengths
  append     a step's new keys and values, quantised into their pages (one scale per page and head)
  attention  a step's queries against the pages
  norm       a block's output normed, gated and added to the residual stream, and the next block's norm

Where ``own`` is false ``run`` computes them with elementary torch operations in 32 bits; where it is
true it makes the calls of ``decode_kernel`` that a user makes.
"""

import math
import os
import sys

import torch

own = False

GOLDEN = 0.6180339887498949
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
FLOOR = 2.0 ** -60  # smallest largest magnitude that a page's scale stands for


def _dk():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "decode-kernel_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import decode_kernel

    return decode_kernel


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # A decode step's tables: 64 requests with one new token each, some of which need a new page.
        dict(name="plan_step", op="plan", requests=64, cached=4096, new=1, released=0.0, block=64),
        # Prompts that arrive together, with requests that ended giving their pages back: 2048 requests, half a million tokens.
        dict(name="plan_prompts", op="plan", requests=2048, cached=2048, new=500, released=0.05, block=16),
        # One decode step of 96 requests, 8 KV heads of 128: a token into each request's last page.
        dict(name="append_step", op="append", requests=96, cached=180, new=1, heads=8, dim=128, block=64, code="int8", dtype="fp16"),
        # Ragged prompt pieces of about 100 tokens over an odd number of small heads, pages of 48 tokens.
        dict(name="append_pieces", op="append", requests=37, cached=75, new=211, heads=5, dim=64, block=48, code="int8", dtype="fp16"),
        # Long prompts being written to the cache: 16 requests, about 16 thousand tokens, in FP8.
        dict(name="append_prompts", op="append", requests=16, cached=0, new=2047, heads=8, dim=128, block=64, code="e4m3", dtype="bf16"),
        # One request of a few hundred tokens: the call's latency.
        dict(name="attention_one", op="attention", requests=1, length=700, low=1.0, queries=1, heads=32, kv_heads=8, dim=128, block=64,
             window=0, code="int8", dtype="fp16"),
        # A decode step over 32 requests whose contexts run from nothing to 8192 tokens: heads of an 8B-shaped stack.
        dict(name="attention_step", op="attention", requests=32, length=8192, low=0.0, queries=1, heads=32, kv_heads=8, dim=128, block=64,
             window=0, code="int8", dtype="fp16"),
        # Drafted tokens checked five at a time: 20 query rows for each KV head.
        dict(name="attention_draft", op="attention", requests=17, length=4001, low=0.2, queries=5, heads=32, kv_heads=8, dim=128, block=32,
             window=0, code="int8", dtype="bf16"),
        # Full multi-head attention with small heads, a sliding window and small pages.
        dict(name="attention_window", op="attention", requests=200, length=1900, low=0.0, queries=1, heads=12, kv_heads=12, dim=64, block=16,
             window=1000, code="e4m3", dtype="fp16"),
        # Four contexts of 128 thousand tokens, heads of a 70B-shaped stack: a gigabyte of cache.
        dict(name="attention_long", op="attention", requests=4, length=131071, low=0.9, queries=1, heads=64, kv_heads=8, dim=128, block=64,
             window=0, code="e4m3", dtype="bf16"),
        # One token between two blocks: the call's latency.
        dict(name="norm_token", op="norm", rows=1, dim=4096, kind="rms", post=False, gate="none", act="none", dtype="fp16", residual="fp16"),
        # A batch of prompts between two blocks, normed on both sides, with a gate for each value.
        dict(name="norm_rows", op="norm", rows=8192, dim=8192, kind="rms", post=True, gate="full", act="sigmoid", dtype="bf16", residual="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, even over the logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = min(max(n, low), high)
    return _not(n)


def _not(n):
    """n, or its neighbour where n is the one size that is left out."""
    return n + 8 if n == 3072 else n


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "attention", "norm", "norm"])
    dtype = rng.choice(["fp16", "bf16"])
    code = rng.choice(["int8", "e4m3"])
    block = rng.choice([16, 32, 48, 64, 128])
    if op == "plan":
        requests = _spread(rng, 1, 2048)
        new = rng.choice([1, 1, _spread(rng, 2, 500)])
        return dict(op=op, requests=requests, cached=_spread(rng, 16, 8192), new=new, released=rng.choice([0.0, 0.05, 0.3]), block=block)
    if op == "append":
        requests = _spread(rng, 1, 400)
        new = rng.choice([1, 1, _spread(rng, 2, max(2, min(4000, 30000 // requests)))])
        heads, dim = rng.choice([(8, 128), (1, 128), (5, 64), (4, 256), (12, 64)])
        return dict(op=op, requests=requests, cached=rng.choice([0, _spread(rng, 1, 300)]), new=new, heads=heads, dim=dim, block=block, code=code, dtype=dtype)
    if op == "attention":
        kv_heads, group, dim = rng.choice([(8, 4, 128), (8, 8, 128), (1, 8, 128), (4, 7, 128), (12, 1, 64), (2, 16, 128), (8, 2, 64), (4, 2, 256)])
        queries = rng.choice([1, 1, 1, _spread(rng, 2, 32)])
        requests = _spread(rng, 1, 256)
        # Keys and values within the longest listed case's, were all requests as long; fewer where many rows read them.
        most = 15 * (1 << 25) // (requests * kv_heads * dim) // max(1, queries * group // 16)
        length = _spread(rng, queries, max(queries, min(131072, most)))
        window = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
        return dict(op=op, requests=requests, length=length, low=rng.choice([0.0, 0.2, 1.0]), queries=queries, heads=kv_heads * group, kv_heads=kv_heads,
                    dim=dim, block=block, window=window, code=code, dtype=dtype)
    dim = rng.choice([_spread(rng, 64, 16384), _not(8 * _spread(rng, 8, 2048)), 4096, 8192])
    rows = _spread(rng, 1, min(16384, (1 << 26) // dim))
    return dict(op=op, rows=rows, dim=dim, kind=rng.choice(["rms", "layer"]), post=rng.choice([True, False]), gate=rng.choice(["none", "channel", "row", "full"]),
                act=rng.choice(["none", "sigmoid", "silu"]), dtype=dtype, residual=rng.choice([dtype, "fp32"]))


def _lengths(n, most, low):
    """n lengths of low * most..most, the first the longest, spread evenly; fixed by the case."""
    if n == 1:
        return [most]
    us = [1.0] + [((i + 1) * GOLDEN) % 1.0 for i in range(n - 1)]
    return [int(round(most * (low + (1.0 - low) * u))) for u in us]


def _plan_lengths(case):
    """(tokens held, new tokens; -1 where a request ended) of each request."""
    n = case["requests"]
    held = _lengths(n, case["cached"], 0.0)
    new = [case["new"]] * n if case["new"] == 1 else _lengths(n, case["new"], 0.0)[::-1]
    every = int(round(1.0 / case["released"])) if case["released"] else 0
    return held, [-1 if every and i % every == every - 1 else new[i] for i in range(n)]


def _append_lengths(case):
    n = case["requests"]
    new = [case["new"]] * n if case["new"] == 1 else [max(1, x) for x in _lengths(n, case["new"], 0.0)]
    return _lengths(n, case["cached"], 0.0), new


def _attention_lengths(case):
    """(tokens held with the new ones among them, new tokens) of each request: no queries where nothing is held is a slot without a request."""
    n, q = case["requests"], case["queries"]
    held = _lengths(n, case["length"], case["low"])
    return [max(x, q) if q > 1 else x for x in held], [q] * n


def work(case):
    op = case["op"]
    if op == "plan":
        held, new = _plan_lengths(case)
        n, b = case["requests"], case["block"]
        pages = sum(-(-(h + max(x, 0)) // b) - -(-h // b) for h, x in zip(held, new))
        given = sum(-(-h // b) for h, x in zip(held, new) if x < 0)
        tokens = sum(max(x, 0) for x in new)
        return {"bytes": 4 * (4 * n + 1) + 8 * tokens + 8 * (pages + given) + 64, "flops": 0}
    if op == "append":
        held, new = _append_lengths(case)
        per, b = case["heads"] * case["dim"], case["block"]
        tokens, pages = sum(new), sum(-(-(h + x) // b) - h // b for h, x in zip(held, new))
        return {"bytes": 2 * tokens * per * 3 + 8 * tokens + 2 * 8 * pages * case["heads"], "flops": 4 * tokens * per}
    if op == "attention":
        held, new = _attention_lengths(case)
        w, b, d = case["window"], case["block"], case["dim"]
        read = [min(h, w + q - 1) if w else h for h, q in zip(held, new)]
        pairs = sum(min(p + 1, w) if w else p + 1 for h, q in zip(held, new) for p in range(h - q, h) if p >= 0)
        pages = sum(-(-x // b) for x in read)
        tokens = sum(new)
        return {"bytes": 2 * sum(read) * case["kv_heads"] * d + pages * (8 * case["kv_heads"] + 4) + 4 * tokens * case["heads"] * d,
                "flops": 4 * pairs * case["heads"] * d}
    n = case["rows"] * case["dim"]
    size = 4 if case["residual"] == "fp32" else 2
    gate = {"none": 0, "channel": case["dim"], "row": case["rows"], "full": n}[case["gate"]]
    weights = case["dim"] * (1 + case["post"]) * (1 + (case["kind"] == "layer"))
    return {"bytes": n * (2 * size + 4) + 2 * gate + 2 * weights, "flops": n * (6 + 4 * case["post"])}


# ---------------------------------------------------------------------------------------------
# What a user's program has in hand
# ---------------------------------------------------------------------------------------------


def _generators(seed):
    return torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)


def _cuda(values, dtype):
    return torch.tensor(values, dtype=dtype).cuda()


def _codes(shape, code, gen):
    """Codes as a cache holds them: normally distributed values over their page's largest."""
    dtype, most = CODES[code]
    x = torch.randn(shape, generator=gen, device="cuda").mul_(most / 3.6).clamp_(-most, most)
    return (x.round_() if code == "int8" else x).to(dtype)


def _pages(held, block, gen):
    """Each request's pages out of a shuffled pool: (pages in the pool, table)."""
    per = [-(-h // block) for h in held]
    total = sum(per)
    pool = total + 7
    order = torch.randperm(pool, generator=gen)[:total].to(torch.int32)
    table = torch.full((len(held), max(1, max(per))), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(per):
        table[r, :n] = order[at:at + n]
        at += n
    return pool, table


def prepare(case, seed):
    cpu, gpu = _generators(seed)
    state = dict(case)
    op = case["op"]
    if op == "plan":
        held, new = _plan_lengths(case)
        mix = torch.randperm(len(held), generator=cpu).tolist()
        held, new = [held[i] for i in mix], [new[i] for i in mix]
        b = case["block"]
        pool, table = _pages(held, b, cpu)
        more = sum(-(-(h + max(x, 0)) // b) - -(-h // b) for h, x in zip(held, new))
        wide = torch.full((len(held), -(-(case["cached"] + case["new"]) // b) + 1), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        free = torch.randperm(pool + more + 64, generator=cpu).to(torch.int32)
        tokens = -(-sum(max(x, 0) for x in new) // 8) * 8  # the step's rows are padded to whole eights
        state |= dict(held=_cuda(held, torch.int32), fresh=_cuda(new, torch.int32), table=wide.cuda(), free=free.cuda(), tokens=tokens,
                      ring=_cuda([11, 11 + more + 20, 0, 0], torch.int64))
    elif op == "append":
        held, new = _append_lengths(case)
        b, heads, dim = case["block"], case["heads"], case["dim"]
        pool, table = _pages([h + x for h, x in zip(held, new)], b, cpu)
        slots = []
        for r, (h, x) in enumerate(zip(held, new)):
            at = torch.arange(h, h + x)
            slots.append(table[r, at // b].to(torch.int64) * b + at % b)
        shape = (sum(new), heads, dim)
        # Keys have a few large channels, as rotary heads do; tokens differ in size.
        size = torch.exp(0.4 * torch.randn((shape[0], heads, 1), generator=gpu, device="cuda"))
        channel = torch.exp(0.7 * torch.randn((1, heads, dim), generator=gpu, device="cuda"))
        k = torch.randn(shape, generator=gpu, device="cuda") * size * channel
        v = torch.randn(shape, generator=gpu, device="cuda") * size
        scale = lambda: torch.exp(0.3 * torch.randn((pool, heads), generator=gpu, device="cuda")) * 3.0 / CODES[case["code"]][1]  # noqa: E731
        state |= dict(k=k.to(DTYPES[case["dtype"]]), v=v.to(DTYPES[case["dtype"]]), slots=torch.cat(slots).cuda(),
                      k_pool=_codes((pool, heads, b, dim), case["code"], gpu), v_pool=_codes((pool, heads, b, dim), case["code"], gpu),
                      k_scale=scale(), v_scale=scale())
    elif op == "attention":
        held, new = _attention_lengths(case)
        mix = torch.randperm(len(held), generator=cpu).tolist()
        held = [held[i] for i in mix]
        pool, table = _pages(held, case["block"], cpu)
        shape = (pool, case["kv_heads"], case["block"], case["dim"])
        most = CODES[case["code"]][1]
        scale = lambda: torch.exp(0.3 * torch.randn(shape[:2], generator=gpu, device="cuda")) * 3.6 / most  # noqa: E731
        q = torch.randn((sum(new), case["heads"], case["dim"]), generator=gpu, device="cuda") * 1.2
        starts = [0]
        for x in new:
            starts.append(starts[-1] + x)
        state |= dict(q=q.to(DTYPES[case["dtype"]]), k_pool=_codes(shape, case["code"], gpu), v_pool=_codes(shape, case["code"], gpu), k_scale=scale(),
                      v_scale=scale(), table=table.cuda(), lengths=_cuda(held, torch.int32),
                      starts=_cuda(starts, torch.int32) if case["queries"] > 1 else None)
    else:
        rows, dim, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
        new = lambda *s: torch.randn(s, generator=gpu, device="cuda")  # noqa: E731
        weight = lambda: (1.0 + 0.2 * new(dim)).to(dtype)  # noqa: E731
        bias = lambda: (0.1 * new(dim)).to(dtype) if case["kind"] == "layer" else None  # noqa: E731
        gate = {"none": None, "channel": (dim,), "row": (rows, 1), "full": (rows, dim)}[case["gate"]]
        state |= dict(y=(2.0 * new(rows, dim) + 0.3).to(dtype), r=(3.0 * new(rows, dim) + 0.5).to(DTYPES[case["residual"]]),
                      post_weight=weight() if case["post"] else None, post_bias=bias() if case["post"] else None, pre_weight=weight(), pre_bias=bias(),
                      g=new(*gate).to(dtype) if gate else None)
    if own and op in ("append", "attention"):
        state["cache"] = _dk().PagedCache8.from_tensors(state["k_pool"], state["v_pool"], state["k_scale"], state["v_scale"])
    return state


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _own_plan(s):
    p = _dk().cache_plan(s["held"], s["fresh"], s["table"], s["free"], s["ring"], s["block"], s["tokens"])
    return {"lengths": p.lengths, "starts": p.starts, "slots": p.slots, "ring": p.ring, "table": s["table"], "free": s["free"]}


def _own_append(s):
    _dk().cache_append(s["k"], s["v"], s["slots"], s["cache"])
    # The codes are whole numbers (int8) or FP8 values, beside the scales that they count in.
    return {"k": s["k_pool"], "v": s["v_pool"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attention(s):
    return _dk().cache_attention(s["q"], s["cache"], s["table"], s["lengths"], s["starts"], window=s["window"])


def _own_norm(s):
    return _dk().block_norm(s["r"], s["y"], kind=s["kind"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["g"], gate_act=s["act"],
                            block_scale=0.7, residual_scale=1.1, pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=1e-5)


def _plain_plan(s):
    b, table, free = s["block"], s["table"], s["free"]
    requests, width = table.shape
    held, fresh = s["held"].clamp(min=0).long(), s["fresh"].clamp(min=0).long()
    ended = s["fresh"] < 0
    have, want = (held + b - 1) // b, (held + fresh + b - 1) // b
    wide = (fresh > 0) & (want > width)
    need = torch.where((fresh > 0) & ~wide, want - have, 0)
    offset = need.cumsum(0) - need
    head, tail = s["ring"][0], s["ring"][1]
    short = (need > 0) & (offset + need > tail - head)
    served = ~wide & ~short
    lengths = torch.where(ended, 0, torch.where(served, held + fresh, held))
    starts = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)])
    # Pages given back go to the ring's end, new pages come from its beginning.
    page = torch.arange(width, device=table.device)[None, :]
    gives = torch.where(ended, have.clamp(max=width), 0)
    back = gives.cumsum(0) - gives
    mine = ended[:, None] & (page < gives[:, None])
    at = torch.where(mine, (tail + back[:, None] + page) % free.numel(), free.numel())
    free_out = torch.cat([free, free.new_zeros(1)]).scatter(0, at.flatten(), table.flatten())[:-1]
    takes = (served & (need > 0))[:, None] & (page >= have[:, None]) & (page < want[:, None])
    table_out = torch.where(takes, free[(head + offset[:, None] + page - have[:, None]) % free.numel()], table)
    # Each token's request is the number of requests that end at or before it.
    t = torch.arange(s["tokens"], device=table.device)
    ends = torch.zeros(s["tokens"] + 1, dtype=torch.long, device=table.device)
    ends.scatter_add_(0, starts[1:].clamp(max=s["tokens"]), torch.ones_like(held))
    of = ends.cumsum(0)[:-1]
    there = of < requests
    of = of.clamp(max=requests - 1)
    position = held[of] + t - starts[of]
    there &= served[of]
    slots = table_out[of, (position // b).clamp(0, width - 1)].long() * b + position % b
    table.copy_(table_out)
    free.copy_(free_out)
    taken = torch.where(served & (need > 0), offset + need, 0).amax()
    return {"lengths": lengths.int(), "starts": starts.int(), "slots": torch.where(there, slots, -1),
            "ring": torch.stack([head + taken, tail + gives.sum(), torch.where(short, need, 0).sum(), wide.sum()]), "table": table, "free": free}


def _encode(x, code):
    dtype, most = CODES[code]
    x = torch.where(x.isnan(), 0.0, x).clamp(-most, most)
    return (x.round() if code == "int8" else x).to(dtype)


def _bytes(x):
    return x.view(torch.uint8)


def _plain_append(s):
    b, slots = s["block"], s["slots"]
    there = slots >= 0
    pages = s["k_pool"].shape[0]
    page, row = torch.where(there, slots // b, pages), slots % b
    first = torch.full((pages + 1,), b, device=slots.device).scatter_reduce(0, page, row, "amin")
    begun = first[:pages, None] > 0
    touched = first[:pages, None] < b
    for x, pool, scale in ((s["k"], s["k_pool"], s["k_scale"]), (s["v"], s["v_pool"], s["v_scale"])):
        x, most = x.float(), CODES[s["code"]][1]
        largest = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        largest = torch.zeros((pages + 1, x.shape[1]), device=x.device).scatter_reduce(0, page[:, None].expand_as(largest), largest, "amax")[:pages]
        want = largest.clamp(min=FLOOR) / torch.full_like(largest, most)
        old = torch.where(begun, scale, 0.0)
        new = torch.where(touched, torch.maximum(old, want), scale)
        grown = touched & begun & (new > old)
        ratio = torch.where(grown, old / new, 1.0)
        before = grown[:, :, None] & (torch.arange(b, device=x.device) < first[:pages, None, None])
        again = _encode(pool.float() * ratio[:, :, None, None], s["code"])
        _bytes(pool).copy_(torch.where(before[..., None], _bytes(again), _bytes(pool)))
        inverse = torch.ones_like(new) / new
        codes = _encode(x * torch.cat([inverse, inverse[:1]])[page][:, :, None], s["code"])
        keep = torch.cat([_bytes(pool), _bytes(pool)[:1]])  # one page more, for what has no slot
        keep[page, :, row] = _bytes(codes)
        _bytes(pool).copy_(keep[:pages])
        scale.copy_(new)
    return {"k": s["k_pool"], "v": s["v_pool"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    q, b, n = s["q"], s["block"], s["queries"]
    requests, width = s["table"].shape
    kv, dim = s["kv_heads"], s["dim"]
    group = s["heads"] // kv
    table = s["table"].clamp(min=0).long()

    def tokens(pool, scale):
        x = _bytes(pool)[table].view(pool.dtype).float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(requests, kv, width * b, dim)

    k, v = tokens(s["k_pool"], s["k_scale"]), tokens(s["v_pool"], s["v_scale"])
    rows = q.float().view(requests, n, kv, group, dim).transpose(1, 2).reshape(requests, kv, n * group, dim)
    scores = (rows @ k.transpose(-1, -2)) / math.sqrt(dim)
    at = torch.arange(width * b, device=q.device)[None, None, :]
    last = (s["lengths"][:, None] - n + torch.arange(n, device=q.device)[None, :])[:, :, None]
    seen = at <= last
    if s["window"]:
        seen &= at > last - s["window"]
    seen = seen[:, None, :, None, :].expand(requests, kv, n, group, width * b).reshape(scores.shape[0], kv, n * group, width * b)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ torch.where((at < s["lengths"][:, None, None])[..., None], v, 0.0)
    return out.view(requests, kv, n, group, dim).transpose(1, 2).reshape(q.shape).to(q.dtype)


def _plain_one_norm(x, weight, bias, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_norm(s):
    y = s["y"].float()
    if s["post_weight"] is not None:
        y = _plain_one_norm(y, s["post_weight"], s["post_bias"], s["kind"])
    if s["g"] is not None:
        g = s["g"].float()
        if s["act"] != "none":
            open_ = 1.0 / (1.0 + torch.exp(-g))
            g = open_ if s["act"] == "sigmoid" else g * open_
        y = y * g
    r = 1.1 * s["r"].float() + 0.7 * y
    return r.to(s["r"].dtype), _plain_one_norm(r, s["pre_weight"], s["pre_bias"], s["kind"]).to(s["y"].dtype)


_own = {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "norm": _own_norm}
_plain = {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "norm": _plain_norm}


# ---------------------------------------------------------------------------------------------
# In 64 bits
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    global own
    if case["op"] == "plan":
        return None  # whole numbers only
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "attention": _exact_attention, "norm": _exact_norm}[case["op"]](s)


def _exact_append(s):
    """The scales, and for FP8 what each code would be without rounding; int8 codes are whole numbers."""
    out = {}
    b, slots = s["block"], s["slots"].cpu()
    runs = []  # (first token, tokens, page, first row)
    for t, slot in enumerate(slots.tolist()):
        if runs and slot // b == runs[-1][2] and slot % b == runs[-1][3] + runs[-1][1]:
            runs[-1][1] += 1
        else:
            runs.append([t, 1, slot // b, slot % b])
    for name in ("k", "v"):
        x, most = s[name].cpu().double(), CODES[s["code"]][1]
        scale, pool = s[name + "_scale"].cpu().double(), s[name + "_pool"].cpu().double()
        for t, n, page, row in runs:
            mine = x[t:t + n]
            new = mine.abs().amax(dim=(0, 2)) / most
            if row:
                old = scale[page].clone()
                new = torch.maximum(new, old)
                pool[page, :, :row] *= (old / new)[:, None, None]
            scale[page] = new
            pool[page, :, row:row + n] = (mine / new[None, :, None]).transpose(0, 1)
        out[name] = pool if s["code"] == "e4m3" else None
        out[name + "_scale"] = scale
    return out


def _exact_attention(s):
    b, n, kv, dim = s["block"], s["queries"], s["kv_heads"], s["dim"]
    group = s["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, held in enumerate(s["lengths"].tolist()):
        if held == 0:
            continue
        pages = s["table"][r, :-(-held // b)].long()
        q = s["q"][r * n:(r + 1) * n].double().view(n, kv, group, dim)
        place = torch.arange(held, device="cuda")
        ahead = place[None, :] - (held - n + torch.arange(n, device="cuda"))[:, None]  # key's place less the query's
        hidden = (ahead > 0) | (ahead <= -s["window"]) if s["window"] else ahead > 0
        for h in range(kv):
            k = (s["k_pool"][pages, h] if s["code"] == "int8" else _bytes(s["k_pool"])[pages, h].view(torch.float8_e4m3fn)).double()
            v = (s["v_pool"][pages, h] if s["code"] == "int8" else _bytes(s["v_pool"])[pages, h].view(torch.float8_e4m3fn)).double()
            k = (k * s["k_scale"][pages, h].double()[:, None, None]).view(-1, dim)[:held]
            v = (v * s["v_scale"][pages, h].double()[:, None, None]).view(-1, dim)[:held]
            z = torch.einsum("qgd,td->qgt", q[:, h], k) * dim ** -0.5
            z = z.masked_fill(hidden[:, None, :], -math.inf)
            out[r * n:(r + 1) * n].view(n, kv, group, dim)[:, h] = torch.einsum("qgt,td->qgd", torch.softmax(z, -1), v)
    return out


def _exact_norm(s):
    def normed(x, w, c):
        if s["kind"] == "layer":
            variance, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            return (x - mean) * torch.rsqrt(variance + 1e-5) * w.double() + c.double()
        return x * torch.rsqrt(x.square().sum(1, keepdim=True) / x.shape[1] + 1e-5) * w.double()

    u = s["y"].double()
    if s["post_weight"] is not None:
        u = normed(u, s["post_weight"], s["post_bias"])
    if s["g"] is not None:
        g = s["g"].double()
        u = u * {"none": lambda a: a, "sigmoid": torch.sigmoid, "silu": lambda a: a * torch.sigmoid(a)}[s["act"]](g)
    r = s["r"].double() * 1.1 + u * 0.7
    return r, normed(r, s["pre_weight"], s["pre_bias"])
