"""The prompt-sized operators of a W4A16 decoder: what is measured, and their plain forms.

  rotary  rotary positions with one or several axes, of queries and keys together, and their gradient
  read    keys and values of a paged 8-bit cache, read back as rows
  gemm    many rows through 4-bit weights, and the gradient through the frozen weights
  gated   a gated feed-forward block's two projections, activation and product, and their gradient

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
GROUP = 128  # weights of a row that share a scale


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
        # A decode step of one request far into its context: the call's latency.
        dict(name="rotary_token", op="rotary", tokens=1, heads=32, kv_heads=8, dim=128, sections="64", paired=False, grad=False, dtype="fp16"),
        # Patches of a video (time, height, width) in one prompt of an 8B-shaped stack.
        dict(name="rotary_video", op="rotary", tokens=8192, heads=32, kv_heads=8, dim=128, sections="16,24,24", paired=False, grad=False, dtype="bf16"),
        # Training on images: two axes, neighbouring values paired, heads of 80 of which 64 values turn, and the gradient.
        dict(name="rotary_image_grad", op="rotary", tokens=1003, heads=12, kv_heads=12, dim=80, sections="16,16", paired=True, grad=True, dtype="fp32"),
        # One request's few hundred tokens.
        dict(name="read_one", op="read", requests=1, length=700, low=1.0, heads=8, dim=128, block=64, code="int8", dtype="fp16"),
        # Ragged prefixes of many requests over small heads and small pages.
        dict(name="read_prefixes", op="read", requests=200, length=1900, low=0.0, heads=12, dim=64, block=16, code="e4m3", dtype="bf16"),
        # A batch of 17 decoding requests through one square layer.
        dict(name="gemm_batch", op="gemm", rows=17, out=4096, width=4096, grad=False, dtype="fp16"),
        # An odd number of prompt tokens through a small layer whose outputs are no multiple of a tile.
        dict(name="gemm_ragged", op="gemm", rows=333, out=1000, width=2816, grad=False, dtype="bf16"),
        # A prompt of 2048 tokens through a 7B-shaped down projection.
        dict(name="gemm_prompt", op="gemm", rows=2048, out=4096, width=11008, grad=False, dtype="fp16"),
        # A training step's 1000 rows through a frozen layer and back.
        dict(name="gemm_grad", op="gemm", rows=1000, out=4096, width=4096, grad=True, dtype="bf16"),
        # One token's gated block: the weights stream once.
        dict(name="gated_token", op="gated", rows=1, out=11008, width=4096, act="silu", grad=False, dtype="fp16"),
        # Prompts of 4096 tokens together through a 7B-shaped gated block.
        dict(name="gated_prompt", op="gated", rows=4096, out=11008, width=4096, act="silu", grad=False, dtype="fp16"),
        # A training step's rows through a frozen gated block and back to its input.
        dict(name="gated_grad", op="gated", rows=1500, out=11008, width=4096, act="gelu", grad=True, dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, even over the logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(max(n, low), high)


def draw(rng):
    op = rng.choice(["rotary", "rotary", "read", "read", "gemm", "gemm", "gemm", "gated", "gated", "gated"])
    if op == "rotary":
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (12, 12, 64), (16, 16, 80), (7, 1, 256), (20, 5, 96), (1, 0, 128)])
        pairs = rng.choice([dim // 2, dim // 2, dim // 4])
        axes = rng.choice([1, 1, 2, 3])
        first = [rng.randint(1, max(1, pairs // 3)) for _ in range(axes - 1)]
        grad = rng.random() < 0.3
        tokens = _spread(rng, 1, 32768 * 40 * 128 // ((heads + kv_heads) * dim) // (4 if grad else 2))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, sections=",".join(str(n) for n in first + [pairs - sum(first)]), paired=rng.choice([False, False, True]),
                    grad=grad, dtype=rng.choice(["fp16", "bf16", "fp32"]))
    if op == "read":
        heads, dim = rng.choice([(8, 128), (1, 128), (5, 64), (4, 256), (12, 64)])
        requests = _spread(rng, 1, 400)
        return dict(op=op, requests=requests, length=_spread(rng, 1, max(1, min(65536, (1 << 27) // (requests * heads * dim)))), low=rng.choice([0.0, 0.2, 1.0]),
                    heads=heads, dim=dim, block=rng.choice([16, 32, 48, 64, 128]), code=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["fp16", "bf16"]))
    shapes = [(4096, 4096), (11008, 4096), (4096, 11008), (2816, 1024), (1024, 2816), (14336, 4096), (_spread(rng, 8, 12000), GROUP * _spread(rng, 1, 80)),
              (_spread(rng, 8, 4000), GROUP * _spread(rng, 1, 40))]
    if op == "gated":
        shapes.append((28672, 8192))
    out, width = rng.choice(shapes)
    grad = rng.random() < 0.4
    # At most the operations of the largest listed case.
    most = 4096 * 11008 * 4096 * 2 // (out * width * (2 if op == "gated" else 1) * (2 if grad else 1))
    case = dict(op=op, rows=_spread(rng, 1, max(1, min(8192, most))), out=out, width=width)
    if op == "gated":
        case["act"] = rng.choice(["silu", "silu", "gelu"])
    return case | dict(grad=grad, dtype=rng.choice(["fp16", "bf16"]))


def _lengths(n, most, low):
    """n lengths of low * most..most, the first the longest, spread evenly; fixed by the case."""
    if n == 1:
        return [most]
    us = [1.0] + [((i + 1) * GOLDEN) % 1.0 for i in range(n - 1)]
    return [int(round(most * (low + (1.0 - low) * u))) for u in us]


def _sections(case):
    """Pairs of each axis."""
    return [int(n) for n in case["sections"].split(",")]


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "rotary":
        pairs = sum(_sections(case))
        heads = case["tokens"] * (case["heads"] + case["kv_heads"])
        both = 2 if case["grad"] else 1
        return {"bytes": both * heads * case["dim"] * size * 2 + 8 * case["tokens"] * len(_sections(case)) + 4 * pairs, "flops": both * 6 * heads * pairs}
    if op == "read":
        held = _lengths(case["requests"], case["length"], case["low"])
        pages = sum(-(-x // case["block"]) for x in held)
        return {"bytes": 2 * 3 * sum(held) * case["heads"] * case["dim"] + pages * (8 * case["heads"] + 4) + 8 * len(held), "flops": 2 * sum(held) * case["heads"] * case["dim"]}
    matrices = 2 if op == "gated" else 1
    weights = matrices * case["out"] * (case["width"] // 2 + case["width"] // GROUP * 2)
    both = 2 if case["grad"] else 1
    return {"bytes": weights + both * size * case["rows"] * (case["out"] + case["width"]), "flops": both * matrices * 2 * case["rows"] * case["out"] * case["width"]}


# ---------------------------------------------------------------------------------------------
# What a user's program has in hand
# ---------------------------------------------------------------------------------------------


def _weights(out, width, gen):
    """4-bit weights as the quantiser leaves them: normally distributed, a group's largest at +-7, eight in a word, lowest first."""
    q = torch.randn((out, width // 8, 8), generator=gen, device="cuda").mul_(2.6).round_().clamp_(-7, 7).to(torch.int32)
    packed = torch.zeros((out, width // 8), dtype=torch.int32, device="cuda")
    for i in range(8):
        packed |= (q[..., i] & 15) << (4 * i)
    scales = torch.exp(0.2 * torch.randn((out, width // GROUP), generator=gen, device="cuda")) * (width ** -0.5 / 2.6)
    return packed, scales.to(torch.float16)


def _codes(shape, code, gen):
    dtype, most = CODES[code]
    x = torch.randn(shape, generator=gen, device="cuda").mul_(most / 3.6).clamp_(-most, most)
    return (x.round_() if code == "int8" else x).to(dtype)


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(s, generator=gpu, device="cuda")  # noqa: E731
    state, dtype, op = dict(case), DTYPES[case["dtype"]], case["op"]
    if op == "rotary":
        sections = state["sections"] = _sections(case)
        n, axes = case["tokens"], len(sections)
        if axes == 1:  # somewhere in a long context, pieces of several requests
            at = torch.arange(n) + 100000 - 37 * torch.randint(0, 2000, (1,), generator=cpu)
            at[n // 2:] -= 70001
            positions = at.cuda()
        else:  # time runs on; rows and columns of an image
            side = max(1, int(math.isqrt(max(1, n // 4))))
            t = torch.arange(n) + int(torch.randint(0, 5000, (1,), generator=cpu))
            positions = torch.stack([t // (side * side), t // side % side, t % side][3 - axes:]).cuda()
        frequency = torch.cat([10000.0 ** (-torch.arange(p).double() / max(p, 1)) for p in sections]).float().cuda()
        channel = torch.exp(0.5 * new(1, 1, case["dim"]))  # a few large channels
        make = lambda heads: (new(n, heads, case["dim"]) * channel).to(dtype) if heads else None  # noqa: E731
        state |= dict(positions=positions, frequency=frequency, q=make(case["heads"]), k=make(case["kv_heads"]))
        if case["grad"]:
            state |= dict(dq=make(case["heads"]), dk=make(case["kv_heads"]))
    elif op == "read":
        held = _lengths(case["requests"], case["length"], case["low"])
        held = [held[i] for i in torch.randperm(len(held), generator=cpu).tolist()]
        per = [-(-x // case["block"]) for x in held]
        order = torch.randperm(sum(per) + 7, generator=cpu).to(torch.int32)
        table = torch.full((len(held), max(1, max(per))), -1, dtype=torch.int32)
        at = 0
        for r, p in enumerate(per):
            table[r, :p] = order[at:at + p]
            at += p
        shape = (len(order), case["heads"], case["block"], case["dim"])
        scale = lambda: torch.exp(0.3 * new(*shape[:2])) * 3.6 / CODES[case["code"]][1]  # noqa: E731
        starts = torch.zeros(len(held) + 1, dtype=torch.int32)
        starts[1:] = torch.tensor(held).cumsum(0)
        state |= dict(k_pool=_codes(shape, case["code"], gpu), v_pool=_codes(shape, case["code"], gpu), k_scale=scale(), v_scale=scale(), table=table.cuda(),
                      lengths=torch.tensor(held, dtype=torch.int32).cuda(), starts=starts.cuda(), tokens=sum(held))
        if own:
            state["cache"] = _dk().PagedCache8.from_tensors(state["k_pool"], state["v_pool"], state["k_scale"], state["v_scale"])
    else:
        # Rows differ in size, and a few channels are large.
        x = new(case["rows"], case["width"]) * torch.exp(0.3 * new(case["rows"], 1)) * torch.exp(0.4 * new(1, case["width"]))
        state |= dict(x=x.to(dtype), w=_weights(case["out"], case["width"], gpu))
        if op == "gated":
            state["w2"] = _weights(case["out"], case["width"], gpu)
        if case["grad"]:
            state["dy"] = (0.1 * new(case["rows"], case["out"])).to(dtype)
    return state


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _own_rotary(s):
    sections = s["sections"] if len(s["sections"]) > 1 else None
    if not s["grad"]:
        return _dk().rotary(s["q"], s["k"], s["positions"], s["frequency"], sections=sections, paired=s["paired"])
    leaves = [x.detach().requires_grad_() for x in (s["q"], s["k"]) if x is not None]
    out = _dk().rotary(leaves[0], leaves[1] if len(leaves) > 1 else None, s["positions"], s["frequency"], sections=sections, paired=s["paired"])
    out = [x for x in out if x is not None]
    grads = torch.autograd.grad(out, leaves, [x for x in (s["dq"], s["dk"]) if x is not None])
    return [x.detach() for x in out], list(grads)


def _own_read(s):
    return _dk().cache_read(s["cache"], s["table"], s["lengths"], s["starts"], s["tokens"], dtype=DTYPES[s["dtype"]])


def _own_gemm(s):
    if not s["grad"]:
        return _dk().gemm(*s["w"], s["x"])
    x = s["x"].detach().requires_grad_()
    y = _dk().gemm(*s["w"], x)
    return y.detach(), torch.autograd.grad(y, x, s["dy"])[0]


def _own_gated(s):
    if not s["grad"]:
        return _dk().gemm_gated(s["w"], s["w2"], s["x"], act=s["act"])
    x = s["x"].detach().requires_grad_()
    h = _dk().gemm_gated(s["w"], s["w2"], x, act=s["act"])
    return h.detach(), torch.autograd.grad(h, x, s["dy"])[0]


def _turn(x, cos, sin, paired):
    """x [tokens, heads, dim] in fp32, turned by angles [tokens, 1, pairs]."""
    n = cos.shape[-1]
    y = x.clone()
    if paired:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_rotary(s):
    positions = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device="cuda"), torch.tensor(s["sections"], device="cuda"), output_size=sum(s["sections"]))
    angle = (positions.double()[axis] * s["frequency"].double()[:, None]).T[:, None]  # far positions: 64 bits
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    turned = lambda x, d: None if x is None else _turn(x.float(), cos, d * sin, s["paired"]).to(x.dtype)  # noqa: E731
    out = turned(s["q"], 1.0), turned(s["k"], 1.0)
    if not s["grad"]:
        return out
    return [x for x in out if x is not None], [turned(x, -1.0) for x in (s["dq"], s["dk"]) if x is not None]


def _plain_read(s):
    b, starts = s["block"], s["starts"].long()
    row = torch.arange(s["tokens"], device="cuda")
    of = torch.repeat_interleave(torch.arange(s["requests"], device="cuda"), starts.diff(), output_size=s["tokens"])
    place = s["lengths"].long()[of] - (starts[of + 1] - row)
    page = s["table"][of, place // b].long()
    out = []
    for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
        codes = pool.view(torch.uint8)[page, :, place % b].view(pool.dtype)
        out.append((codes.float() * scale[page][..., None]).to(DTYPES[s["dtype"]]))
    return tuple(out)


def _plain_weights(w):
    packed, scales = w
    q = torch.stack([(packed << (28 - 4 * i)) >> 28 for i in range(8)], -1).view(packed.shape[0], -1, GROUP)
    return (q.float() * scales.float()[..., None]).view(packed.shape[0], -1)


def _plain_gemm(s):
    w = _plain_weights(s["w"])
    y = (s["x"].float() @ w.T).to(s["x"].dtype)
    return (y, (s["dy"].float() @ w).to(s["x"].dtype)) if s["grad"] else y


def _plain_gated(s):
    x, w, w2 = s["x"].float(), _plain_weights(s["w"]), _plain_weights(s["w2"])
    g, u = x @ w.T, x @ w2.T
    if s["act"] == "silu":
        p, slope = g, 1.0
    else:  # gelu, its tanh form
        c = 2.0 * math.sqrt(2.0 / math.pi)
        p, slope = c * (g + 0.044715 * g ** 3), c * (1.0 + 3 * 0.044715 * g ** 2)
    gate = 1.0 / (1.0 + torch.exp(-p))
    h = (g * gate * u).to(s["x"].dtype)
    if not s["grad"]:
        return h
    dh = s["dy"].float()
    dg = dh * u * (gate + g * gate * (1.0 - gate) * slope)
    return h, (dg @ w + (dh * g * gate) @ w2).to(s["x"].dtype)


_own = {"rotary": _own_rotary, "read": _own_read, "gemm": _own_gemm, "gated": _own_gated}
_plain = {"rotary": _plain_rotary, "read": _plain_read, "gemm": _plain_gemm, "gated": _plain_gated}


# ---------------------------------------------------------------------------------------------
# In 64 bits
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"rotary": _exact_rotary, "read": _exact_read, "gemm": _exact_gemm, "gated": _exact_gated}[case["op"]](s)


def _exact_rotary(s):
    """Pairs as complex numbers, turned by exp(i angle)."""
    positions = s["positions"].view(len(s["sections"]), -1).double()
    angle = torch.cat([positions[a][:, None] * f.double() for a, f in enumerate(s["frequency"].split(s["sections"]))], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    n = angle.shape[1]

    def turned(x, by):
        if x is None:
            return None
        x = x.double()
        pairs = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) if s["paired"] else torch.complex(x[..., :n], x[..., n:2 * n])
        pairs = pairs * by
        new = torch.view_as_real(pairs).flatten(-2) if s["paired"] else torch.cat([pairs.real, pairs.imag], -1)
        return torch.cat([new, x[..., 2 * n:]], -1)

    out = turned(s["q"], turn), turned(s["k"], turn)
    if not s["grad"]:
        return out
    return [x for x in out if x is not None], [turned(x, turn.conj()) for x in (s["dq"], s["dk"]) if x is not None]


def _exact_read(s):
    out = []
    for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
        rows = []
        for r, held in enumerate(s["lengths"].tolist()):
            pages = s["table"][r, :-(-held // s["block"])].long()
            x = pool.view(torch.uint8).index_select(0, pages).view(pool.dtype).double() * scale.index_select(0, pages).double()[:, :, None, None]
            rows.append(x.permute(0, 2, 1, 3).flatten(0, 1)[:held])
        out.append(torch.cat(rows))
    return tuple(out)


def _exact_weights(w):
    packed, scales = w
    parts = []
    for i in range(8):
        nibble = torch.bitwise_right_shift(packed, 4 * i).bitwise_and(15)
        parts.append(torch.where(nibble > 7, nibble - 16, nibble).double())
    q = torch.stack(parts, 2).flatten(1)
    return q * torch.repeat_interleave(scales.double(), GROUP, 1)


def _exact_gemm(s):
    w = _exact_weights(s["w"])
    y = torch.einsum("tk,mk->tm", s["x"].double(), w)
    return (y, torch.einsum("tm,mk->tk", s["dy"].double(), w)) if s["grad"] else y


def _exact_gated(s):
    w, w2 = _exact_weights(s["w"]), _exact_weights(s["w2"])
    x = s["x"].double()
    g, u = x @ w.T, x @ w2.T
    leaf = g.clone().requires_grad_(s["grad"])
    a = torch.nn.functional.silu(leaf) if s["act"] == "silu" else torch.nn.functional.gelu(leaf, approximate="tanh")
    if not s["grad"]:
        return a * u
    dh = s["dy"].double()
    dg, = torch.autograd.grad(a, leaf, dh * u)
    return a.detach() * u, dg @ w + (dh * a.detach()) @ w2
