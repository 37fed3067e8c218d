"""Edges of the prompt operators: token tiles that end behind the last row while
memory is busy, outputs beside their inputs, rounding against the weights as
they are, gradients at the ends of the types' range, and what they refuse."""

from __future__ import annotations

import pytest
import torch

import decode_kernel as dk
from decode_kernel import _cuda
from test_prompt_ops_gpu import check_product, half_step, rows_of, sum_error, values, weights

pytestmark = pytest.mark.gpu

# Rows, outputs and width of calls whose results leave in boxes, and how many of the last token tile's boxes of 32 tokens
# no row reaches (on 148 SMs).  Odd numbers of output tiles leave a pair's second half without outputs.
BOXED = [
    ("plain", 1100, 4096, 640, 1), ("plain", 1044, 2176, 256, 2), ("plain", 1044, 2048, 1024, 3), ("plain", 4096, 4096, 4096, 4),
    ("plain", 5000, 1024, 256, 3), ("plain", 1000, 4096, 4096, 0), ("gated", 2500, 2112, 128, 1), ("gated", 300, 2816, 1024, 2), ("gated", 900, 2048, 256, 3),
    ("gated", 4096, 11008, 4096, 4), ("kept", 1300, 1088, 384, 1), ("kept", 700, 1104, 2048, 2), ("kept", 900, 2048, 256, 3),
    ("transposed", 200, 256, 18944, 1), ("transposed", 700, 1100, 2048, 2), ("transposed", 900, 512, 4224, 3), ("transposed", 1300, 256, 4096, 4),
]


@pytest.mark.parametrize("mode,T,M,K,empty", BOXED)
def test_results_in_boxes_do_not_depend_on_the_run(mode, T, M, K, empty):
    w, w2 = weights(M, K, T), weights(M, K, T + 1)
    x = rows_of(T, M if mode == "transposed" else K, torch.float16, T + 2)
    call = {"plain": lambda: (dk.gemm(*w, x),), "gated": lambda: (dk.gemm_gated(w, w2, x),), "kept": lambda: _cuda.w4a16_gemm(*w, *w2, x, 0, True),
            "transposed": lambda: (dk.gemm_t(*w, x),)}[mode]
    first = [t.clone() for t in call()]
    if mode == "plain":
        check_product(first[0], x, values(w, x.dtype, T).t(), depth=K)
    elif mode == "transposed":
        check_product(first[0], x, values(w, x.dtype), depth=M)
    elif mode == "kept":
        for got, v in zip(first[1:], (w, w2)):
            check_product(got, x, values(v, x.dtype, T, 32).t(), depth=K)
    # Copies on another stream keep the memory busy: a store takes longer to read its box.
    side, room = torch.cuda.Stream(), torch.empty(2, 1 << 27, dtype=torch.uint8, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(400):
        if i % 4 == 0:
            with torch.cuda.stream(side):
                room[1].copy_(room[0])
        for a, b in zip(first, call()):
            wrong += (a != b).sum()
    assert int(wrong) == 0
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("rows", [1, 31, 33, 64, 95, 97, 160, 191, 193, 255, 257])
@pytest.mark.parametrize("mode", ["plain", "kept", "transposed"])
def test_rows_at_the_boxes_edges(mode, rows):
    """The last row of a tile is the last that is written, for whole and odd numbers of output tiles."""
    M, K, T = (640, 512, 1344 + rows) if mode != "transposed" else (384, 640, 1344 + rows)
    w, w2 = weights(M, K, rows), weights(M, K, rows + 1)
    x = rows_of(T, M if mode == "transposed" else K, torch.bfloat16, rows + 2)
    wide = torch.full((T + 40, M if mode != "transposed" else K), 7.0, dtype=torch.bfloat16, device="cuda")
    if mode == "plain":
        check_product(dk.gemm(*w, x, out=wide[:T]), x, values(w, x.dtype, T).t(), depth=K)
    elif mode == "transposed":
        check_product(dk.gemm_t(*w, x, out=wide[:T]), x, values(w, x.dtype), depth=M)
    else:
        h, g, u = _cuda.w4a16_gemm(*w, *w2, x, 0, True, wide[:T])
        for got, v in ((g, w), (u, w2)):
            check_product(got, x, values(v, x.dtype, T, 32).t(), depth=K)
        assert torch.equal(h, dk.gemm_gated(w, w2, x))
    assert (wide[T:] == 7).all()


def test_outputs_over_inputs_are_refused_and_beside_them_are_not():
    M, K, T = 192, 256, 40
    w, w2 = weights(M, K, 1), weights(M, K, 2)
    wide = rows_of(T, 1024, torch.float16, 3)
    x, g = wide[:, :K], wide[:, :M]
    fused = torch.randn(6, 9, 64, device="cuda")
    positions, frequency = torch.arange(6, device="cuda"), torch.rand(32, device="cuda")
    cache = dk.PagedCache8(4, 16, 2, 64)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lengths, starts = ints([[0, 1]]), ints([20]), ints([0, 20])
    rows = torch.zeros(41, 2, 64, dtype=torch.float16, device="cuda")
    read = lambda k, v: dk.cache_read(cache, table, lengths, starts, 20, out=(k, v))  # noqa: E731
    words = lambda t, n: t.view(torch.float16).view(-1)[:n]  # noqa: E731
    bad = {
        "gemm": lambda: dk.gemm(*w, x, out=wide[:, K - 64:K - 64 + M]), "gemm, few rows": lambda: dk.gemm(*w, x[:4], out=wide[:4, 8:8 + M]),
        "gemm, rows": lambda: dk.gemm(*w, x[:20], out=wide[19:39, :M]), "gated": lambda: dk.gemm_gated(w, w2, x, out=wide[:, K - 1:K - 1 + M]),
        "gemm_t": lambda: dk.gemm_t(*w, g, out=wide[:, M - 8:M - 8 + K]), "gemm_t, the second rows": lambda: _cuda.w4a16_gemm_t(*w, *w2, wide[:, 512:512 + M], g, wide[:, M - 8:M - 8 + K]),
        "packed": lambda: dk.gemm(*w, x, out=words(w[0], T * M).view(T, M)), "scales": lambda: dk.gemm(*w, x[:2], out=words(w[1], 2 * M).view(2, M)),
        "up": lambda: dk.gemm_gated(w, w2, x, out=words(w2[0], T * M).view(T, M)), "packed, transposed": lambda: dk.gemm_t(*w, g, out=words(w[0], T * K).view(T, K)),
        "heads": lambda: dk.rotary(fused[:, :4], fused[:, 3:6], positions, frequency, inplace=True),
        "frequency": lambda: dk.rotary(fused[:, :4], None, positions, fused.view(-1)[:32], inplace=True),
        "k and v": lambda: read(rows[:20], rows[19:39]), "pool": lambda: read(cache.k.view(-1).view(torch.float16).view(-1, 2, 64)[:20], rows[:20]),
        "heads of k and v": lambda: read(rows.view(41, 128)[:20].view(20, 2, 64), rows.view(-1)[64:64 + 20 * 128].view(20, 2, 64)),
    }
    before = [t.clone() for t in (wide, *w, *w2, fused, cache.k, rows)]
    for name, call in bad.items():
        with pytest.raises(RuntimeError, match="overlap"):
            call()
            pytest.fail(f"{name} was not refused")
    assert all(torch.equal(a, b) for a, b in zip(before, (wide, *w, *w2, fused, cache.k, rows)))
    # Beside one another in the same memory.
    want = dk.gemm(*w, x)
    assert torch.equal(dk.gemm(*w, x, out=wide[:, K:K + M]), want) and torch.equal(wide[:, K:K + M], want)
    want = dk.gemm_gated(w, w2, x)
    assert torch.equal(dk.gemm_gated(w, w2, x, out=wide[:, K + 1:K + 1 + M]), want)
    assert torch.equal(dk.gemm(*w, x[::2], out=wide[1::2, :M]), dk.gemm(*w, before[0][::2, :K]))
    q, k = fused[:, :4], fused[:, 4:6]
    want = dk.rotary(q, k, positions, frequency)
    assert all(torch.equal(a, b) for a, b in zip(dk.rotary(q, k, positions, frequency, inplace=True), want))
    both = torch.zeros(20, 2, 2, 64, dtype=torch.float16, device="cuda")
    want = dk.cache_read(cache, table, lengths, starts, 20)
    assert all(torch.equal(a, b) for a, b in zip(read(both[:, 0], both[:, 1]), want))


def test_every_second_head_is_turned_in_place():
    """Heads that lie two apart, of an odd number: a token's last one ends before the next token's first."""
    positions, frequency = torch.arange(6, device="cuda"), torch.rand(32, device="cuda")
    fused = torch.randn(6, 9, 64, device="cuda")
    for base in (fused, fused.transpose(0, 1).contiguous().transpose(0, 1)):
        q, k = base[:, ::2], base[:, 1::2]
        want = [t.clone() for t in dk.rotary(q, k, positions, frequency)]
        assert all(torch.equal(a, b) for a, b in zip(dk.rotary(q, k, positions, frequency, inplace=True), want))
    alike = torch.as_strided(fused, (6, 3, 64), (160, 64, 1))
    with pytest.raises(RuntimeError, match="overlap themselves"):  # a token's last head begins before the next token's first
        dk.rotary(alike, None, positions, frequency, inplace=True)


def test_outputs_of_a_graph_are_refused_but_under_no_grad():
    w = weights(128, 256, 1)
    x = rows_of(20, 256, torch.float16, 3)
    leaf = torch.zeros(20, 128, dtype=torch.float16, device="cuda", requires_grad=True)
    cache = dk.PagedCache8(4, 16, 2, 64)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    kv = [torch.zeros(20, 2, 64, dtype=torch.float16, device="cuda", requires_grad=i == 1) for i in range(2)]
    calls = [lambda: dk.gemm(*w, x, out=leaf), lambda: dk.gemm_gated(w, w, x, out=leaf * 2), lambda: dk.cache_read(cache, ints([[0, 1]]), ints([20]), ints([0, 20]), 20, out=kv)]
    for call in calls:
        with pytest.raises(RuntimeError, match="out takes no part"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(leaf.detach(), dk.gemm(*w, x))


def test_calls_on_threads_of_their_own():
    """A thread's first CUDA call may be one of the products, as in autograd's threads: nothing has made a context current there."""
    from concurrent.futures import ThreadPoolExecutor

    w, w2 = weights(128, 256, 1), weights(128, 256, 2)
    large = weights(16384, 256, 3)
    xs = [rows_of(T, 256, torch.float16, T) for T in (1, 4, 12, 20, 300)]
    gs = [rows_of(T, 128, torch.float16, T) for T in (4, 20, 300)]
    calls = [lambda x=x: dk.gemm(*w, x) for x in xs] + [lambda x=x: dk.gemm_gated(w, w2, x) for x in xs] + [lambda g=g: dk.gemm_t(*w, g) for g in gs]
    calls += [lambda x=x: dk.gemv(*large, x) for x in xs[:4]]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    for call, expected in zip(calls, want):
        with ThreadPoolExecutor(1) as thread:
            got = thread.submit(call).result()
        torch.cuda.synchronize()
        assert torch.equal(got, expected)


def test_the_linear_layers_gradient_compiled_and_twice():
    layer = dk.W4A16Linear(*weights(128, 256, 1))
    x = rows_of(20, 256, torch.float16, 3).requires_grad_()
    dy = rows_of(20, 128, torch.float16, 4).requires_grad_()
    want, = torch.autograd.grad(layer(x), x, dy)
    assert torch.equal(want, dk.gemm_t(layer.packed, layer.scales, dy.detach()))
    got, = torch.autograd.grad(torch.compile(layer, backend="aot_eager", fullgraph=True)(x), x, dy)
    assert torch.equal(got, want)
    once, = torch.autograd.grad(layer(x), x, dy, create_graph=True)
    twice, = torch.autograd.grad(once, dy, x.detach())
    assert torch.equal(twice, dk.gemm(layer.packed, layer.scales, x.detach()))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_hooks_and_adapters_of_a_gated_blocks_layers_count(act):
    class Adapter(torch.nn.Module):
        def __init__(self, layer):
            super().__init__()
            self.layer, self.more = layer, torch.nn.Parameter(torch.full((layer.out_features,), 0.5, dtype=torch.float16, device="cuda"))

        def forward(self, x):
            return self.layer(x) + self.more

    def block():
        return dk.W4A16GatedMLP(*(dk.W4A16Linear(*weights(m, k, s)) for m, k, s in ((384, 256, 1), (384, 256, 2), (256, 384, 3))), act=act)

    class Named(dk.W4A16Linear):
        pass

    class Negative(dk.W4A16Linear):
        def forward(self, x):
            return -super().forward(x)

    x = rows_of(20, 256, torch.float16, 4)
    bare = block()
    want = bare(x)
    named, negative = block(), block()
    named.up = Named(bare.up.packed, bare.up.scales)  # a layer's own product under another name
    assert torch.equal(named(x), want)
    negative.down = Negative(bare.down.packed, bare.down.scales)
    assert torch.equal(negative(x), -bare.down(dk.gemm_gated((bare.gate.packed, bare.gate.scales), (bare.up.packed, bare.up.scales), x, act=act)))
    f = torch.nn.functional.silu if act == "silu" else lambda g: torch.nn.functional.gelu(g, approximate="tanh")
    for name in ("gate", "up", "down"):
        mlp, seen = block(), []
        handle = getattr(mlp, name).register_forward_hook(lambda m, args, out: seen.append(out.shape) or out * 0)
        assert (mlp(x) == 0).all() and len(seen) == 1
        handle.remove()
        assert torch.equal(mlp(x), want)
        adapter = Adapter(getattr(mlp, name))
        setattr(mlp, name, adapter)
        got = mlp(x)
        parts = {n: getattr(mlp, n) for n in ("gate", "up", "down")}
        if name == "down":
            h = dk.gemm_gated((bare.gate.packed, bare.gate.scales), (bare.up.packed, bare.up.scales), x, act=act)
            assert torch.equal(got, parts["down"](h))
        else:
            h = f(parts["gate"](x)) * parts["up"](x)
            assert torch.equal(got, dk.gemm(bare.down.packed, bare.down.scales, h))
        got.float().square().mean().backward()
        assert adapter.more.grad.abs().max() > 0


@pytest.mark.parametrize("act", [0, 1], ids=["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_gradients_of_projections_at_the_ends_of_the_range(dtype, act):
    """act' is 1 far above zero and 0 far below, also where the kept projection has become infinite or its square would."""
    far = torch.tensor([1e4, 6e4, 1e20, 3e38, float("inf")], device="cuda").to(dtype)
    g = torch.cat([far, -far]).repeat(3, 1)
    u = torch.tensor([[0.5], [-2.0], [0.0]], device="cuda").expand_as(g).to(dtype).contiguous()
    dh = torch.tensor([[1.0], [0.25], [-3.0]], device="cuda").expand_as(g).to(dtype).contiguous()
    dg, du = _cuda.gated_grad(dh, g, u, act)
    high, low = slice(0, 5), slice(5, 10)
    assert torch.equal(dg[:, high], (dh * u)[:, high]) and (dg[:, low] == 0).all()
    assert torch.equal(du[:, high], (dh.float() * g.float())[:, high].to(dtype)) and (du[:, low] == 0).all()
    nan = torch.full_like(g, float("nan"))
    assert all(t.isnan().all() for t in _cuda.gated_grad(dh, nan, u, act) + _cuda.gated_grad(nan, g, u, act))


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_where_gates_are_shut_past_the_range(T, act):
    """Gates of -358400, which fp16 does not hold: the block's outputs are zeros and so are its gradients."""
    gate = torch.full((64, 32), -0x66666667, dtype=torch.int32, device="cuda"), torch.ones((64, 2), dtype=torch.float16, device="cuda")  # every code -7
    up = weights(64, 256, 5)
    x = torch.full((T, 256), 200.0, dtype=torch.float16, device="cuda", requires_grad=True)
    h = dk.gemm_gated(gate, up, x, act=act)
    dx, = torch.autograd.grad(h, x, torch.ones_like(h))
    assert (h == 0).all() and (dx == 0).all()


def against_weights_as_they_are(x, w, depth):
    """(x @ w in 64 bits, what a sum of rounded weights may be off): each weight is half a step of the rows' type off, or half of
    fp16's smallest step, and the sum has its own error."""
    total = x.double().abs() @ w.abs()
    smallest = 2.0 ** -25 * x.double().abs().sum(-1, keepdim=True) if x.dtype == torch.float16 else 0.0
    return x.double() @ w, total * half_step(x.dtype) + smallest + sum_error(total, depth)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,M,K", [(17, 4096, 1408), (40, 1000, 384), (333, 1000, 2816), (1044, 640, 512)])
def test_products_against_the_weights_as_they_are(T, M, K, dtype):
    w, w2 = weights(M, K, T), weights(M, K, T + 1)
    real, real2 = (values(v, torch.float64, 0) for v in (w, w2))
    x, g = rows_of(T, K, dtype, T + 2), rows_of(T, M, dtype, T + 3)
    half = half_step(dtype)
    for got, rows, v, depth in ((dk.gemm(*w, x), x, real.t(), K), (dk.gemm_t(*w, g), g, real, M)):
        want, off = against_weights_as_they_are(rows, v, depth)
        assert ((got.double() - want).abs() <= want.abs() * half + off * (1 + half) + 2.0 ** -25).all()
        # Roundings that go either way add up as their root: the whole stays below four times the result's own rounding.
        assert (got.double() - want).norm() <= 4 * half * want.norm()
    (a, ea), (b, eb) = (against_weights_as_they_are(x, v.t(), K) for v in (real, real2))
    s, p = torch.sigmoid(a), a.abs()
    want = a * s * b
    # |act'| <= 1.13; the sigmoid is 2^-21 off times its argument.
    off = want.abs() * (2 + p) * 2.0 ** -21 + 1.13 * ea * (b.abs() + eb) + (a * s).abs() * eb
    got = dk.gemm_gated(w, w2, x)
    assert ((got.double() - want).abs() <= want.abs() * half + off * (1 + half) + 2.0 ** -25).all()


def test_boxed_results_on_streams_and_in_graphs():
    M, K = 704, 1024
    w, w2 = weights(M, K, 60), weights(M, K, 61)
    xs = [rows_of(T, K, torch.float16, 62 + T) for T in (300, 1044, 2500)]
    call = lambda x: (dk.gemm(*w, x), dk.gemm_gated(w, w2, x), dk.gemm_t(*w, dk.gemm(*w, x)))  # noqa: E731
    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[] for _ in xs]
    for _ in range(10):
        for s, x, out in zip(streams, xs, got):
            with torch.cuda.stream(s):
                out.append(call(x))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for out in b for p, q in zip(a, out))
    held = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [call(x) for x in held]
    for scale in (1.0, -0.5):
        for x, h in zip(xs, held):
            h.copy_(x * scale)
        graph.replay()
        for h, b in zip(held, out):
            assert all(torch.equal(p, q) for p, q in zip(call(h), b))
