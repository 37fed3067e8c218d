"""The prompt operators against plain computations in 64 bits: products of many
rows through 4-bit weights, the gated pair, their gradients, rotary positions,
and the cache read back."""

from __future__ import annotations

import math

import pytest
import torch

import decode_kernel as dk
from decode_kernel import capi

pytestmark = pytest.mark.gpu

HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weights(M, K, seed):
    """Every code of -8..7, scales of about the size that keeps products near 1."""
    g = gen(seed)
    packed = torch.randint(-2 ** 31, 2 ** 31, (M, K // 8), generator=g, device="cuda").to(torch.int32)
    scales = (torch.rand((M, K // 128), generator=g, device="cuda") + 0.5) * (K ** -0.5 / 4.6)
    return packed, scales.half()


FEW, FEW_OF_PAIR = 16, 32  # rows up to which the products take the weights as they are


def values(w, dtype, rows=1000, few=FEW):
    """The weights as the products use them: q * scale, rounded once to the rows' type where there are many."""
    packed, scales = w
    q = torch.stack([(packed << (28 - 4 * i)) >> 28 for i in range(8)], -1).reshape(packed.shape[0], -1)
    v = q.float() * scales.float().repeat_interleave(128, 1)
    return (v.to(dtype) if rows > few else v).double()


def rows_of(T, n, dtype, seed):
    g = gen(seed)
    x = torch.randn((T, n), generator=g, device="cuda") * torch.exp(0.5 * torch.randn((T, 1), generator=g, device="cuda"))
    return x.to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sum_error(total, depth):
    """Bound on an fp32 sum of `depth` products whose magnitudes add up to `total`: the products are exact in the tensor
    cores, sums are taken 16 products at a time and may be cut off instead of rounded (2^-23 of what is there), and up to
    16 partial sums of a split depth are added at the end."""
    return total * (depth / 16 + 16) * 2.0 ** -23


def lost(x, w, few=FEW):
    """What few rows lose of values that are small beside their row's largest in the group: 2^-25 of that (fp16) or 2^-21 (bf16)."""
    if x.shape[0] > few or x.shape[1] % 128:
        return 0.0
    most = x.double().abs().unflatten(1, (-1, 128)).amax(-1, keepdim=True).expand(-1, -1, 128).flatten(1)
    return most @ w.abs() * (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -21)


def check_product(y, x, w, *, depth):
    """y = x @ w: rounded once, beside the sum's own error."""
    want = x.double() @ w
    bound = want.abs() * half_step(y.dtype) + sum_error(x.double().abs() @ w.abs(), depth) + lost(x, w) + 2.0 ** -25  # fp16's smallest half step
    off = (y.double() - want).abs()
    assert y.isfinite().all()
    assert (off <= bound).all(), float((off / bound).max())


# rows, M, K: one row, tiles' edges and their neighbours, odd outputs, one group, many
SHAPES = [(1, 1, 128), (1, 4096, 4096), (2, 100, 256), (7, 129, 384), (8, 64, 2048), (9, 1000, 128), (16, 128, 4096), (17, 4096, 1408), (31, 200, 1024),
          (33, 255, 640), (64, 511, 512), (65, 1500, 2816), (127, 257, 256), (129, 130, 1024), (255, 2816, 1024), (257, 384, 2816), (300, 4100, 512),
          (513, 1000, 384), (1000, 640, 1024), (1537, 2050, 256)]


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("T,M,K", SHAPES)
def test_gemm(T, M, K, dtype):
    w = weights(M, K, T + M)
    x = rows_of(T, K, HALF[dtype], K + T)
    check_product(dk.gemm(*w, x), x, values(w, x.dtype, T).t(), depth=K)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("T,M,K", SHAPES)
def test_gemm_t(T, M, K, dtype):
    w = weights(M, K, T + M + 1)
    g = rows_of(T, M, HALF[dtype], K + T + 1)
    check_product(dk.gemm_t(*w, g), g, values(w, g.dtype), depth=M)


def act_parts(g, act):
    """act(g), act'(g), and the sigmoid's argument."""
    if act == "silu":
        p, slope = g, torch.ones_like(g)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        p, slope = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
    s = torch.sigmoid(p)
    return g * s, s + g * s * (1 - s) * slope, p


def check_gated(h, x, wg, wu, act, depth):
    """|act'| <= 1.13 for both forms; the sigmoid's exponential is 2^-21 off times its argument."""
    xd = x.double()
    g, u = xd @ wg.t(), xd @ wu.t()
    eg, eu = (sum_error(xd.abs() @ w.abs().t(), depth) + lost(x, w.t(), FEW_OF_PAIR) for w in (wg, wu))
    a, _, p = act_parts(g, act)
    want = a * u
    bound = want.abs() * (half_step(h.dtype) + (2 + p.abs()) * 2.0 ** -21) + 1.2 * eg * (u.abs() + eu) + a.abs() * eu + 2.0 ** -25
    off = (h.double() - want).abs()
    assert h.isfinite().all()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("dtype,act", [("fp16", "silu"), ("bf16", "gelu"), ("bf16", "silu"), ("fp16", "gelu")])
@pytest.mark.parametrize("T,M,K", SHAPES)
def test_gemm_gated(T, M, K, dtype, act):
    wg, wu = weights(M, K, T + M + 2), weights(M, K, T + M + 3)
    x = rows_of(T, K, HALF[dtype], K + T + 2)
    check_gated(dk.gemm_gated(wg, wu, x, act=act), x, values(wg, x.dtype, T, FEW_OF_PAIR), values(wu, x.dtype, T, FEW_OF_PAIR), act, K)


def gated_gradient(x, dh, wg, wu, act, depth, M):
    """(dx, its bound): the projections are kept rounded, dg and du are rounded, then summed over 2 M products.
    |act''| <= 1.2, |act'| <= 1.2 and |act| <= |g|.  wg and wu: as the gradient's product uses them, rounded; the projections
    of few rows use them unrounded, which moves each product by half a step of its weight."""
    e = half_step(x.dtype)
    xd, d = x.double(), dh.double()
    g, u = xd @ wg.t(), xd @ wu.t()
    few = e if len(x) <= FEW_OF_PAIR else 0.0
    eg, eu = (p.abs() * e + few * (xd.abs() @ w.abs().t()) + sum_error(xd.abs() @ w.abs().t(), depth) + lost(x, w.t(), FEW_OF_PAIR) for p, w in ((g, wg), (u, wu)))
    a, slope, p = act_parts(g, act)
    dg, du = d * u * slope, d * a
    more = (2 + p.abs()) * 2.0 ** -20 + e
    edg = dg.abs() * more + d.abs() * (1.2 * u.abs() * eg + 1.2 * eu + 1.2 * eg * eu) + 2.0 ** -25
    edu = du.abs() * more + d.abs() * 1.2 * eg + 2.0 ** -25
    dx = dg @ wg + du @ wu
    bound = dx.abs() * e + edg @ wg.abs() + edu @ wu.abs() + sum_error((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs(), 2 * M) + 2.0 ** -25
    return dx, bound


@pytest.mark.parametrize("dtype,act", [("fp16", "silu"), ("bf16", "gelu")])
@pytest.mark.parametrize("T,M,K", [(1, 64, 128), (5, 100, 256), (40, 1001, 384), (130, 256, 1024), (300, 2816, 1024), (600, 520, 640)])
def test_gemm_gated_gradient(T, M, K, dtype, act):
    wg, wu = weights(M, K, T + M + 4), weights(M, K, T + M + 5)
    x = rows_of(T, K, HALF[dtype], K + T + 4).requires_grad_()
    dh = rows_of(T, M, HALF[dtype], K + T + 5)
    h = dk.gemm_gated(wg, wu, x, act=act)
    dx, = torch.autograd.grad(h, x, dh)
    vg, vu = values(wg, x.dtype), values(wu, x.dtype)
    check_gated(h.detach(), x.detach(), values(wg, x.dtype, T, FEW_OF_PAIR), values(wu, x.dtype, T, FEW_OF_PAIR), act, K)
    want, bound = gated_gradient(x.detach(), dh, vg, vu, act, K, M)
    off = (dx.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    # Against differences of the formula in 64 bits, along a direction: the step's error is h^2 |f'''| / 6.
    v = torch.randn((T, K), generator=gen(9), device="cuda").double()
    step = 1e-4
    f = lambda z: (act_parts(z @ vg.t(), act)[0] * (z @ vu.t()) * dh.double()).sum()  # noqa: E731
    xd = x.detach().double()
    slope = (f(xd + step * v) - f(xd - step * v)) / (2 * step)
    assert abs(float((dx.double() * v).sum() - slope)) <= float((bound * v.abs()).sum()) + 1e-3 * abs(float(slope)) + 1e-3


@pytest.mark.parametrize("dtype", list(HALF))
def test_gradient_of_gemm_and_linear(dtype):
    T, M, K = 37, 500, 640
    w = weights(M, K, 6)
    v = values(w, HALF[dtype])
    dy = rows_of(T, M, HALF[dtype], 7)
    x = rows_of(T, K, HALF[dtype], 8).requires_grad_()
    dx, = torch.autograd.grad(dk.gemm(*w, x), x, dy)
    check_product(dx, dy, v, depth=M)
    g = dy.clone().requires_grad_()
    back, = torch.autograd.grad(dk.gemm_t(*w, g), g, x.detach())
    check_product(back, x.detach(), values(w, x.dtype, T).t(), depth=K)
    # The operators are linear: a gradient's gradient is the product itself.
    seed = dy.clone().requires_grad_()
    once, = torch.autograd.grad(dk.gemm(*w, x), x, seed, create_graph=True)
    twice, = torch.autograd.grad(once, seed, x.detach())
    assert torch.equal(twice, dk.gemm(*w, x.detach()))
    if dtype == "fp16":
        layer = dk.W4A16Linear(*w)
        y = layer(x)
        assert torch.equal(y, dk.w4a16_linear(x.detach(), *w, reuse_weights=False))  # the forward pass is what it was
        dx2, = torch.autograd.grad(y, x, dy)
        assert torch.equal(dx, dx2)


def test_gradients_of_any_layout():
    """Gradients that come broadcast, transposed or with more dimensions, of inputs that are views."""
    M, K, T = 120, 256, 24
    w, w2 = weights(M, K, 14), weights(M, K, 15)
    base = rows_of(T, 2 * K, torch.float16, 16)
    for view in (lambda b: b[:, :K], lambda b: b[:, 8:K + 8].reshape(2, T // 2, K), lambda b: b[:1, :K].expand(T, K)):
        for call in (lambda x: dk.gemm(*w, x), lambda x: dk.gemm_gated(w, w2, x)):
            leaf = base.clone().requires_grad_()
            x = view(leaf)
            call(x).float().sum().backward()  # the gradient of the output is one number, broadcast
            alone = x.detach().clone().requires_grad_()
            dx, = torch.autograd.grad(call(alone), alone, torch.ones(*alone.shape[:-1], M, dtype=torch.float16, device="cuda"))
            want = base.clone().requires_grad_()
            view(want).backward(dx)
            assert torch.equal(leaf.grad, want.grad)
    g = rows_of(M, T, torch.float16, 17).t()
    x = rows_of(T, K, torch.float16, 18).requires_grad_()
    dx, = torch.autograd.grad(dk.gemm(*w, x), x, g)
    assert torch.equal(dx, dk.gemm_t(*w, g.contiguous()))


def test_gated_mlp_module_runs_and_trains():
    dim, hidden = 256, 384
    g = gen(10)
    layers = [dk.W4A16Linear(*weights(m, k, s)) for m, k, s in ((hidden, dim, 11), (hidden, dim, 12), (dim, hidden, 13))]
    mlp = dk.W4A16GatedMLP(*layers)
    x = torch.randn((2, 5, dim), generator=g, device="cuda").half().requires_grad_()
    y = mlp(x)
    pairs = [(m.packed, m.scales) for m in layers]
    h = dk.gemm_gated(pairs[0], pairs[1], x.detach())
    assert y.shape == x.shape and torch.equal(y, dk.gemm(*pairs[2], h))
    y.float().square().mean().backward()
    assert x.grad.shape == x.shape and x.grad.isfinite().all() and x.grad.abs().max() > 0


# ---------------------------------------------------------------------------
# Shapes, strides, places
# ---------------------------------------------------------------------------


def test_products_of_views():
    M, K, T = 200, 256, 30
    w = weights(M, K, 20)
    v = values(w, torch.float16, T)
    wide = rows_of(T, 3 * K + 8, torch.float16, 21)
    base = rows_of(1, K, torch.float16, 22)
    for x in (wide[:, K:2 * K], wide[:, 1:K + 1], wide[:, :K][::2], wide.t()[:K].t(), rows_of(K, T, torch.float16, 23).t(), base.expand(T, K),
              wide[:, 8:K + 8].flip(0)):
        check_product(dk.gemm(*w, x), x, values(w, x.dtype, len(x)).t(), depth=K)
    g3 = rows_of(T, M, torch.float16, 24).view(2, 15, M)
    assert torch.equal(dk.gemm_t(*w, g3), dk.gemm_t(*w, g3.reshape(T, M)).view(2, 15, K))
    assert dk.gemm(*w, base[0]).shape == (M,)
    assert torch.equal(dk.gemm(*w, base[0]), dk.gemm(*w, base)[0])
    assert dk.gemm(*w, base[:0]).shape == (0, M) and dk.gemm_t(*w, base[:0, :M]).shape == (0, K)
    # Outputs given: rows apart, and what lies between them stays.
    out = torch.full((T, M + 5), 7.0, dtype=torch.float16, device="cuda")
    x = wide[:, :K]
    assert dk.gemm(*w, x, out=out[:, 2:M + 2]).data_ptr() == out[:, 2:].data_ptr()
    assert torch.equal(out[:, 2:M + 2], dk.gemm(*w, x)) and (out[:, :2] == 7).all() and (out[:, M + 2:] == 7).all()
    out = torch.full((T, K + 3), 7.0, dtype=torch.float16, device="cuda")
    g = rows_of(T, M, torch.float16, 25)
    dk.gemm_t(*w, g, out=out[:, :K])
    assert torch.equal(out[:, :K], dk.gemm_t(*w, g)) and (out[:, K:] == 7).all()
    out = torch.full((T, M + 5), 7.0, dtype=torch.float16, device="cuda")
    dk.gemm_gated(w, w, x, out=out[:, :M])
    assert torch.equal(out[:, :M], dk.gemm_gated(w, w, x)) and (out[:, M:] == 7).all()


def test_packed_that_begins_off_16_bytes():
    M, K = 96, 256
    packed, scales = weights(M, K, 30)
    room = torch.empty(M * K // 8 + 1, dtype=torch.int32, device="cuda")
    shifted = room[1:].view(M, K // 8).copy_(packed)
    x = rows_of(20, K, torch.bfloat16, 31)
    assert torch.equal(dk.gemm(shifted, scales, x), dk.gemm(packed, scales, x))


@pytest.mark.parametrize("T", [3, 12, 24, 40, 300])
def test_rows_with_infinities_and_nan_stay_to_themselves(T):
    M, K = 300, 512
    w, w2 = weights(M, K, 40), weights(M, K, 41)
    x = rows_of(T, K, torch.float16, 42)
    clean = [dk.gemm(*w, x), dk.gemm_gated(w, w2, x)]
    x[1, 7] = math.nan
    x[2, 100] = math.inf
    dirty = [dk.gemm(*w, x), dk.gemm_gated(w, w2, x)]
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    for a, b in zip(clean, dirty):
        assert torch.equal(a[keep], b[keep]) and b[1].isnan().all()
    assert not dirty[0][2].isfinite().any()


@pytest.mark.parametrize("T", [1, 12, 50, 100, 200, 700])
def test_results_do_not_depend_on_the_run(T):
    M, K = 1100, 2048
    w, w2 = weights(M, K, 50), weights(M, K, 51)
    x = rows_of(T, K, torch.float16, 52)
    g = rows_of(T, M, torch.float16, 53)
    first = [dk.gemm(*w, x), dk.gemm_gated(w, w2, x), dk.gemm_t(*w, g)]
    for _ in range(40):
        for a, b in zip(first, (dk.gemm(*w, x), dk.gemm_gated(w, w2, x), dk.gemm_t(*w, g))):
            assert torch.equal(a, b)


def test_streams_and_graphs():
    M, K = 700, 1024
    w, w2 = weights(M, K, 60), weights(M, K, 61)
    xs = [rows_of(T, K, torch.float16, 62 + T) for T in (5, 100, 400)]
    call = lambda x: (dk.gemm(*w, x), dk.gemm_gated(w, w2, x), dk.gemm_t(*w, dk.gemm(*w, x)))  # noqa: E731
    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            for _ in range(4):
                out = call(x)
            got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    held = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [call(x) for x in held]
    for scale in (1.0, 0.5, -2.0):
        for x, h in zip(xs, held):
            h.copy_(x * scale)
        graph.replay()
        for h, b in zip(held, got):
            assert all(torch.equal(p, q) for p, q in zip(call(h), b))


def test_captured_training_step():
    """Forward and backward of the gated block and the rotary positions in one graph, replayed with new inputs."""
    M, K, T = 300, 256, 50
    wg, wu, wd = weights(M, K, 70), weights(M, K, 71), weights(K, M // 128 * 128 + 128, 72)
    wd = (wd[0][:, :256 // 8].contiguous(), wd[1][:, :2].contiguous())
    freq = torch.rand(16, device="cuda")
    pos = torch.arange(T, device="cuda")
    x = rows_of(T, K, torch.float16, 73)
    dy = rows_of(T, M, torch.float16, 74)

    def step(x):
        leaf = x.detach().requires_grad_()
        q, _ = dk.rotary(leaf.view(T, 8, 32), None, pos, freq)
        h = dk.gemm_gated(wg, wu, dk.gemm(*wd, q.reshape(T, K)))
        return torch.autograd.grad(h, leaf, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(held)
    for scale in (1.0, 0.25):
        held.copy_(x * scale)
        graph.replay()
        assert torch.equal(got, step(held))


def test_product_refusals():
    M, K = 64, 256
    packed, scales = weights(M, K, 80)
    x = rows_of(4, K, torch.float16, 81)
    bad = [
        lambda: dk.gemm(packed, scales, x.float()), lambda: dk.gemm(packed, scales, x[:, :128]), lambda: dk.gemm(packed.long(), scales, x),
        lambda: dk.gemm(packed, scales.float(), x), lambda: dk.gemm(packed, scales[:, :1], x), lambda: dk.gemm(packed[:, ::2], scales, x),
        lambda: dk.gemm(packed[:, :24], scales, x), lambda: dk.gemm(packed, scales, x.cpu()), lambda: dk.gemm(packed.cpu(), scales, x),
        lambda: dk.gemm(packed, scales, x, out=torch.empty(4, M + 1, dtype=torch.float16, device="cuda")),
        lambda: dk.gemm(packed, scales, x, out=torch.empty(M, 4, dtype=torch.float16, device="cuda").t()),
        lambda: dk.gemm(packed, scales, x, out=torch.empty(4, M, dtype=torch.bfloat16, device="cuda")),
        lambda: dk.gemm_gated((packed, scales), (packed[:32], scales[:32]), x), lambda: dk.gemm_t(packed, scales, x),
        lambda: dk.gemm(packed, scales, x.clone().requires_grad_(), out=torch.empty(4, M, dtype=torch.float16, device="cuda")),
        lambda: dk.gemm(packed, scales, torch.zeros((), dtype=torch.float16, device="cuda")),
        lambda: dk.gemm(packed, scales, x, out=x.view(-1)[:4 * M].view(4, M)),
        lambda: dk.gemm(packed, scales.clone().requires_grad_(), x), lambda: dk.gemm_gated((packed, scales), (packed, scales.clone().requires_grad_()), x),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------


def turned(x, positions, frequency, sections, paired, sign=1.0):
    """(the turned values in 64 bits, what they may be off): sines and cosines of an angle in turns are 2^-21 right, and the angle itself
    2^-52 of its turns."""
    positions = positions.reshape(-1, x.shape[0]).double()
    n = frequency.shape[0]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = (positions[axis.cuda()] * frequency.double()[:, None]).t()[:, None] * sign
    x = x.double()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if paired else (x[..., :n], x[..., n:2 * n])
    want, off = x.clone(), torch.zeros_like(x)
    new = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    error = (a.abs() + b.abs()) * (2.0 ** -21 + angle.abs() * 2.0 ** -52)
    for i in range(2):
        at = slice(i, 2 * n, 2) if paired else slice(i * n, i * n + n)
        want[..., at], off[..., at] = new[i], error
    return want, off


def check_turned(y, x, positions, frequency, sections, paired, sign=1.0):
    want, off = turned(x, positions, frequency, sections, paired, sign)
    bound = want.abs() * half_step(y.dtype) + off + 2.0 ** -25
    assert ((y.double() - want).abs() <= bound).all(), float(((y.double() - want).abs() / bound).max())
    n = 2 * frequency.shape[0]
    assert torch.equal(y[..., n:], x[..., n:])


ROTARY = [  # tokens, q heads, kv heads, dim, sections, paired, dtype
    (1, 32, 8, 128, [64], False, "fp16"), (1, 1, 0, 2, [1], False, "fp32"), (3, 7, 1, 256, [128], True, "bf16"), (33, 5, 2, 80, [13, 19], False, "fp16"),
    (100, 12, 12, 64, [8, 12, 12], True, "bf16"), (257, 16, 16, 80, [20], False, "fp32"), (65, 3, 3, 33, [5, 0, 11], True, "fp32"),
    (65, 3, 3, 35, [16], True, "fp16"), (40, 2, 1, 34, [17], False, "bf16"), (1000, 32, 8, 128, [16, 24, 24], False, "bf16"),
    (700, 1, 0, 128, [64], False, "fp16"), (20, 2, 2, 1024, [100, 200, 12, 200], False, "fp16"), (4099, 4, 1, 96, [48], True, "fp16"),
    (50, 3, 1, 66, [31], True, "bf16"), (64, 600, 8, 64, [32], False, "fp16"),
]
TYPES = dict(HALF, fp32=torch.float32)


def rotary_case(tokens, heads, kv, dim, sections, paired, dtype, seed=0):
    g = gen(seed + tokens)
    make = lambda h: torch.randn((tokens, h, dim), generator=g, device="cuda").to(TYPES[dtype]) if h else None  # noqa: E731
    positions = torch.randint(0, 200000, (len(sections), tokens), generator=g, device="cuda", dtype=torch.int32 if tokens % 2 else torch.int64)
    frequency = torch.rand(sum(sections), generator=g, device="cuda") ** 4
    return make(heads), make(kv), positions, frequency


@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary(case):
    tokens, heads, kv, dim, sections, paired, dtype = case
    q, k, positions, frequency = rotary_case(*case)
    given = positions if len(sections) > 1 else positions[0]
    for inverse in (False, True):
        qo, ko = dk.rotary(q, k, given, frequency, sections=sections if len(sections) > 1 else None, paired=paired, inverse=inverse)
        check_turned(qo, q, positions, frequency, sections, paired, -1.0 if inverse else 1.0)
        if kv:
            check_turned(ko, k, positions, frequency, sections, paired, -1.0 if inverse else 1.0)
        else:
            assert ko is None
    # In place, and as parts of one projection whose rows hold more.
    fused = torch.randn((tokens, heads + kv + 1, dim), generator=gen(1), device="cuda").to(q.dtype)
    before = fused.clone()
    a, b = fused[:, :heads], fused[:, heads:heads + kv] if kv else None
    dk.rotary(a, b, positions, frequency, sections=sections, paired=paired, inplace=True)
    check_turned(fused[:, :heads + kv], before[:, :heads + kv], positions, frequency, sections, paired)
    assert torch.equal(fused[:, heads + kv:], before[:, heads + kv:])
    assert torch.equal(dk.rotary(before[:, :heads], None, positions, frequency, sections=sections, paired=paired)[0], fused[:, :heads])


@pytest.mark.parametrize("case", [ROTARY[i] for i in (3, 4, 5, 7, 9)], ids=str)
def test_rotary_gradient(case):
    tokens, heads, kv, dim, sections, paired, dtype = case
    q, k, positions, frequency = rotary_case(*case, seed=5)
    q.requires_grad_(), k.requires_grad_()
    qo, ko = dk.rotary(q, k, positions, frequency, sections=sections, paired=paired)
    dq, dk_ = torch.randn_like(q), torch.randn_like(k)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk_))
    check_turned(gq, dq, positions, frequency, sections, paired, -1.0)
    check_turned(gk, dk_, positions, frequency, sections, paired, -1.0)
    # Against differences: the turning is linear, so they are exact but for the roundings.
    v = torch.randn_like(q)
    want, off = turned(v.detach(), positions, frequency, sections, paired)
    left, right = (gq.double() * v.double()).sum(), (dq.double() * want).sum()
    _, off_g = turned(dq, positions, frequency, sections, paired, -1.0)
    room = (v.double().abs() * (gq.double().abs() * 2 * half_step(q.dtype) + off_g)).sum() + (dq.double().abs() * off).sum()
    assert abs(float(left - right)) <= float(room)


def test_rotary_of_one_tensor_when_only_it_wants_a_gradient():
    q, k, positions, frequency = rotary_case(10, 4, 2, 64, [32], False, "fp16")
    k.requires_grad_()
    qo, ko = dk.rotary(q, k, positions[0], frequency)
    gk, = torch.autograd.grad(ko, k, torch.ones_like(ko))
    check_turned(gk, torch.ones_like(k), positions, frequency, [32], False, -1.0)


def test_rotary_of_far_positions():
    q = torch.randn((4, 2, 128), generator=gen(3), device="cuda")
    positions = torch.tensor([2 ** 31 + 12345, 10 ** 9 + 7, -5, 2 ** 24 + 1], device="cuda")
    frequency = 10000.0 ** (-torch.arange(64, device="cuda") / 64)
    out, _ = dk.rotary(q, None, positions, frequency)
    check_turned(out, q, positions, frequency, [64], False)
    assert dk.rotary(q[:0], None, positions[:0], frequency)[0].shape == (0, 2, 128)
    strided = torch.stack([positions, positions + 1], 1)[:, 1]
    assert torch.equal(dk.rotary(q, None, strided, frequency)[0], dk.rotary(q, None, positions + 1, frequency)[0])
    # Heads that all read one row, and transposed heads.
    one = q[:, :1].expand(4, 3, 128)
    assert torch.equal(dk.rotary(one, None, positions, frequency)[0][:, 2], out[:, 0])
    across = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(dk.rotary(across, None, positions, frequency)[0], out)
    odd = torch.empty(4 * 2 * 128 + 1, device="cuda")[1:].view(4, 2, 128).copy_(q)
    assert torch.equal(dk.rotary(odd, None, positions, frequency)[0], out)


def test_rotary_gradient_of_a_gradient():
    """Turning is linear: the gradient's gradient is the turning itself."""
    q, k, positions, frequency = rotary_case(9, 4, 2, 64, [20, 12], False, "fp32")
    dq = torch.randn_like(q).requires_grad_()
    q.requires_grad_()
    out, _ = dk.rotary(q, k, positions, frequency, sections=[20, 12])
    once, = torch.autograd.grad(out, q, dq, create_graph=True)
    v = torch.randn_like(q)
    twice, = torch.autograd.grad(once, dq, v)
    assert torch.equal(twice, dk.rotary(v, None, positions, frequency, sections=[20, 12])[0])


def test_rotary_refusals():
    q, k, positions, frequency = rotary_case(6, 4, 2, 64, [20, 12], False, "fp16")
    good = dict(sections=[20, 12])
    bad = [
        lambda: dk.rotary(q, k, positions, frequency), lambda: dk.rotary(q, k, positions, frequency, sections=[20, 13]),
        lambda: dk.rotary(q, k, positions, frequency, sections=[32]), lambda: dk.rotary(q, k, positions, frequency, sections=[40, -8]),
        lambda: dk.rotary(q, k[:5], positions, frequency, **good), lambda: dk.rotary(q, k.float(), positions, frequency, **good),
        lambda: dk.rotary(q, k, positions.float(), frequency, **good), lambda: dk.rotary(q, k, positions[:, :5], frequency, **good),
        lambda: dk.rotary(q, k, positions, frequency.double(), **good), lambda: dk.rotary(q, k, positions.cpu(), frequency, **good),
        lambda: dk.rotary(q.cpu(), None, positions, frequency, **good), lambda: dk.rotary(q[..., :63], None, positions, torch.ones(32, device="cuda"), **good),
        lambda: dk.rotary(q, q, positions, frequency, inplace=True, **good), lambda: dk.rotary(q[0], None, positions, frequency, **good),
        lambda: dk.rotary(q[:, :1].expand(6, 4, 64), None, positions, frequency, inplace=True, **good),
        lambda: dk.rotary(q.view(-1)[:768].view(6, 2, 64), q.view(-1)[64:832].view(6, 2, 64), positions, frequency, inplace=True, **good),
        lambda: dk.rotary(q.double(), None, positions, frequency, **good), lambda: dk.rotary(q, k, positions.repeat(3, 1), frequency, **good),
        lambda: dk.rotary(q.transpose(1, 2), None, positions, frequency[:2], sections=[1, 1], inplace=True),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---------------------------------------------------------------------------
# The cache read back
# ---------------------------------------------------------------------------

READS = [  # lengths, rows (None: all), kv heads, dim, block, code
    ([700], None, 8, 128, 64, "int8"), ([1], None, 1, 64, 16, "e4m3"), ([0, 5, 0, 0, 33, 16, 1], None, 3, 64, 16, "int8"),
    ([100, 37, 250], [7, 37, 0], 2, 256, 48, "e4m3"), ([3, 90], [5, 100], 4, 128, 32, "int8"),
    ([(37 * i) % 211 for i in range(300)], None, 5, 64, 48, "e4m3"), ([2 * (i % 2) for i in range(3000)], None, 1, 128, 16, "int8"),
]


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("lengths,rows,heads,dim,block,code", READS, ids=[f"{len(r[0])}x{r[3]}{r[5]}" for r in READS])
def test_cache_read(lengths, rows, heads, dim, block, code, dtype):
    g = torch.Generator().manual_seed(len(lengths))
    rows = lengths if rows is None else rows
    per = [-(-x // block) for x in lengths]
    blocks, width = sum(per) + 3, max(per) + 2
    order = torch.randperm(blocks, generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for r, p in enumerate(per):
        table[r, :p] = order[at:at + p]
        at += p
    cache = dk.PagedCache8(blocks, block, heads, dim, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn)
    for pool in (cache.k, cache.v):
        raw = torch.randint(0, 256, pool.shape, generator=g, dtype=torch.int32).to(torch.uint8)
        if code == "e4m3":
            raw[(raw & 127) == 127] = 5  # no NaN
        pool.view(torch.uint8).copy_(raw)
    for scale in (cache.k_scale, cache.v_scale):
        scale.copy_(torch.rand(scale.shape, generator=g) * 0.01 + 1e-3)
    starts = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    total, pad = int(starts[-1]), 3
    sentinel = [torch.full((total + pad, heads, dim), 99.0, dtype=HALF[dtype], device="cuda") for _ in range(2)]
    k, v = dk.cache_read(cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), starts.cuda(), total + pad, dtype=HALF[dtype], out=sentinel)
    assert k is sentinel[0] or k.data_ptr() == sentinel[0].data_ptr()
    for out, pool, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        real = pool.float() * scale[:, :, None, None]
        want = torch.full_like(out, 99.0)
        for r, (n, m) in enumerate(zip(lengths, rows)):
            mine = real[table[r, :per[r]].long().cuda()].transpose(1, 2).reshape(-1, heads, dim)[:n].to(out.dtype)
            part = torch.zeros((m, heads, dim), dtype=out.dtype, device="cuda")
            have = min(m, n)
            if have:
                part[m - have:] = mine[n - have:]
            want[int(starts[r]):int(starts[r + 1])] = part
        assert torch.equal(out, want)
    if total:
        k2, _ = dk.cache_read(cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), starts.cuda(), total, dtype=HALF[dtype])
        assert torch.equal(k2, k[:total])
        fewer = total // 2  # rows behind the call's are not asked for
        k3, _ = dk.cache_read(cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), starts.cuda(), fewer, dtype=HALF[dtype])
        assert torch.equal(k3, k[:fewer])


def test_cache_read_of_other_layouts_and_bad_pages():
    blocks, block, heads, dim = 6, 16, 2, 64
    g = torch.Generator().manual_seed(3)
    pool = torch.randint(-128, 128, (2, blocks, block, heads, dim), generator=g, dtype=torch.int32).to(torch.int8).cuda()
    scale = torch.rand((2, blocks, heads), generator=g).cuda()
    cache = dk.PagedCache8.from_tensors(pool[0].transpose(1, 2), pool[1].transpose(1, 2), scale[0].contiguous(), scale[1].contiguous())
    table = torch.tensor([[2, 99, -7, 4]], dtype=torch.int32).cuda()
    lengths, starts = torch.tensor([80], dtype=torch.int32).cuda(), torch.tensor([0, 80], dtype=torch.int32).cuda()
    wide = torch.zeros((80, 3 * heads * dim), dtype=torch.float16, device="cuda")
    out = tuple(wide[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in (0, 2))
    k, v = dk.cache_read(cache, table, lengths, starts, 80, out=out)
    for o, p, s in ((k, pool[0], scale[0]), (v, pool[1], scale[1])):
        assert torch.equal(o[:16], (p[2].float() * s[2][:, None]).half()) and torch.equal(o[48:64], (p[4].float() * s[4][:, None]).half())
        assert (o[16:48] == 0).all() and (o[64:] == 0).all()  # outside the pool; past the table
    assert (wide[:, heads * dim:2 * heads * dim] == 0).all()
    for bad in (dict(out=(k, k)), dict(out=(k, v[:, :1])), dict(dtype=torch.float32), dict(out=(wide[:, 1:129].unflatten(1, (2, 64)), v))):
        with pytest.raises(RuntimeError):
            dk.cache_read(cache, table, lengths, starts, 80, **bad)
    with pytest.raises(RuntimeError):
        dk.cache_read(cache, table, lengths.long(), starts, 80)
    with pytest.raises(RuntimeError):
        dk.cache_read(cache, table, lengths, starts[:1], 80)


def test_cache_read_far_into_a_large_pool():
    """Pages whose bytes lie past 2^32."""
    blocks, block, heads, dim = (1 << 32) // (256 * 8 * 256) + 8, 256, 8, 256
    k = torch.zeros((blocks, heads, block, dim), dtype=torch.int8, device="cuda")
    k[-1] = torch.randint(-127, 128, k[-1].shape, generator=gen(2), device="cuda").to(torch.int8)
    scale = torch.full((blocks, heads), 0.25, device="cuda")
    cache = dk.PagedCache8.from_tensors(k, k, scale, scale)
    table = torch.tensor([[blocks - 1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([200], dtype=torch.int32, device="cuda")
    a, b = dk.cache_read(cache, table, n, torch.tensor([0, 200], dtype=torch.int32, device="cuda"), 200)
    want = (k[-1].transpose(0, 1)[:200].float() * 0.25).half()
    assert torch.equal(a, want) and torch.equal(b, want)


# ---------------------------------------------------------------------------
# Together: a prompt's step
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_a_prompt_step(code):
    """Projections, positions, append, read back, attention over the rows read, and the gated block, against the same in 64 bits of the
    values that each step was given."""
    dim, heads, kv, d, hidden, n = 256, 4, 2, 64, 384, 150
    w = {name: weights(m, k, 100 + i) for i, (name, m, k) in enumerate(
        (("qkv", (heads + 2 * kv) * d, dim), ("o", dim, heads * d), ("gate", hidden, dim), ("up", hidden, dim), ("down", dim, hidden)))}
    x = rows_of(n, dim, torch.float16, 110)
    qkv = dk.gemm(*w["qkv"], x).view(n, heads + 2 * kv, d)
    q, k, v = qkv.split([heads, kv, kv], 1)
    positions = torch.stack([torch.arange(n), torch.arange(n) // 12, torch.arange(n) % 12]).cuda()
    frequency = (0.9 ** torch.arange(32)).cuda()
    before = qkv.clone()
    dk.rotary(q, k, positions, frequency, sections=[8, 12, 12], inplace=True)
    check_turned(qkv[:, :heads + kv], before[:, :heads + kv], positions, frequency, [8, 12, 12], False)
    assert torch.equal(v, before[:, heads + kv:])
    cache = dk.PagedCache8(12, 16, kv, d, dtype=code)
    free, ring = cache.free_list()
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.full((2, 12), -1, dtype=torch.int32, device="cuda")
    plan = dk.cache_plan(ints([0, 0]), ints([n - 40, 40]), table, free, ring, 16, n)
    dk.cache_append(k, v, plan.slots, cache)
    kr, vr = dk.cache_read(cache, table, plan.lengths, plan.starts, n)
    # A code is half a step off: int8's step is its page's largest over 127, e4m3's 2^-3 of the value, or 2^-9 of the scale; and fp16's rounding.
    for rows, given in ((kr, k), (vr, v)):
        largest = given.float().abs().amax()
        step = largest / 127 / 2 if code == torch.int8 else given.float().abs() * 2.0 ** -4 + largest / 448 * 2.0 ** -10
        assert ((rows.float() - given.float()).abs() <= step * 1.001 + given.float().abs() * 2.0 ** -11).all()
    # The same as the attention sees: over the rows read back, in 64 bits.
    out = dk.cache_attention(q, cache, table, plan.lengths, plan.starts)
    for a, b in ((0, n - 40), (n - 40, n)):
        kk, vv = (t[a:b].double().repeat_interleave(heads // kv, 1) for t in (kr, vr))
        s = torch.einsum("qhd,khd->hqk", q[a:b].double(), kk) * d ** -0.5
        s = s.masked_fill(torch.ones(b - a, b - a, device="cuda").triu(1).bool(), -math.inf)
        want = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), vv)
        # fp16 rows (2^-11), weights (2^-11 of those that count) and result; scores move by 2^-11 of sum |q k|.
        moved = torch.einsum("qhd,khd->hqk", q[a:b].double().abs(), kk.abs()).amax() * d ** -0.5 * 2.0 ** -10
        assert ((out[a:b].double() - want).abs() <= vv.abs().amax() * (4 * 2.0 ** -11 + 2 * float(moved))).all()
    y = dk.gemm(*w["o"], out.reshape(n, -1))
    check_product(y, out.reshape(n, -1), values(w["o"], torch.float16).t(), depth=heads * d)
    h = dk.gemm_gated(w["gate"], w["up"], y)
    check_gated(h, y, values(w["gate"], torch.float16), values(w["up"], torch.float16), "silu", dim)
    check_product(dk.gemm(*w["down"], h), h, values(w["down"], torch.float16).t(), depth=hidden)


def test_first_call_of_a_process_may_be_captured():
    """Nothing that a first call sets up stands in a capture's way."""
    code = """
import torch, sys
sys.path.insert(0, "decode-kernel_b200")
import decode_kernel as dk
from decode_kernel import _cuda
packed, scales = torch.zeros(256, 64, dtype=torch.int32, device="cuda"), torch.ones(256, 4, dtype=torch.float16, device="cuda")
packed += 0x11111111
xs = [torch.ones(T, 512, dtype=torch.float16, device="cuda") for T in (1, 12, 40, 300)]
q, pos, freq = torch.ones(5, 2, 64, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ys = [dk.gemm(packed, scales, x) for x in xs]
    back = [dk.gemm_t(packed, scales, y) for y in ys]
    hs = [dk.gemm_gated((packed, scales), (packed, scales), x) for x in xs]
    turned = dk.rotary(q, None, pos, freq)[0]
graph.replay()
torch.cuda.synchronize()
assert all((y == 512).all() for y in ys) and all((b == torch.inf).all() for b in back) and torch.equal(turned, q)
assert all((h == torch.inf).all() for h in hs)
"""
    import subprocess
    import sys
    from pathlib import Path

    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240, cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0, done.stderr[-2000:]


def test_no_wait_ran_out():
    torch.cuda.synchronize()
    assert capi.load().dk_device_error(-1, 0) == 0


@pytest.mark.parametrize("T", [1, 12, 24, 60, 300])
def test_weights_that_change_between_calls(T):
    """New weights written into the same tensors just before a call: no form reads what stood there before."""
    M, K = 700, 1024
    sets = [(weights(M, K, 300 + i), weights(M, K, 310 + i)) for i in range(2)]
    x, g = rows_of(T, K, torch.float16, 320), rows_of(T, M, torch.float16, 321)
    call = lambda a, b: (dk.gemm(*a, x), dk.gemm_gated(a, b, x), dk.gemm_t(*a, g))  # noqa: E731
    want = [call(a, b) for a, b in sets]
    held = [tuple(t.clone() for t in w) for w in sets[0]]
    for i in range(60):
        for mine, given in zip(held, sets[i % 2]):
            for t, n in zip(mine, given):
                t.copy_(n)
        assert all(torch.equal(p, q) for p, q in zip(call(*held), want[i % 2])), i


def test_few_rows_on_several_streams_at_once():
    M, K = 1500, 1024
    w, w2 = weights(M, K, 330), weights(M, K, 331)
    xs = [rows_of(T, K, dtype, 332 + T) for T, dtype in ((3, torch.bfloat16), (9, torch.float16), (16, torch.float16), (24, torch.bfloat16), (32, torch.float16))]
    call = lambda x: (dk.gemm(*w, x), dk.gemm_gated(w, w2, x), dk.gemm_t(*w, dk.gemm(*w, x)))  # noqa: E731
    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
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


def test_keys_and_values_read_on_another_stream_and_in_a_graph():
    cache = dk.PagedCache8(20, 16, 2, 64)
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        pool.copy_(torch.randint(-127, 128, pool.shape, generator=gen(1), device="cuda"))
        scale.uniform_(0.01, 0.02)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lengths, starts = ints([[3, 5, 7], [11, 13, 2]]), ints([40, 20]), ints([0, 40, 60])
    want = dk.cache_read(cache, table, lengths, starts, 60)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = dk.cache_read(cache, table, lengths, starts, 60)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dk.cache_read(cache, table, lengths, starts, 60)
    lengths.copy_(ints([33, 44]))  # rows that a request does not hold become zeros
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(dk.cache_read(cache, table, lengths, starts, 60), got))
    assert (got[0][:7] == 0).all() and torch.equal(got[0][7:40], want[0][:33])


@pytest.mark.parametrize("which", ["gemm", "few", "gated", "gemm_t", "rotary q", "rotary k", "cache_read"])
def test_a_graph_learns_that_what_it_saved_was_written_over(which):
    M, K = 256, 256
    w, T = weights(M, K, 340), 4 if which == "few" else 40
    x = rows_of(T, K, torch.float16, 341)
    out = torch.zeros(T, M, dtype=torch.float16, device="cuda")
    q, k = (torch.randn(6, h, 64, device="cuda") for h in (4, 2))
    frequency = torch.rand(32, device="cuda")
    cache = dk.PagedCache8(4, 16, 2, 64)
    kv = tuple(torch.zeros(6, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    saved = {"rotary q": q, "rotary k": k, "cache_read": kv[1]}.get(which, out)
    factor = torch.ones_like(saved, requires_grad=True)
    loss = (factor * saved).sum()
    if which in ("gemm", "few"):
        dk.gemm(*w, x, out=out)
    elif which == "gated":
        dk.gemm_gated(w, w, x, out=out)
    elif which == "gemm_t":
        dk.gemm_t(*w, x, out=out)
    elif which == "cache_read":
        dk.cache_read(cache, ints([[0]]), ints([6]), ints([0, 6]), 6, out=kv)
    else:
        dk.rotary(q, k, torch.arange(6, device="cuda"), frequency, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_outputs_are_written_under_inference_mode():
    w = weights(256, 256, 342)
    with torch.inference_mode():
        x = rows_of(40, 256, torch.float16, 343)
        out = torch.zeros(40, 256, dtype=torch.float16, device="cuda")
        dk.gemm(*w, x, out=out)
        assert torch.equal(out, dk.gemm(*w, x))
    dk.gemm(*w, x, out=out)  # inference tensors outside of it
    assert torch.equal(out, dk.gemm(*w, x))
