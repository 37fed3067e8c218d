"""Edges of the prompt operators that need no device: which tensors share memory."""

from __future__ import annotations

import random

import pytest
import torch

import decode_kernel as dk
from decode_kernel import _cuda


def bytes_of(t):
    """Every byte's address."""
    at = torch.zeros((), dtype=torch.int64)
    for size, stride in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(size) * stride * t.element_size()
    at = at.reshape(-1, 1) + torch.arange(t.element_size()) + t.data_ptr()
    return set(at.flatten().tolist())


def any_tensor(rng, home):
    t = home.view(rng.choice([torch.uint8, torch.float16, torch.float32]))
    sizes, strides, room = [], [], t.numel() - 1
    for _ in range(rng.randint(0, 4)):
        sizes.append(rng.choice([0, 1, 2, 3, 5, 8, 13] if rng.random() < 0.2 else [1, 2, 3, 5, 8, 13]))
        most = room // max(1, sizes[-1] - 1)
        strides.append(rng.choice([0, 1, rng.randint(0, most), rng.randint(0, min(most, 20))]) if most else 0)
        room -= (max(1, sizes[-1]) - 1) * strides[-1]
        if room < 0:
            return any_tensor(rng, home)
    return t.as_strided(sizes, strides, rng.randint(0, room))


def test_shared_memory_of_any_strides():
    rng, home = random.Random(1), torch.zeros(600, dtype=torch.uint8)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        a, b = any_tensor(rng, home), any_tensor(rng, home)
        want = bool(bytes_of(a) & bytes_of(b))
        assert _cuda.shares_memory(a, b) == want, (a.dtype, a.shape, a.stride(), a.storage_offset(), b.dtype, b.shape, b.stride(), b.storage_offset())
        seen[want] += 1
    assert min(seen.values()) > 1000


@pytest.mark.parametrize("heads", [5, 6, 48])
def test_slices_of_a_projection(heads):
    fused = torch.zeros(1 << 13, heads, 64, dtype=torch.float16)
    share = _cuda.shares_memory
    for i in range(heads):
        assert not share(fused[:, :i], fused[:, i:]) and share(fused[:, :i + 1], fused[:, i:])
    assert not share(fused[:, ::2], fused[:, 1::2]) and share(fused[:, ::2], fused[:, 4:5])
    assert not share(fused[::2], fused[1::2]) and not share(fused[:100], fused[100:]) and share(fused[:101], fused[100:])
    flat = fused.view(1 << 13, -1)
    assert not share(flat[:, :100], flat[:, 100:]) and share(flat[:, :101], flat[:, 100:]) and share(flat[:, 5:6], flat.t()[5:7])
    assert not share(fused[..., :32], fused[..., 32:]) and share(fused[..., :33], fused[..., 32:])
    assert not share(fused, fused.clone()) and share(fused, fused.view(torch.int8)[..., 127:])


PACKED, SCALES = torch.zeros(64, 32, dtype=torch.int32), torch.zeros(64, 2, dtype=torch.float16)
PAIR = (PACKED, SCALES)
DIFFERENTIABLE = {
    "gemm": (lambda x: dk.gemm(*PAIR, x), (3, 256)), "gemm_t": (lambda x: dk.gemm_t(*PAIR, x), (3, 64)), "gemm_gated": (lambda x: dk.gemm_gated(PAIR, PAIR, x), (3, 256)),
    "rotary": (lambda x: dk.rotary(x, None, torch.zeros(3, dtype=torch.int32), torch.ones(4)), (3, 2, 8)),
    "rotary in place": (lambda x: dk.rotary(x, None, torch.zeros(3, dtype=torch.int32), torch.ones(4), inplace=True), (3, 2, 8)),
    "linear": (lambda x: dk.W4A16Linear(*PAIR)(x), (3, 256)), "linear's op": (lambda x: torch.ops.decode_kernel.w4a16_linear(x, *PAIR), (3, 256)),
}


@pytest.mark.parametrize("which", list(DIFFERENTIABLE))
def test_forward_mode_is_refused(which):
    call, shape = DIFFERENTIABLE[which]
    x = torch.zeros(shape, dtype=torch.float16)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    if which == "linear":
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="CUDA"):  # without a tangent it is the device that is refused
        call(x)


def test_outputs_that_require_a_gradient_are_refused():
    x, g = torch.zeros(3, 256, dtype=torch.float16), torch.zeros(3, 64, dtype=torch.float16)
    y, dx = torch.zeros(3, 64, dtype=torch.float16, requires_grad=True), torch.zeros(3, 256, dtype=torch.float16, requires_grad=True)
    calls = (lambda out: dk.gemm(*PAIR, x, out=out), y), (lambda out: dk.gemm_gated(PAIR, PAIR, x, out=out), y), (lambda out: dk.gemm_t(*PAIR, g, out=out), dx)
    for call, out in calls:
        for given in (out, out * 2):
            with pytest.raises(RuntimeError, match="out takes no part"):
                call(given)
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
                call(given)


def test_the_linear_layers_gradient_is_traced():
    """Forward and backward with tensors that have no data, as a compiler runs them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, dy, packed, scales):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(torch.ops.decode_kernel.w4a16_linear(x, packed, scales), x, dy)[0]

    for shape in ((3,), (2, 5), ()):
        with FakeTensorMode():
            args = (torch.empty(*shape, 256, dtype=torch.float16), torch.empty(*shape, 64, dtype=torch.float16), torch.empty(64, 32, dtype=torch.int32), torch.empty(64, 2, dtype=torch.float16))
            dx = step(*args)
            assert dx.shape == (*shape, 256) and dx.dtype == torch.float16
    graph = make_fx(step, tracing_mode="fake")(torch.zeros(3, 256, dtype=torch.float16), torch.zeros(3, 64, dtype=torch.float16), PACKED, SCALES)
    assert sum("w4a16_linear" in str(n.target) for n in graph.graph.nodes) == 2
