"""The W4A16 GEMV as a PyTorch operator and module.

``torch.ops.decode_kernel.w4a16_linear(x, packed, scales) -> y`` is a
``torch.library`` custom op around this package's CUDA kernel (the caller
side of the reference's ``w4a16_linear``, python/decode_kernel/__init__.py:
62-83): it has a fake (meta) implementation, so code that traces or captures
-- torch.fx, ``torch.cuda.CUDAGraph`` capture of a decode step -- sees a
proper operator with a known output shape instead of an opaque Python call.
``W4A16Linear`` is a bias-free ``nn.Linear`` replacement holding the packed
weights and scales as buffers.  ``torch.ops.decode_kernel.w4a16_silu_mul(x,
packed_gate, scales_gate, packed_up, scales_up)`` is a gated MLP's gate/up
pair with its SiLU-mul epilogue in one launch.  ``w4a16_linear`` has a gradient
for x, the transposed product with the frozen weights.  ``W4A16GatedMLP`` is a
gated feed-forward block over the many-row products, for prompts and training.

There is no CPU implementation: the op raises on CPU tensors, like the rest of
the package.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from .quantize import GROUP_SIZE, quantize_and_pack_cuda

__all__ = ["W4A16GatedMLP", "W4A16Linear", "w4a16_linear_op", "w4a16_silu_mul_op"]


def _no_tangent(x: torch.Tensor) -> None:
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError("forward-mode derivatives are not supported")


@torch.library.custom_op("decode_kernel::w4a16_linear", mutates_args=())
def w4a16_linear_op(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """y[..., M] = x[..., K] . dequant(W)^T (fp16), any number of leading dims."""
    from . import gemv

    _no_tangent(x)
    if not x.is_cuda:
        raise RuntimeError("decode_kernel::w4a16_linear runs on CUDA tensors only")
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    y = gemv(packed, scales, x2)
    return y.reshape(*lead, packed.shape[0])


@w4a16_linear_op.register_fake
def _(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    torch._check(x.shape[-1] == packed.shape[1] * 8, lambda: "x.shape[-1] must equal K")
    torch._check(x.dtype == torch.float16, lambda: "x must be fp16")
    return x.new_empty((*x.shape[:-1], packed.shape[0]), dtype=torch.float16)


@torch.library.custom_op("decode_kernel::w4a16_linear_grad", mutates_args=())
def w4a16_linear_grad_op(dy: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """dx[..., K] = dy[..., M] . dequant(W): the gradient of w4a16_linear, an operator so that it can be traced."""
    from . import gemm_t

    return gemm_t(packed, scales, dy)


@w4a16_linear_grad_op.register_fake
def _(dy: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return dy.new_empty((*dy.shape[:-1], packed.shape[1] * 8))


def _linear_context(ctx, inputs, output) -> None:
    _, packed, scales = inputs
    ctx.save_for_backward(packed, scales)


def _linear_backward(ctx, dy: torch.Tensor):
    if ctx.needs_input_grad[2]:
        raise RuntimeError("the weights are frozen: scales must not require a gradient")
    return (w4a16_linear_grad_op(dy, *ctx.saved_tensors) if ctx.needs_input_grad[0] else None), None, None


def _linear_grad_backward(ctx, ddx: torch.Tensor):
    from . import gemm

    if ctx.needs_input_grad[2]:
        raise RuntimeError("the weights are frozen: scales must not require a gradient")
    return (gemm(*ctx.saved_tensors, ddx) if ctx.needs_input_grad[0] else None), None, None


w4a16_linear_op.register_autograd(_linear_backward, setup_context=_linear_context)
w4a16_linear_grad_op.register_autograd(_linear_grad_backward, setup_context=_linear_context)


@torch.library.custom_op("decode_kernel::w4a16_silu_mul", mutates_args=())
def w4a16_silu_mul_op(x: torch.Tensor, packed_gate: torch.Tensor, scales_gate: torch.Tensor,
                      packed_up: torch.Tensor, scales_up: torch.Tensor) -> torch.Tensor:
    """h[..., M] = silu(x . Wg^T) * (x . Wu^T) (fp16), one launch for both GEMVs."""
    from . import gemv_silu_mul

    if not x.is_cuda:
        raise RuntimeError("decode_kernel::w4a16_silu_mul runs on CUDA tensors only")
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    h = gemv_silu_mul((packed_gate, scales_gate), (packed_up, scales_up), x2)
    return h.reshape(*lead, packed_gate.shape[0])


@w4a16_silu_mul_op.register_fake
def _(x, packed_gate, scales_gate, packed_up, scales_up):
    torch._check(x.shape[-1] == packed_gate.shape[1] * 8, lambda: "x.shape[-1] must equal K")
    torch._check(packed_up.shape[0] == packed_gate.shape[0], lambda: "gate and up rows differ")
    torch._check(x.dtype == torch.float16, lambda: "x must be fp16")
    return x.new_empty((*x.shape[:-1], packed_gate.shape[0]), dtype=torch.float16)


class W4A16Linear(torch.nn.Module):
    """Bias-free linear layer with symmetric int4 weights (group 128 along K,
    fp16 scales), computed by the B200 GEMV kernels."""

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor):
        super().__init__()
        if packed.dtype != torch.int32 or scales.dtype != torch.float16:
            raise ValueError("packed must be int32 [M, K/8] and scales fp16 [M, K/128]")
        if scales.shape != (packed.shape[0], packed.shape[1] * 8 // GROUP_SIZE):
            raise ValueError("scales shape must be [M, K/128]")
        self.register_buffer("packed", packed.contiguous())
        self.register_buffer("scales", scales.contiguous())

    @property
    def in_features(self) -> int:
        return self.packed.shape[1] * 8

    @property
    def out_features(self) -> int:
        return self.packed.shape[0]

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, device: Optional[torch.device] = None) -> "W4A16Linear":
        """Quantize an ``nn.Linear``'s weight (the reference quantizer's
        arithmetic, on the GPU); a bias is refused."""
        if linear.bias is not None:
            raise ValueError("W4A16Linear has no bias")
        w = linear.weight.detach().to(device or "cuda", torch.float32)
        packed, scales = quantize_and_pack_cuda(w)
        return cls(packed, scales)

    @classmethod
    def from_gptq(cls, qweight: torch.Tensor, scales: torch.Tensor,
                  qzeros: Optional[torch.Tensor] = None, g_idx: Optional[torch.Tensor] = None, *,
                  zeros_minus_one: bool = False) -> "W4A16Linear":
        """A layer from a symmetric 4-bit GPTQ checkpoint's tensors (group 128,
        no act-order), converted exactly by ``decode_kernel.gptq.from_gptq``;
        the buffers stay on the tensors' device."""
        from .gptq import from_gptq

        packed, s = from_gptq(qweight, scales, qzeros, g_idx, zeros_minus_one=zeros_minus_one)
        return cls(packed, s)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _no_tangent(x)
        return torch.ops.decode_kernel.w4a16_linear(x, self.packed, self.scales)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bits=4, group={GROUP_SIZE}"


def _plain(layer: torch.nn.Module) -> bool:
    """Whether a call of the layer is its product and nothing else: no adapter in its place or round its forward, no hooks."""
    return (isinstance(layer, W4A16Linear) and type(layer).forward is W4A16Linear.forward and "forward" not in layer.__dict__
            and not layer._forward_hooks and not layer._forward_pre_hooks
            and not layer._backward_hooks and not layer._backward_pre_hooks)


class W4A16GatedMLP(torch.nn.Module):
    """A gated feed-forward block with frozen 4-bit weights: down(act(gate(x)) * up(x)).

    ``gate``, ``up`` and ``down`` are ``W4A16Linear`` layers; ``act`` is "silu"
    or "gelu" (its tanh form).  Two products for any number of rows
    (``gemm_gated`` and ``gemm``, fp16 or bf16), and gradients for x.  Layers
    that have hooks, or that an adapter has taken the place of, are called as
    modules, and the activation is torch's then: gate and up both where one of
    them is, down by itself.
    """

    def __init__(self, gate: W4A16Linear, up: W4A16Linear, down: W4A16Linear, act: str = "silu"):
        super().__init__()
        if gate.packed.shape != up.packed.shape or down.in_features != gate.out_features:
            raise ValueError("gate and up must have the same shape, and down their rows as its input")
        if act not in ("silu", "gelu"):
            raise ValueError("act is 'silu' or 'gelu'")
        self.gate, self.up, self.down, self.act = gate, up, down, act

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        from . import gemm, gemm_gated

        if _plain(self.gate) and _plain(self.up):
            h = gemm_gated((self.gate.packed, self.gate.scales), (self.up.packed, self.up.scales), x, act=self.act)
        else:
            g = self.gate(x)
            h = (torch.nn.functional.silu(g) if self.act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")) * self.up(x)
        return gemm(self.down.packed, self.down.scales, h) if _plain(self.down) else self.down(h)
