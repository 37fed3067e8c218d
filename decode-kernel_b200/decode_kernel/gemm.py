"""Many rows through 4-bit weights, with gradients through the frozen weights.

``gemm`` is a layer's product for prompts and batches, ``gemm_gated`` the two
projections, activation and product of a gated block in one kernel (calls of few
rows have a small one before it that splits the rows), ``gemm_t`` the transposed
product.  The weights are frozen: gradients reach the rows, not
the packed weights or their scales.  There is no CPU fallback.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .cache import _extension

__all__ = ["gemm", "gemm_gated", "gemm_t"]

_ACTS = {"silu": 0, "gelu": 1}


class _GemmGated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, gate_scales, up, up_scales, act):
        h, g, u = _extension().w4a16_gemm(gate, gate_scales, up, up_scales, x, act, True)
        ctx.save_for_backward(gate, gate_scales, up, up_scales, g, u)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        gate, gate_scales, up, up_scales, g, u = ctx.saved_tensors
        dg, du = _extension().gated_grad(dh, g, u, ctx.act)
        dx = _extension().w4a16_gemm_t(gate, gate_scales, up, up_scales, dg, du)
        return dx.view(*dh.shape[:-1], dx.shape[-1]), None, None, None, None, None


def gemm(packed: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, *,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x . dequant(W)^T for any number of rows: fp16 or bf16 [..., K] -> [..., M].

    packed: int32 [M, K/8]; scales: fp16 [M, K/128].  Past 16 rows (32 of a
    gated pair) a weight q * scale is rounded once to x's type (past its range to
    infinity), for fewer it is not, so a row's last bits depend on how many stand
    beside it (and, up to 8 rows in fp16, on the GEMV's order of sums); products
    and sums are fp32, and so is the result until it is rounded once.  A row with an infinity or a NaN gives
    results that are not finite; which of the two is the formula's answer for a
    single infinity in a group of 128.  x may be any view;
    rows that do not begin on 16-byte boundaries are copied first.  ``out`` is
    contiguous or has contiguous rows.  Differentiable in x (reverse mode).
    """
    return _extension().linear(False, packed, scales, x, out)


def gemm_t(packed: torch.Tensor, scales: torch.Tensor, g: torch.Tensor, *,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """g . dequant(W): fp16 or bf16 [..., M] -> [..., K], the gradient of ``gemm``'s x.

    The types of ``gemm``; weights are rounded as for its many rows.  Differentiable
    in g (reverse mode).
    """
    return _extension().linear(True, packed, scales, g, out)


def gemm_gated(gate: Tuple[torch.Tensor, torch.Tensor], up: Tuple[torch.Tensor, torch.Tensor], x: torch.Tensor, *,
               act: str = "silu", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x . Wg^T) * (x . Wu^T) in one kernel: fp16 or bf16 [..., K] -> [..., M].

    ``gate`` and ``up``: ``(packed, scales)`` of two [M, K] matrices; ``act``:
    "silu" or "gelu" (its tanh form).  Everything between the products' fp32
    sums and the result is fp32, rounded once (``gemv_silu_mul`` rounds as the
    unfused fp16 sequence does).  Differentiable in x (reverse mode, once): the
    two projections are kept in x's type for that.
    """
    if act not in _ACTS:
        raise ValueError("act is 'silu' or 'gelu'")
    if torch.is_grad_enabled() and (x.requires_grad or gate[1].requires_grad or up[1].requires_grad):
        if gate[1].requires_grad or up[1].requires_grad:
            raise RuntimeError("the weights are frozen: scales must not require a gradient")
        if out is not None:
            raise RuntimeError("out takes no part in a gradient: call without it or under torch.no_grad()")
        return _GemmGated.apply(x, *gate, *up, _ACTS[act])
    return _extension().w4a16_gemm(*gate, *up, x, _ACTS[act], False, out)[0]
