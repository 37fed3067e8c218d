"""Rotary positions of queries and keys, with one axis or several, in one launch."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from .cache import _extension

__all__ = ["rotary"]


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequency, sections, paired, inverse):
        ctx.save_for_backward(positions, frequency)
        ctx.form = sections, paired, inverse
        q, k = _extension().rotary(q, k, positions, frequency, sections, paired, inverse, False)
        return q, k

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        sections, paired, inverse = ctx.form
        dq, dk = _extension().rotary(dq, dk, *ctx.saved_tensors, sections, paired, not inverse, False)
        return dq, dk, None, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequency: torch.Tensor, *,
           sections: Optional[Sequence[int]] = None, paired: bool = False, inverse: bool = False,
           inplace: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turn the value pairs of every head by their tokens' positions; returns (q, k).

        a_i = positions[axis(i), token] * frequency[i]
        (x, y) -> (x cos a - y sin a, x sin a + y cos a)

    q: fp16, bf16 or fp32 [tokens, q_heads, head_dim]; k: [tokens, kv_heads,
    head_dim] in q's type, or None.  Both may be views, as slices of a fused
    projection are.  ``frequency``: fp32 [pairs], radians a position; pair i is
    the values i and i + pairs, or 2i and 2i + 1 if ``paired``; values past
    2 * pairs are copied.  ``positions``: int32 or int64 [tokens], or [axes,
    tokens] (time, height, width, say; up to 4) with ``sections``, each axis's
    number of pairs in order.

    Angles are taken in fp64, so far positions are right; sines, cosines and the
    turning are fp32, rounded once.  ``inverse`` turns back.  ``inplace`` writes
    over q and k.  Differentiable in q and k (not in place).
    """
    if frequency.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("frequency must not require a gradient")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if inplace:
            raise RuntimeError("q and k that require a gradient are not turned in place")
        return _Rotary.apply(q, k, positions, frequency, sections, paired, inverse)
    return _extension().rotary(q, k, positions, frequency, sections, paired, inverse, inplace)
