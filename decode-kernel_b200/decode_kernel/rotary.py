"""Rotary positions of queries and keys, with one axis or several, in one launch."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from .cache import _extension

__all__ = ["rotary"]


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
    over q and k.  Differentiable in q and k (reverse mode, not in place).
    """
    return _extension().rotary(q, k, positions, frequency, sections, paired, inverse, inplace)
