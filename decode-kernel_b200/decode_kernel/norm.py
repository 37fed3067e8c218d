"""Norms before and after a block, with its gate and residual scale, in one launch."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .cache import _extension

__all__ = ["block_norm"]

_KINDS = {"rms": 0, "layer": 1}
_ACTS = {"none": 0, "sigmoid": 1, "silu": 2}


def block_norm(residual: torch.Tensor, y: Optional[torch.Tensor] = None, *, kind: str = "rms",
               post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, gate_act: str = "none",
               residual_scale: float = 1.0, block_scale: float = 1.0,
               pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
               eps: float = 1e-6, inplace: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """A block's output y into the residual stream, and the next block's input:

        u = norm(y) * post_weight + post_bias     (y itself without post_weight)
        r = residual_scale * residual + block_scale * act(gate) * u
        h = norm(r) * pre_weight + pre_bias       (None without pre_weight)

    and returns (r, h).  ``kind``: "rms" or "layer".  residual: [..., dim] in
    y's type or fp32; y, gate and weights in fp16 or bf16; gate: [dim],
    [..., 1] or [..., dim], through ``gate_act`` "none", "sigmoid" or "silu".
    Without y, h = norm(residual_scale * residual).  Computed in fp32 and
    rounded once, h from the unrounded r.  ``inplace`` writes r over residual.
    """
    if kind not in _KINDS or gate_act not in _ACTS:
        raise ValueError("kind is 'rms' or 'layer', gate_act 'none', 'sigmoid' or 'silu'")
    return _extension().block_norm(residual, y, _KINDS[kind], post_weight, post_bias, gate, _ACTS[gate_act],
                            residual_scale, block_scale, pre_weight, pre_bias, eps, inplace)
