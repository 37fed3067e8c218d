"""A paged cache of keys and values in 8 bits, and a decode step over it.

``PagedCache8`` is the pool of pages; ``cache_plan`` builds a step's block
tables, slot maps and lengths on the GPU from the requests' lengths;
``cache_append`` quantises the step's keys and values into their pages (one
fp32 scale per page and KV head, int8 or float8_e4m3fn codes);
``cache_attention`` attends over the pages; ``cache_read`` gives them back as
rows of keys and values.  Nothing waits for the GPU, so a
whole step can be captured in a CUDA graph.  There is no CPU fallback.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

__all__ = ["CachePlan", "PagedCache8", "cache_append", "cache_attention", "cache_plan", "cache_read", "release_workspaces"]

_module = None


def _extension():
    """decode_kernel._cuda, imported at the first call: the package loads without it."""
    global _module
    if _module is None:
        from . import _cuda

        _module = _cuda
    return _module


class PagedCache8:
    """Pages of ``block_size`` tokens of every KV head.

    ``k``, ``v``: int8 or float8_e4m3fn [blocks, kv_heads, block_size, head_dim];
    ``k_scale``, ``v_scale``: fp32 [blocks, kv_heads].  A value is its code
    times its page's and head's scale; scales are positive (V's below 2^-70,
    negative ones too, count as 2^-70).  block_size is a multiple of 16 up to
    256, head_dim 64, 128 or 256.
    """

    def __init__(self, blocks: int, block_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.int8, device: Union[str, torch.device] = "cuda"):
        shape = (blocks, kv_heads, block_size, head_dim)
        self._set(torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype),
                  torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype),
                  torch.zeros(shape[:2], dtype=torch.float32, device=device),
                  torch.zeros(shape[:2], dtype=torch.float32, device=device))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor) -> "PagedCache8":
        """A cache over tensors that the caller owns.  k and v may be views
        with other strides (multiples of 32, the last dimension contiguous),
        for example a transposed [blocks, block_size, kv_heads, head_dim]."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale) -> None:
        self._handle = _extension().Cache8(k, v, k_scale, v_scale)
        self._tensors = (k, v, k_scale, v_scale)

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    blocks = property(lambda self: self._tensors[0].shape[0])
    kv_heads = property(lambda self: self._tensors[0].shape[1])
    block_size = property(lambda self: self._tensors[0].shape[2])
    head_dim = property(lambda self: self._tensors[0].shape[3])
    dtype = property(lambda self: self._tensors[0].dtype)
    device = property(lambda self: self._tensors[0].device)

    def free_list(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Every page free: the ring of page numbers and its state, as
        ``cache_plan`` takes them."""
        free = torch.arange(self.blocks, dtype=torch.int32, device=self.device)
        ring = torch.tensor([0, self.blocks, 0, 0], dtype=torch.int64, device=self.device)
        return free, ring


class CachePlan(NamedTuple):
    """What ``cache_plan`` writes for a step."""

    lengths: torch.Tensor  #: int32 [requests], tokens held after the step
    starts: torch.Tensor   #: int32 [requests + 1], first row of each request's new tokens
    slots: torch.Tensor    #: int64 [tokens], page * block_size + row in the page, or -1
    ring: torch.Tensor     #: int64 [4], the ring's beginning and end, pages missing, requests too wide


def cache_plan(held: torch.Tensor, fresh: torch.Tensor, block_table: torch.Tensor,
               free_blocks: torch.Tensor, ring: torch.Tensor, block_size: int, tokens: int, *,
               out: Optional[CachePlan] = None) -> CachePlan:
    """Block tables and slot maps of a step, in one launch.

    Request r holds ``held[r]`` tokens and brings ``fresh[r]`` new ones
    (``fresh[r] < 0``: it has ended).  New pages come from the beginning of the
    ring ``free_blocks`` (entries ``ring[0] <= i < ring[1]``, modulo its
    length) into ``block_table`` [requests, max_blocks], which is updated in
    place like the ring's entries; ended requests' pages go to its end: all
    ceil(held / block_size) of them, so none may be released before.  ``held``
    may be lowered between calls (drafts taken back); pages that it leaves have
    to be put at the ring's end by the caller, or they are lost.
    ``tokens`` is the number of rows of the step, padding included.  A request
    that the free pages or the table's width cannot serve keeps its length, its
    rows have slot -1, and the returned ring's entries 2 and 3 say how many
    pages were missing and how many requests were too wide.

    ``out`` reuses tensors of an earlier plan; its ``lengths`` may be ``held``
    and its ``ring`` may be ``ring`` (the call then runs on one SM, which steps
    of many thousand tokens feel).
    """
    if out is None:
        return CachePlan(*_extension().cache_plan(held, fresh, block_table, free_blocks, ring, block_size, tokens))
    return CachePlan(*_extension().cache_plan(held, fresh, block_table, free_blocks, ring, block_size, tokens, *out))


def cache_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: PagedCache8) -> None:
    """Quantise k and v (fp16 or bf16 [tokens, kv_heads, head_dim]) into the
    pages that ``slots`` names (``cache_plan``'s; -1 skips the row).

    A page's scale for a head is the largest magnitude over 127 (int8) or 448
    (e4m3) and grows with later tokens, when the page's earlier codes are
    rounded to the new scale; tokens that begin a page begin its scale.  Values
    past the scale saturate, NaN becomes 0.  The rows of a page must be
    neighbours (none skipped between them) with rising slots; rows of the page
    between them keep their codes.
    """
    _extension().cache_append(k, v, slots, cache._handle)


def cache_attention(q: torch.Tensor, cache: PagedCache8, block_table: torch.Tensor,
                    lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0,
                    out: Optional[torch.Tensor] = None, lse: bool = False):
    """softmax(scale * q . K) . V over each request's pages.

    q: fp16 or bf16 [tokens, q_heads, head_dim]; q_heads a multiple of the
    cache's kv_heads (query head h reads KV head h // (q_heads / kv_heads)).
    Request r's queries are rows ``starts[r]:starts[r + 1]`` and the last of
    its ``lengths[r]`` tokens; without ``starts`` each request has one.
    ``causal`` hides the tokens after a query, ``window`` > 0 also those
    ``window`` or more before it.  A query that sees no token gets zeros.
    ``scale`` defaults to head_dim ** -0.5.

    Rows past ``starts[-1]`` are not written (a new ``out`` holds anything there),
    and rows of a request that ``cache_plan`` could not serve (slot -1) mean
    nothing: its last old tokens are taken for theirs.

    Scores and sums are fp32; the softmax's weights are rounded to fp16 for the
    product with V (2^-12 of each), and bf16 queries scaled by a power of two
    into fp16 (which values below 2^-31 of their row's largest lose bits by).

    Returns out, or (out, lse) with the fp32 [tokens, q_heads] log of the sums
    of exponentials.
    """
    o, l = _extension().cache_attention(q, cache._handle, block_table, lengths, starts, scale, causal, window, out, lse)
    return (o, l) if lse else o


def cache_read(cache: PagedCache8, block_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
               tokens: int, *, dtype: torch.dtype = torch.float16,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cache's keys and values as rows: (k, v), fp16 or bf16 [tokens, kv_heads, head_dim].

    Request r's rows are ``starts[r]:starts[r + 1]`` and the last of its
    ``lengths[r]`` tokens, as ``cache_attention`` takes its queries; with
    ``starts`` the running sum of ``lengths`` they are all of them.  ``tokens``
    is the number of rows, padding included.  A value is its code times its
    page's and head's scale in fp32, rounded once (past fp16's range to
    infinity).  Rows without a token (more rows than tokens, table entries
    outside the pool) are zeros; rows from ``starts[-1]`` on are not written.

    ``out``: (k, v) of an earlier call, or views with contiguous rows a multiple
    of 8 values apart.
    """
    return _extension().cache_read(cache._handle, block_table, lengths, starts, tokens, dtype, *(out or (None, None)))


def release_workspaces() -> None:
    """Give the memory that ``cache_attention`` keeps back to torch's allocator.

    It keeps one workspace (24 MB; 12 MB for heads of 64) for each device and
    stream that it was called on outside a capture.  Call this after a change of
    streams, and before a stream of one's own is destroyed: a new stream could
    get its handle.  The next call on a stream makes a new workspace.
    """
    _extension().release_workspaces()
