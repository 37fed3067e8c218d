"""The decode-step operators at the edges of what their callers may do: hidden
pages that hold anything, wide tables, rows of a page with gaps, plans in
place, captured calls, and the sizes at which a launch takes another form."""

from __future__ import annotations

import pytest
import torch

import decode_kernel as dk
from test_decode_ops_gpu import attention_case, check_attention, run_attention

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kv,dim,bs,fresh", [
    (2, 64, 16, None), (2, 64, 48, None), (2, 64, 16, [3, 1, 9, 2]), (1, 64, 16, [20, 1, 30, 2]), (2, 128, 16, None), (1, 256, 48, [3, 1, 9, 2]),
])
def test_attention_ignores_hidden_pages_scales(code, kv, dim, bs, fresh):
    """Pages that lie wholly before a request's window may hold anything, their scales too."""
    lengths, window = [100, 70, 500, 49], 50
    case = attention_case(lengths, fresh, 4 * kv, kv, dim, bs, code, "fp16", seed=dim + bs)
    q, k, v, ks, vs, table, lengths, starts = case
    clean = run_attention(case, window=window)
    kb, vb, ks, vs = k.clone().view(torch.uint8), v.clone().view(torch.uint8), ks.clone(), vs.clone()
    hidden = 0
    for r, n in enumerate(lengths):
        low = n - (fresh[r] if fresh else 1) + 1 - window  # the first token that the first query sees
        for page in table[r, :max(0, low) // bs].tolist():
            kb[page] = vb[page] = 0x7F  # NaN in e4m3
            ks[page] = vs[page] = float("nan")
            hidden += 1
    assert hidden
    dirty = run_attention((q, kb.view(k.dtype), vb.view(v.dtype), ks, vs, table, lengths, starts), window=window)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("hq,kv,dim", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("window", [0, 2, 2 ** 31 - 100, 2 ** 31 - 1])
def test_attention_of_more_queries_than_tokens_and_the_largest_windows(hq, kv, dim, window):
    """Queries that stand before a request's first token see none; a window of any size hides no more than it says."""
    check_attention(attention_case([2, 40, 3, 0, 0, 70], [5, 3, 9, 2, 3, 1], hq, kv, dim, 16, "int8", "fp16", seed=dim), window=window)
