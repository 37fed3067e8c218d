"""Limits of the decode-step operators that the C ABI checks before any launch."""

from __future__ import annotations

import ctypes

import pytest

from decode_kernel import capi
from test_decode_ops_cpu import attention_args, cache


def attention_status(**kw):
    """The call's status without a workspace: DK_ERR_WORKSPACE where nothing but that is missing."""
    a = attention_args(**kw)
    return capi.load().dk_cache_attention(ctypes.byref(a), None, 0, None)


def prompts(rows, width, requests=64, q_heads=64, kv_heads=8, **kw):
    return dict(cache=cache(block_size=64, kv_heads=kv_heads, **kw), q_heads=q_heads, starts=64, requests=requests, tokens=rows, max_blocks=width // 64,
                table_stride=width // 64)


@pytest.mark.parametrize("kw", [
    prompts(16384, 131072), prompts(65536, 131072), prompts(16384, 1 << 20, requests=8), prompts(1 << 20, 8192, requests=4096),
    prompts(16384, 131072, head_dim=64), prompts(16384, 131072, head_dim=256), prompts(1, 1 << 30, requests=1, q_heads=640, kv_heads=80),
])
def test_attention_takes_wide_tables_and_many_rows(kw):
    assert attention_status(**kw) == capi.DK_ERR_WORKSPACE


@pytest.mark.parametrize("kw", [
    prompts(1 << 20, 1 << 20), prompts(1024, 1 << 30, requests=1024), prompts(1 << 26, 64), prompts(1, (1 << 31) - 64, requests=1),
])
def test_attention_refuses_lines_past_32_bits(kw):
    assert attention_status(**kw) == capi.DK_ERR_UNSUPPORTED
