"""Refusals of the decode-step operators (cache plan, append, attention, block
norm) that need no device: bad shapes, types, strides and pointers come back as
a status from the C ABI, and CPU tensors raise from the package."""

from __future__ import annotations

import ctypes

import pytest
import torch

import decode_kernel as dk
from decode_kernel import capi


def cache(**kw) -> capi.Cache8:
    c = capi.Cache8(k=1024, v=2048, k_scale=64, v_scale=64, blocks=4, block_size=16, kv_heads=2,
                    head_dim=128, code=capi.DK_INT8, k_block_stride=4096, k_head_stride=2048,
                    k_token_stride=128, v_block_stride=4096, v_head_stride=2048, v_token_stride=128)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def attention_args(**kw) -> capi.CacheAttentionArgs:
    a = capi.CacheAttentionArgs(cache=cache(), q=1024, out=1024, lse=None, dtype=capi.DK_FP16,
                                q_token_stride=1024, q_head_stride=128, block_table=64, max_blocks=4,
                                table_stride=4, lengths=64, starts=None, requests=2, tokens=2,
                                q_heads=8, scale=0.1, causal=1, window=0)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def attention(a, workspace=256, size=1 << 30):
    return capi.load().dk_cache_attention(ctypes.byref(a), workspace, size, None)


@pytest.mark.parametrize("kw", [
    dict(cache=cache(block_size=8)), dict(cache=cache(block_size=272)), dict(cache=cache(block_size=24)),
    dict(cache=cache(blocks=0)), dict(cache=cache(kv_heads=0)), dict(cache=cache(kv_heads=3)),
    dict(cache=cache(code=capi.DK_FP16)), dict(cache=cache(k_token_stride=136)), dict(cache=cache(v=2056)),
    dict(cache=cache(k=None)), dict(cache=cache(v_head_stride=-2048)),
    dict(dtype=capi.DK_FP32), dict(q=1032), dict(q=None), dict(out=None), dict(q_token_stride=1020),
    dict(block_table=None), dict(lengths=None), dict(max_blocks=0), dict(requests=-1), dict(tokens=3),
    dict(window=-1), dict(window=4, causal=0), dict(q_heads=0),
])
def test_attention_rejects(kw):
    assert attention(attention_args(**kw)) == capi.DK_ERR_INVALID_ARG


def test_attention_refuses_what_it_has_no_kernel_for():
    assert attention(attention_args(cache=cache(head_dim=96))) == capi.DK_ERR_UNSUPPORTED
    assert attention(attention_args(max_blocks=1 << 27)) == capi.DK_ERR_UNSUPPORTED
    need = capi.load().dk_cache_attention_workspace_bytes(128)
    assert need > 0
    assert attention(attention_args(), 0) == capi.DK_ERR_WORKSPACE
    assert attention(attention_args(), 256, need - 1) == capi.DK_ERR_WORKSPACE
    assert attention(attention_args(), 128) == capi.DK_ERR_WORKSPACE  # not 256-byte aligned
    assert capi.load().dk_cache_attention_workspace_bytes(96) == 0
    assert capi.load().dk_cache_attention(None, 256, need, None) == capi.DK_ERR_INVALID_ARG


def test_attention_of_nothing_is_a_noop():
    assert attention(attention_args(requests=0, tokens=0)) == capi.DK_OK
    assert attention(attention_args(requests=2, tokens=0, starts=64)) == capi.DK_OK


def append(c, k=256, v=256, dtype=capi.DK_FP16, tokens=2, strides=(256, 128, 256, 128), slots=64):
    return capi.load().dk_cache_append(ctypes.byref(c) if c else None, k, v, dtype, tokens, *strides, slots, None)


@pytest.mark.parametrize("kw", [
    dict(c=None), dict(c=cache(block_size=20)), dict(c=cache(code=capi.DK_BF16)), dict(c=cache(v_token_stride=100)),
    dict(dtype=capi.DK_FP32), dict(tokens=-1), dict(k=None), dict(slots=None), dict(strides=(254, 128, 256, 128)),
    dict(v=260), dict(c=cache(k_scale=None)),
])
def test_append_rejects(kw):
    kw.setdefault("c", cache())
    assert append(**kw) == capi.DK_ERR_INVALID_ARG


def test_append_refuses_and_noop():
    assert append(cache(head_dim=96)) == capi.DK_ERR_UNSUPPORTED
    assert append(cache(), tokens=0) == capi.DK_OK


def plan(held=64, fresh=64, requests=4, table=64, width=4, stride=4, block=16, free=64, capacity=8, ring=64,
         ring_out=128, lengths=256, starts=64, slots=64, tokens=8):
    return capi.load().dk_cache_plan(held, fresh, requests, table, width, stride, block, free, capacity, ring,
                                     ring_out, lengths, starts, slots, tokens, None)


@pytest.mark.parametrize("kw", [
    dict(requests=-1), dict(width=0), dict(stride=3), dict(block=0), dict(block=264), dict(block=17),
    dict(capacity=-1), dict(tokens=-1), dict(held=None), dict(fresh=None), dict(table=None), dict(free=None),
    dict(ring=None), dict(ring_out=None), dict(lengths=None), dict(starts=None), dict(slots=None),
])
def test_plan_rejects(kw):
    assert plan(**kw) == capi.DK_ERR_INVALID_ARG


def test_plan_refuses_more_requests_than_it_sums_up():
    assert plan(requests=capi.DK_PLAN_MAX_REQUESTS + 1) == capi.DK_ERR_UNSUPPORTED


def norm(**kw):
    a = capi.BlockNormArgs(residual=256, y=256, gate=None, post_weight=None, post_bias=None, pre_weight=256,
                           pre_bias=None, residual_out=256, h=256, residual_stride=64, y_stride=64, gate_stride=0,
                           gate_column_stride=1, residual_out_stride=64, h_stride=64, rows=2, dim=64,
                           dtype=capi.DK_FP16, residual_dtype=capi.DK_FP16, kind=0, act=0, residual_scale=1,
                           block_scale=1, eps=1e-6)
    for name, value in kw.items():
        setattr(a, name, value)
    return capi.load().dk_block_norm(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(dim=0), dict(gate_column_stride=2), dict(dtype=capi.DK_FP32), dict(residual_dtype=capi.DK_BF16),
    dict(kind=2), dict(act=3), dict(y=None, gate=256), dict(y=None, post_weight=256), dict(post_bias=256),
    dict(pre_weight=None), dict(pre_weight=None, pre_bias=256, h=None), dict(residual=None),
    dict(residual_out=None, h=None),
])
def test_norm_rejects(kw):
    assert norm(**kw) == capi.DK_ERR_INVALID_ARG


def test_norm_refuses_and_noop():
    assert norm(dim=32769) == capi.DK_ERR_UNSUPPORTED
    assert norm(rows=0) == capi.DK_OK


def test_no_cpu_fallback():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        dk.block_norm(x, x, pre_weight=x[0])
    with pytest.raises(ValueError, match="kind"):
        dk.block_norm(x, x, kind="batch")
    with pytest.raises(ValueError, match="gate_act"):
        dk.block_norm(x, x, gate_act="tanh")
    with pytest.raises(RuntimeError, match="CUDA"):
        dk.PagedCache8(2, 16, 1, 64, device="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        dk.cache_plan(i, i, i.view(2, 1), i, torch.zeros(4, dtype=torch.int64), 16, 2)
