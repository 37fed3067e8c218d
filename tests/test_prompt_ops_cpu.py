"""Refusals of the prompt operators (many-row products and their gradients,
rotary positions, the cache read back) that need no device: bad shapes, types,
strides and pointers come back as a status from the C ABI, and CPU tensors and
bad arguments raise from the package."""

from __future__ import annotations

import ctypes

import pytest
import torch

import decode_kernel as dk
from decode_kernel import capi
from test_decode_ops_cpu import cache


def gemm_args(**kw) -> capi.GemmArgs:
    a = capi.GemmArgs(packed=1024, scales=64, x=1024, y=1024, ldx=256, ldy=64, ldk=64, rows=4, M=64, K=256, dtype=capi.DK_FP16, act=0)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    dict(K=200), dict(K=0), dict(rows=-1), dict(M=-1), dict(dtype=capi.DK_FP32), dict(act=2), dict(packed=None), dict(scales=None),
    dict(x=None), dict(y=None), dict(packed=1032), dict(x=1032), dict(ldx=248), dict(ldx=260), dict(ldy=63),
    dict(packed2=1024), dict(scales2=64), dict(packed2=1032, scales2=64), dict(packed2=1024, scales2=64, gate_out=64),
    dict(gate_out=64, up_out=64), dict(packed2=1024, scales2=64, gate_out=64, up_out=64, ldk=60),
])
def test_gemm_rejects(kw):
    assert capi.load().dk_w4a16_gemm(ctypes.byref(gemm_args(**kw)), None) == capi.DK_ERR_INVALID_ARG


def gemm_t_args(**kw) -> capi.GemmTArgs:
    a = capi.GemmTArgs(packed=1024, scales=64, g=1024, dx=1024, ldg=64, lddx=256, rows=4, M=64, K=256, dtype=capi.DK_BF16)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    dict(K=200), dict(rows=-1), dict(M=0), dict(dtype=capi.DK_INT8), dict(packed=None), dict(scales=None), dict(g=None), dict(dx=None),
    dict(packed=1032), dict(g=1032), dict(ldg=60), dict(ldg=68), dict(lddx=255), dict(packed2=1024, scales2=64), dict(g2=1024),
    dict(packed2=1024, scales2=64, g2=1032),
])
def test_gemm_t_rejects(kw):
    assert capi.load().dk_w4a16_gemm_t(ctypes.byref(gemm_t_args(**kw)), None) == capi.DK_ERR_INVALID_ARG


def test_few_rows_need_a_workspace():
    need = capi.load().dk_w4a16_gemm_workspace_bytes
    assert need(1, 256, 1, capi.DK_FP16) > 0 and need(16, 256, 1, capi.DK_BF16) > 0 and need(32, 256, 2, capi.DK_BF16) > 0
    for bad in ((17, 256, 1, capi.DK_FP16), (33, 256, 2, capi.DK_FP16), (0, 256, 1, capi.DK_FP16), (1, 200, 1, capi.DK_FP16), (1, 256, 1, capi.DK_FP32),
                (1, 256, 0, capi.DK_FP16), (1, 256, 3, capi.DK_FP16)):
        assert need(*bad) == 0
    size = need(4, 256, 1, capi.DK_FP16)
    for kw in (dict(), dict(workspace=1024, workspace_bytes=size - 1), dict(workspace=1088, workspace_bytes=size)):
        assert capi.load().dk_w4a16_gemm(ctypes.byref(gemm_args(**kw)), None) == capi.DK_ERR_WORKSPACE


def test_empty_products_are_noops():
    lib = capi.load()
    assert lib.dk_w4a16_gemm(None, None) == capi.DK_ERR_INVALID_ARG
    assert lib.dk_w4a16_gemm_t(None, None) == capi.DK_ERR_INVALID_ARG
    assert lib.dk_w4a16_gemm(ctypes.byref(gemm_args(rows=0)), None) == capi.DK_OK
    assert lib.dk_w4a16_gemm(ctypes.byref(gemm_args(M=0)), None) == capi.DK_OK
    assert lib.dk_w4a16_gemm_t(ctypes.byref(gemm_t_args(rows=0)), None) == capi.DK_OK
    assert lib.dk_w4a16_gemm_t(ctypes.byref(gemm_t_args(K=0)), None) == capi.DK_OK


def gated_grad(dh=64, g=64, u=64, dg=64, du=64, rows=2, M=8, ld=(8, 8, 8), dtype=capi.DK_FP16, act=0):
    return capi.load().dk_gated_grad(dh, g, u, dg, du, rows, M, *ld, dtype, act, None)


@pytest.mark.parametrize("kw", [dict(dh=None), dict(g=None), dict(u=None), dict(dg=None), dict(du=None), dict(rows=-1), dict(M=-1),
                                dict(ld=(7, 8, 8)), dict(ld=(8, 7, 8)), dict(ld=(8, 8, 7)), dict(dtype=capi.DK_FP32), dict(act=-1)])
def test_gated_grad_rejects(kw):
    assert gated_grad(**kw) == capi.DK_ERR_INVALID_ARG
    assert gated_grad(rows=0) == capi.DK_OK and gated_grad(M=0) == capi.DK_OK


def rotary_args(**kw) -> capi.RotaryArgs:
    ends = kw.pop("section_end", (16, 32, 64, 0))
    a = capi.RotaryArgs(q=1024, k=1024, q_out=2048, k_out=2048, q_token_stride=512, q_head_stride=128, k_token_stride=256, k_head_stride=128,
                        q_out_token_stride=512, q_out_head_stride=128, k_out_token_stride=256, k_out_head_stride=128, positions=64, frequency=64,
                        position_stride=3, tokens=3, q_heads=4, kv_heads=2, head_dim=128, pairs=64, axes=3, dtype=capi.DK_FP16)
    a.section_end = (ctypes.c_int * 4)(*ends)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    dict(tokens=-1), dict(q_heads=0), dict(kv_heads=-1), dict(head_dim=1), dict(pairs=0), dict(pairs=65), dict(axes=0), dict(axes=5),
    dict(dtype=capi.DK_INT8), dict(section_end=(32, 16, 64, 0)), dict(section_end=(16, 32, 63, 0)), dict(q=None), dict(q_out=None),
    dict(k_out=None), dict(positions=None), dict(frequency=None), dict(q=1025), dict(k_out=2049),
])
def test_rotary_rejects(kw):
    assert capi.load().dk_rotary(ctypes.byref(rotary_args(**kw)), None) == capi.DK_ERR_INVALID_ARG


def test_rotary_refuses_what_it_has_no_kernel_for():
    lib = capi.load()
    assert lib.dk_rotary(None, None) == capi.DK_ERR_INVALID_ARG
    assert lib.dk_rotary(ctypes.byref(rotary_args(head_dim=1026)), None) == capi.DK_ERR_UNSUPPORTED
    assert lib.dk_rotary(ctypes.byref(rotary_args(q_heads=1 << 20)), None) == capi.DK_ERR_UNSUPPORTED
    assert lib.dk_rotary(ctypes.byref(rotary_args(tokens=0)), None) == capi.DK_OK


def read_args(**kw) -> capi.CacheReadArgs:
    a = capi.CacheReadArgs(cache=cache(), block_table=64, max_blocks=4, table_stride=4, lengths=64, starts=64, requests=2, tokens=9, k=1024,
                           v=2048, k_token_stride=256, v_token_stride=256, dtype=capi.DK_FP16)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    dict(cache=cache(block_size=8)), dict(cache=cache(block_size=24)), dict(cache=cache(blocks=0)), dict(cache=cache(kv_heads=0)),
    dict(cache=cache(code=capi.DK_FP16)), dict(cache=cache(k_token_stride=136)), dict(cache=cache(v=2056)), dict(cache=cache(k=None)),
    dict(cache=cache(v_scale=None)), dict(cache=cache(v_head_stride=-2048)), dict(dtype=capi.DK_FP32), dict(k=None), dict(v=None),
    dict(k=1032), dict(v_token_stride=260), dict(block_table=None), dict(lengths=None), dict(starts=None), dict(max_blocks=0),
    dict(table_stride=3), dict(requests=-1), dict(tokens=-1),
])
def test_read_rejects(kw):
    assert capi.load().dk_cache_read(ctypes.byref(read_args(**kw)), None) == capi.DK_ERR_INVALID_ARG


def test_read_refuses_what_it_has_no_kernel_for():
    lib = capi.load()
    assert lib.dk_cache_read(None, None) == capi.DK_ERR_INVALID_ARG
    assert lib.dk_cache_read(ctypes.byref(read_args(cache=cache(head_dim=96))), None) == capi.DK_ERR_UNSUPPORTED
    assert lib.dk_cache_read(ctypes.byref(read_args(tokens=0)), None) == capi.DK_OK
    assert lib.dk_cache_read(ctypes.byref(read_args(requests=0)), None) == capi.DK_OK


def test_cpu_tensors_raise():
    packed, scales = torch.zeros(64, 32, dtype=torch.int32), torch.zeros(64, 2, dtype=torch.float16)
    x, g = torch.zeros(3, 256, dtype=torch.float16), torch.zeros(3, 64, dtype=torch.float16)
    for call in (lambda: dk.gemm(packed, scales, x), lambda: dk.gemm_t(packed, scales, g),
                 lambda: dk.gemm_gated((packed, scales), (packed, scales), x),
                 lambda: dk.gemm(packed, scales, x.requires_grad_()),
                 lambda: dk.rotary(torch.zeros(3, 2, 8), None, torch.zeros(3, dtype=torch.int32), torch.ones(4))):
        with pytest.raises(RuntimeError):
            call()


def test_bad_arguments_raise_before_the_device():
    packed, scales = torch.zeros(64, 32, dtype=torch.int32), torch.zeros(64, 2, dtype=torch.float16)
    x = torch.zeros(3, 256, dtype=torch.float16)
    with pytest.raises(ValueError):
        dk.gemm_gated((packed, scales), (packed, scales), x, act="relu")
    with pytest.raises(RuntimeError, match="frozen"):
        dk.gemm(packed, scales.clone().requires_grad_(), x)
    with pytest.raises(RuntimeError, match="frequency"):
        dk.rotary(torch.zeros(3, 2, 8), None, torch.zeros(3, dtype=torch.int32), torch.ones(4, requires_grad=True))
    with pytest.raises(RuntimeError, match="in place"):
        dk.rotary(torch.zeros(3, 2, 8, requires_grad=True), None, torch.zeros(3, dtype=torch.int32), torch.ones(4), inplace=True)
    lin = lambda m, k: dk.W4A16Linear(torch.zeros(m, k // 8, dtype=torch.int32), torch.zeros(m, k // 128, dtype=torch.float16))  # noqa: E731
    with pytest.raises(ValueError):
        dk.W4A16GatedMLP(lin(128, 256), lin(256, 256), lin(256, 128))
    with pytest.raises(ValueError):
        dk.W4A16GatedMLP(lin(128, 256), lin(128, 256), lin(256, 128), act="relu")


@pytest.mark.parametrize("call", [
    *(lambda kw=kw: capi.load().dk_w4a16_gemm(ctypes.byref(gemm_args(rows=40, **kw)), None) for kw in (
        dict(scales=65), dict(y=1025), dict(packed2=1024, scales2=65), dict(packed2=1024, scales2=64, gate_out=65, up_out=64),
        dict(packed2=1024, scales2=64, gate_out=64, up_out=65))),
    *(lambda kw=kw: capi.load().dk_w4a16_gemm_t(ctypes.byref(gemm_t_args(**kw)), None) for kw in (
        dict(scales=65), dict(dx=1025), dict(packed2=1024, scales2=65, g2=1024))),
    *(lambda kw=kw: gated_grad(**kw) for kw in (dict(dh=65), dict(g=65), dict(u=65), dict(dg=65), dict(du=65))),
    *(lambda kw=kw: capi.load().dk_rotary(ctypes.byref(rotary_args(**kw)), None) for kw in (
        dict(positions=66), dict(positions=68, positions_64=1), dict(frequency=66))),
    *(lambda kw=kw: capi.load().dk_cache_read(ctypes.byref(read_args(**kw)), None) for kw in (
        dict(block_table=66), dict(lengths=66), dict(starts=66), dict(cache=cache(k_scale=66)), dict(cache=cache(v_scale=66)))),
])
def test_addresses_between_values_are_refused(call):
    assert call() == capi.DK_ERR_INVALID_ARG
