"""Edges of the prompt operators: token tiles that end behind the last row while
memory is busy, outputs beside their inputs, rounding against the weights as
they are, gradients at the ends of the types' range, and what they refuse."""

from __future__ import annotations

import pytest
import torch

import decode_kernel as dk
from decode_kernel import _cuda
from test_prompt_ops_gpu import check_product, rows_of, values, weights

pytestmark = pytest.mark.gpu

# Rows, outputs and width of calls whose results leave in boxes, and how many of the last token tile's boxes of 32 tokens
# no row reaches (on 148 SMs).  Odd numbers of output tiles leave a pair's second half without outputs.
BOXED = [
    ("plain", 1100, 4096, 640, 1), ("plain", 1044, 2176, 256, 2), ("plain", 1044, 2048, 1024, 3), ("plain", 4096, 4096, 4096, 4),
    ("plain", 5000, 1024, 256, 3), ("plain", 1000, 4096, 4096, 0), ("gated", 2500, 2112, 128, 1), ("gated", 300, 2816, 1024, 2), ("gated", 900, 2048, 256, 3),
    ("gated", 4096, 11008, 4096, 4), ("kept", 1300, 1088, 384, 1), ("kept", 700, 1104, 2048, 2), ("kept", 900, 2048, 256, 3),
    ("transposed", 200, 256, 18944, 1), ("transposed", 700, 1100, 2048, 2), ("transposed", 900, 512, 4224, 3), ("transposed", 1300, 256, 4096, 4),
]


@pytest.mark.parametrize("mode,T,M,K,empty", BOXED)
def test_results_in_boxes_do_not_depend_on_the_run(mode, T, M, K, empty):
    w, w2 = weights(M, K, T), weights(M, K, T + 1)
    x = rows_of(T, M if mode == "transposed" else K, torch.float16, T + 2)
    call = {"plain": lambda: (dk.gemm(*w, x),), "gated": lambda: (dk.gemm_gated(w, w2, x),), "kept": lambda: _cuda.w4a16_gemm(*w, *w2, x, 0, True),
            "transposed": lambda: (dk.gemm_t(*w, x),)}[mode]
    first = [t.clone() for t in call()]
    if mode == "plain":
        check_product(first[0], x, values(w, x.dtype, T).t(), depth=K)
    elif mode == "transposed":
        check_product(first[0], x, values(w, x.dtype), depth=M)
    elif mode == "kept":
        for got, v in zip(first[1:], (w, w2)):
            check_product(got, x, values(v, x.dtype, T, 32).t(), depth=K)
    # Copies on another stream keep the memory busy: a store takes longer to read its box.
    side, room = torch.cuda.Stream(), torch.empty(2, 1 << 27, dtype=torch.uint8, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(400):
        if i % 4 == 0:
            with torch.cuda.stream(side):
                room[1].copy_(room[0])
        for a, b in zip(first, call()):
            wrong += (a != b).sum()
    assert int(wrong) == 0
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("rows", [1, 31, 33, 64, 95, 97, 160, 191, 193, 255, 257])
@pytest.mark.parametrize("mode", ["plain", "kept", "transposed"])
def test_rows_at_the_boxes_edges(mode, rows):
    """The last row of a tile is the last that is written, for whole and odd numbers of output tiles."""
    M, K, T = (640, 512, 1344 + rows) if mode != "transposed" else (384, 640, 1344 + rows)
    w, w2 = weights(M, K, rows), weights(M, K, rows + 1)
    x = rows_of(T, M if mode == "transposed" else K, torch.bfloat16, rows + 2)
    wide = torch.full((T + 40, M if mode != "transposed" else K), 7.0, dtype=torch.bfloat16, device="cuda")
    if mode == "plain":
        check_product(dk.gemm(*w, x, out=wide[:T]), x, values(w, x.dtype, T).t(), depth=K)
    elif mode == "transposed":
        check_product(dk.gemm_t(*w, x, out=wide[:T]), x, values(w, x.dtype), depth=M)
    else:
        h, g, u = _cuda.w4a16_gemm(*w, *w2, x, 0, True, wide[:T])
        for got, v in ((g, w), (u, w2)):
            check_product(got, x, values(v, x.dtype, T, 32).t(), depth=K)
        assert torch.equal(h, dk.gemm_gated(w, w2, x))
    assert (wide[T:] == 7).all()
