"""The example's decoder, served from the paged 8-bit cache, against the same
decoder with plain norms and plain attention over unquantised keys and values."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

import decode_kernel as dk

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "decode_step.py"
    spec = importlib.util.spec_from_file_location("decode_step", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_logits(model, sequence):
    """The last row's logits for one request's whole sequence, fp32 between the products."""
    n, d = len(sequence), model.head_dim
    positions = torch.arange(n, device="cuda")
    norm = lambda r, w: (r.float() / torch.sqrt(r.float().square().mean(-1, keepdim=True) + 1e-6) * w.float()).half()  # noqa: E731
    product = lambda w, x: (x.float() @ dk.dequantize(*[t.cpu() for t in w]).cuda().t()).half()  # noqa: E731
    r = model.embedding[torch.tensor(sequence, device="cuda")]
    mask = torch.full((n, n), -math.inf, device="cuda").triu(1)
    for w in model.layers:
        h = norm(r, w["norm1"])
        q, k, v = (product(w[x], h).view(n, -1, d) for x in "qkv")
        q, k = model.rotate(q, positions).float(), model.rotate(k, positions).float()
        k, v = (x.float().repeat_interleave(model.heads // model.kv_heads, 1) for x in (k, v))
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5 + mask, -1)
        r = r + product(w["o"], torch.einsum("hqk,khd->qhd", p, v).half().reshape(n, -1))
        h = norm(r, w["norm2"])
        gate = product(w["gate"], h).float()
        r = r + product(w["down"], (gate * torch.sigmoid(gate) * product(w["up"], h).float()).half())
    return product(model.head, norm(r, model.norm))[-1].float()


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_served_decoder_follows_the_plain_one(code):
    m = example()
    model = m.Decoder(layers=2, dim=256, heads=4, kv_heads=2, head_dim=64, hidden=512, vocab=512)
    prompts = [[3], list(range(40)), list(range(100, 115)), list(range(200, 333))]
    server = m.Server(model, len(prompts), blocks=40, block_size=16, max_blocks=12, code=code)
    seqs = [list(p) for p in prompts]
    # int8 keys and values are 2^-8 of their page's largest off, e4m3 ones 2^-4 of themselves, at random and averaged
    # by the attention: the logits' share is a few times that of one layer's relative error.
    share = 0.03 if code == torch.int8 else 0.12

    def check(logits):
        for r, s in enumerate(seqs):
            want = plain_logits(model, s)
            assert (logits[r].float() - want).norm() <= share * want.norm(), r

    logits = server.prefill(prompts)
    check(logits)
    server.tokens.copy_(logits.argmax(-1))
    for _ in range(20):
        for r, t in enumerate(server.tokens.tolist()):
            seqs[r].append(t)
        logits = server.decode()
    check(logits)
    assert server.held.tolist() == [len(s) for s in seqs]
    assert server.ring[2:].tolist() == [0, 0]
