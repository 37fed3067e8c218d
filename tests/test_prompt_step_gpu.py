"""The example's decoder with its prompt operators: prompts of many rows through
the products, requests that move to a second server's pages, and its rotary
positions against a plain turning."""

from __future__ import annotations

import pytest
import torch

from test_decode_step_gpu import example, plain_logits

pytestmark = pytest.mark.gpu


def test_rotate_is_a_plain_turning():
    model = example().Decoder(layers=1, dim=256, heads=4, kv_heads=2, head_dim=64, hidden=512, vocab=512)
    x = torch.randn(50, 4, 64, device="cuda").half()
    positions = torch.arange(1000, 1050, device="cuda")
    angle = positions.double()[:, None, None] * model.frequency.double()
    a, b = x.double().chunk(2, -1)
    want = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)
    # Half a step of fp16, and 2^-21 of the pair for the sines and cosines.
    bound = want.abs() * 2.0 ** -11 + torch.cat([a.abs() + b.abs()] * 2, -1) * 2.0 ** -21 + 2.0 ** -25
    assert ((model.rotate(x, positions).double() - want).abs() <= bound).all()


@pytest.mark.parametrize("first,second", [(torch.int8, torch.float8_e4m3fn), (torch.float8_e4m3fn, torch.int8)])
def test_requests_move_to_another_servers_pages(first, second):
    m = example()
    model = m.Decoder(layers=2, dim=256, heads=4, kv_heads=2, head_dim=64, hidden=512, vocab=512)
    prompts = [[3], list(range(40)), list(range(100, 115)), list(range(200, 333))]
    server = m.Server(model, len(prompts), blocks=40, block_size=16, max_blocks=12, code=first)
    seqs = [list(p) for p in prompts]
    server.tokens.copy_(server.prefill(prompts).argmax(-1))

    def steps(n):
        for _ in range(n):
            for s, t in zip(seqs, server.tokens.tolist()):
                s.append(t)
            logits = server.decode()
        return logits

    steps(3)
    held = server.held.tolist()
    moved = m.Server(model, len(prompts), blocks=30, block_size=48, max_blocks=8, code=second)
    moved.take_over(server)
    server = moved
    assert server.held.tolist() == held
    logits = steps(6)
    # As for one server (its share of the logits is that of the coarser code, e4m3), and a second rounding beside the first.
    for r, s in enumerate(seqs):
        want = plain_logits(model, s)
        assert (logits[r].float() - want).norm() <= (0.12 + 0.03) * want.norm(), r
    assert server.held.tolist() == [len(s) for s in seqs]
    assert server.ring[2:].tolist() == [0, 0]
