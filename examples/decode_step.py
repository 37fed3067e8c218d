"""A small W4A16 decoder served from a paged 8-bit cache.

    PYTHONPATH=decode-kernel_b200 python examples/decode_step.py [--steps 64] [--code int8|e4m3]

Ragged prompts go in as one step (the products of many rows, the gated block in
one kernel), then every request decodes token by token with the whole step --
plan, norms, W4A16 products, rotary positions, append, attention -- replayed as
one CUDA graph: nothing in it waits for the host.  Half-way the requests move to
a second server with other pages: their cache is read back and written into its.
At the end requests end and their pages go back to the free ring.
"""

from __future__ import annotations

import argparse
import math
import time

import torch

import decode_kernel as dk


class Decoder:
    """Pre-norm decoder blocks with grouped-query attention and a gated MLP, random weights."""

    def __init__(self, layers=4, dim=1024, heads=8, kv_heads=2, head_dim=128, hidden=2816, vocab=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def linear(rows, cols):
            return dk.quantize_and_pack_cuda(torch.randn(rows, cols, generator=g, device="cuda") * cols ** -0.5)

        def ones():
            return 1 + 0.1 * torch.randn(dim, generator=g, device="cuda").half()

        self.heads, self.kv_heads, self.head_dim, self.dim = heads, kv_heads, head_dim, dim
        self.embedding = torch.randn(vocab, dim, generator=g, device="cuda").half()
        self.layers = [dict(norm1=ones(), norm2=ones(), q=linear(heads * head_dim, dim), k=linear(kv_heads * head_dim, dim),
                            v=linear(kv_heads * head_dim, dim), o=linear(dim, heads * head_dim), gate=linear(hidden, dim),
                            up=linear(hidden, dim), down=linear(dim, hidden)) for _ in range(layers)]
        self.norm, self.head = ones(), linear(vocab, dim)
        self.frequency = 10000.0 ** (-torch.arange(0, head_dim, 2, device="cuda").float() / head_dim)

    def rotate(self, x, positions):
        return dk.rotary(x, None, positions, self.frequency)[0]

    def step(self, tokens, positions, attend):
        """Logits of every row; attend(layer, q, k, v) keeps k and v and returns the attention's output."""
        n = tokens.shape[0]
        r = self.embedding[tokens]
        _, h = dk.block_norm(r, pre_weight=self.layers[0]["norm1"])
        many = n > 8  # prompts and batches; a few rows go by the GEMV's launches of several matrices
        product = dk.gemm if many else dk.gemv
        for i, w in enumerate(self.layers):
            parts = [w["q"], w["k"], w["v"]]
            q, k, v = (x.view(n, -1, self.head_dim) for x in ([dk.gemm(*p, h) for p in parts] if many else dk.gemv_multi(parts, h)))
            dk.rotary(q, k, positions, self.frequency, inplace=True)
            a = attend(i, q, k, v)
            r, h = dk.block_norm(r, product(*w["o"], a.reshape(n, -1)), pre_weight=w["norm2"])
            y = product(*w["down"], (dk.gemm_gated if many else dk.gemv_silu_mul)(w["gate"], w["up"], h))
            after = self.layers[i + 1]["norm1"] if i + 1 < len(self.layers) else self.norm
            r, h = dk.block_norm(r, y, pre_weight=after)
        return product(*self.head, h)


class Server:
    """A decoder's requests over one cache a layer; the pages of all layers share one table."""

    def __init__(self, model, requests, blocks, block_size=64, max_blocks=32, code=torch.int8):
        self.model, self.block_size = model, block_size
        self.caches = [dk.PagedCache8(blocks, block_size, model.kv_heads, model.head_dim, dtype=code) for _ in model.layers]
        self.free, self.ring = self.caches[0].free_list()
        self.held = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.table = torch.full((requests, max_blocks), -1, dtype=torch.int32, device="cuda")
        self.fresh = torch.ones(requests, dtype=torch.int32, device="cuda")
        self.tokens = torch.zeros(requests, dtype=torch.long, device="cuda")
        self.starts = torch.empty(requests + 1, dtype=torch.int32, device="cuda")
        self.graph = None

    def step(self, tokens, fresh, single):
        """One step of all requests: each brings fresh[r] tokens (rows of `tokens`, request after request)."""
        slots = torch.empty(tokens.shape[0], dtype=torch.int64, device="cuda")
        before = self.held.clone()
        plan = dk.cache_plan(self.held, fresh, self.table, self.free, self.ring, self.block_size, tokens.shape[0],
                             out=dk.CachePlan(self.held, self.starts, slots, self.ring))
        row = torch.arange(tokens.shape[0], device="cuda")
        of = row if single else torch.searchsorted(plan.starts[1:].contiguous(), row.int(), right=True)
        positions = before[of] + row - plan.starts[of]

        def attend(layer, q, k, v):
            dk.cache_append(k, v, plan.slots, self.caches[layer])
            return dk.cache_attention(q, self.caches[layer], self.table, plan.lengths, None if single else plan.starts)

        return self.model.step(tokens, positions, attend)

    def prefill(self, prompts):
        """Prompts (lists of tokens, one a request) in one step; returns each one's next token's logits."""
        fresh = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
        tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
        logits = self.step(tokens, fresh, single=False)
        return logits[self.starts[1:].long() - 1]

    def take_over(self, other):
        """The other server's requests: their keys and values read back from its pages and written into this one's, of
        whatever size and type those are.  This server holds none yet, and serves as many."""
        lengths = other.held.clone()
        starts = torch.cat([lengths.new_zeros(1), lengths.cumsum(0, dtype=torch.int32)])
        tokens = int(starts[-1])  # waits for the GPU
        slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        plan = dk.cache_plan(self.held, lengths, self.table, self.free, self.ring, self.block_size, tokens,
                             out=dk.CachePlan(self.held, self.starts, slots, self.ring))
        for mine, theirs in zip(self.caches, other.caches):
            k, v = dk.cache_read(theirs, other.table, lengths, starts, tokens)
            dk.cache_append(k, v, plan.slots, mine)
        self.tokens.copy_(other.tokens)

    def decode(self):
        """One token for every request, from self.tokens; the step is captured once and replayed."""
        if self.graph is None:
            state = [self.held.clone(), self.ring.clone(), self.table.clone(), self.free.clone()]
            caches = [[x.clone() for x in (c.k, c.v, c.k_scale, c.v_scale)] for c in self.caches]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # what a first call sets up must not be captured
                self.step(self.tokens, self.fresh, single=True)
            torch.cuda.current_stream().wait_stream(side)
            for x, y in zip((self.held, self.ring, self.table, self.free), state):
                x.copy_(y)
            for c, kept in zip(self.caches, caches):
                for x, y in zip((c.k, c.v, c.k_scale, c.v_scale), kept):
                    x.copy_(y)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.logits = self.step(self.tokens, self.fresh, single=True)
                self.tokens.copy_(self.logits.argmax(-1))
        self.graph.replay()
        return self.logits


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--code", choices=("int8", "e4m3"), default="int8")
    a = ap.parse_args()
    model = Decoder()
    code = torch.int8 if a.code == "int8" else torch.float8_e4m3fn
    server = Server(model, a.requests, blocks=a.requests * 16, code=code)
    prompts = [[(7 * r + 13 * t) % 4096 for t in range(5 + 37 * r)] for r in range(a.requests)]
    server.tokens.copy_(server.prefill(prompts).argmax(-1))
    server.decode()
    moved = Server(model, a.requests, blocks=a.requests * 24, block_size=32, code=torch.float8_e4m3fn if code == torch.int8 else torch.int8, max_blocks=64)
    moved.take_over(server)
    server = moved
    server.decode()
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.steps):
        server.decode()
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / a.steps
    print(f"{a.requests} requests, {sum(len(p) for p in prompts)} prompt tokens, then {a.steps + 2} steps: {took * 1e6:.0f} us a step "
          f"of {len(model.layers)} layers; lengths {server.held.tolist()}, pages missing {int(server.ring[2])}")
    server.fresh.fill_(-1)  # every request ends
    dk.cache_plan(server.held, server.fresh, server.table, server.free, server.ring, server.block_size, 0,
                  out=dk.CachePlan(server.held, server.starts, torch.empty(0, dtype=torch.int64, device="cuda"), server.ring))
    head, tail = server.ring[:2].tolist()
    print(f"all ended: {tail - head} of {server.caches[0].blocks} pages free")
    assert math.isfinite(float(server.logits.float().abs().max()))


if __name__ == "__main__":
    main()
