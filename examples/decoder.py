"""A decoder layer on the device: attention over a paged cache, then the mixture-of-experts block.

    python examples/decoder.py [--layers 4] [--requests 8] [--tokens 64]

Prompts of several requests are taken in, in chunks, then one token after another is decoded, each step
as one CUDA graph: pages and slots for the new tokens (``PagedCache.extend``, once a step), and in every
layer rotary positions with the store into the pages, attention, and the expert block on the residual.
Weights are random; the projections around the attention are plain torch products.
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from biv_b200 import workloads as W                      # noqa: E402
from biv_b200.cache import PagedCache, Rope              # noqa: E402
from biv_b200.moe import Moe, MoeStack                   # noqa: E402

EPS = 1e-6


def rms_norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


class Layer:
    """Attention half and expert half of one layer; every second layer sees a window and four first tokens."""

    def __init__(self, cache: PagedCache, n_pages: int, moe: Moe, window: int, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cache, self.window = cache, window
        self.k_pool, self.v_pool = cache.pools(n_pages)
        e, d, rows = moe.n_embd, cache.head_dim, cache.n_head + 2 * cache.n_head_kv
        new = lambda *shape: (torch.randn(shape, generator=g, device="cuda") / shape[0] ** 0.5).to(cache.dtype)  # noqa: E731
        self.qkv, self.out = new(e, rows * d), new(cache.n_head * d, e)
        self.norm = torch.ones(e, device="cuda")
        moe.set_post_norm(np.ones(e, np.float32), EPS)
        self.ffn = MoeStack([moe])

    def attention(self, x, step, table, max_new):
        c = self.cache
        rows = (rms_norm(x, self.norm).to(c.dtype) @ self.qkv).view(x.shape[0], -1, c.head_dim)
        q, k, v = rows.split_with_sizes((c.n_head, c.n_head_kv, c.n_head_kv), 1)
        q = c.store(q, k, v, self.k_pool, self.v_pool, step.slots, step.positions)
        o = c.attend(q, self.k_pool, self.v_pool, table, step.first, step.length, max_new=max_new,
                     window=self.window, sinks=4 if self.window else 0)
        return (o.view(x.shape[0], -1) @ self.out).float()

    def forward_(self, x, step, table, max_new):
        x += self.attention(x, step, table, max_new)
        return self.ffn.forward_(x)


class Decoder:
    def __init__(self, layers=2, requests=4, max_tokens=512, n_pages=512, page_size=16, heads=8, heads_kv=2, head_dim=64,
                 window=128, seed=0):
        wl = W.decode_q4k(n=1, n_embd=512, n_expert=32, k=4, ff=256, ff_sh=256)
        self.moe = [Moe(wl.layer, max_tokens) for _ in range(layers)]
        self.cache = PagedCache(heads, heads_kv, head_dim, page_size, requests, max_tokens, rope=Rope(head_dim))
        self.layers = [Layer(self.cache, n_pages, m, window if i % 2 else 0, seed + i) for i, m in enumerate(self.moe)]
        ints = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((requests, n_pages // requests), -1, **ints)
        self.free = torch.arange(n_pages, **ints)
        self.free_count = torch.full((1,), n_pages, **ints)
        self.past = torch.zeros(requests, **ints)
        self.n_embd = self.moe[0].n_embd

    def step(self, x, added, max_new):
        """Rows x [n, n_embd] of `added` new tokens a request through all layers, in place."""
        s = self.cache.extend(self.past, added, self.free, self.free_count, self.table, x.shape[0])
        for layer in self.layers:
            layer.forward_(x, s, self.table, max_new)
        # the step's lists are the next step's: copied, since the graph of a step has its addresses
        self.past.copy_(s.length)
        self.free_count.copy_(s.left[:1])
        return s

    def close(self):
        self.cache.close()
        for m in self.moe:
            m.close()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=64)
    a = ap.parse_args()
    d = Decoder(a.layers, a.requests, n_pages=64 * a.requests)
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = [37 + 61 * (i % 5) for i in range(a.requests)]
    chunk, done = 64, [0] * a.requests
    while any(k < n for k, n in zip(done, lengths)):          # prompts, a chunk of each request at a time
        added = [min(chunk, n - k) for k, n in zip(done, lengths)]
        x = torch.randn((sum(added), d.n_embd), generator=g, device="cuda")
        s = d.step(x, torch.tensor(added, dtype=torch.int32, device="cuda"), max(added))
        done = [k + n for k, n in zip(done, added)]
    rows = x[s.first[1:].long() - 1].contiguous()             # some rows to go on from
    one = torch.ones(a.requests, dtype=torch.int32, device="cuda")
    d.step(rows, one, 1)                                      # as it will run in the graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        last = d.step(rows, one, 1)
    t = time.perf_counter()
    for _ in range(a.tokens):
        graph.replay()
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    d.cache.status()
    left, lost = int(last.left[0]), d.cache.unstored()
    print(f"prompts of {lengths} tokens, then {a.tokens} steps of {a.requests} tokens through {a.layers} layers: "
          f"{t / a.tokens * 1e6:.0f} us a step; lengths {d.past.tolist()}, {left} pages left, {lost} tokens without one, "
          f"rows finite: {bool(rows.isfinite().all())}")
    d.close()


if __name__ == "__main__":
    main()
