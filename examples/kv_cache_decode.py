"""One attention layer of a serving loop: INT4 projections beside a 4-bit
key/value cache.

    python examples/kv_cache_decode.py [--requests 8] [--steps 32] ...

Ragged prompts go through the layer in one step, then every request decodes a
token at a time:

    h -> int4_linear (q, k, v) -> append (rotates q and k, writes k and v)
      -> attention over the paged cache -> int4_linear

with the pages of a request handed out as it grows.  Decoding steps are
captured once into a CUDA graph and replayed: the graph reads the lengths and
the page table, which the loop updates in place.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from openquant_b200.groupwise import quantize_int4_groupwise  # noqa: E402
from openquant_b200.kv_cache import Int4KVCache, KVBatch, rotary_table  # noqa: E402
from openquant_b200.triton_int4 import Int4Linear  # noqa: E402


class Attention:
    """The layer: its two quantized projections, its cache and its rotary table."""

    def __init__(self, heads, kv_heads, head_dim, pages, page_size, max_positions, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        hidden = heads * head_dim

        def linear(rows):
            w = torch.randn(rows, hidden, device="cuda", generator=gen) * hidden**-0.5
            q = quantize_int4_groupwise(w, 128)
            return Int4Linear(q.data, q.scales, rows, 128, out_dtype=torch.float16, static_weights=True)

        self.qkv, self.out = linear((heads + 2 * kv_heads) * head_dim), linear(hidden)
        self.cache = Int4KVCache.allocate(pages, page_size, kv_heads, head_dim)
        self.table = rotary_table(max_positions, head_dim)

    def __call__(self, h, batch):
        d = self.head_dim
        q, k, v = (x.unflatten(1, (-1, d))  # views of the fused projection: nothing is copied
                   for x in self.qkv(h).split([self.heads * d, self.kv_heads * d, self.kv_heads * d], 1))
        q = self.cache.append(k, v, batch, q=q, table=self.table)
        y = self.cache.attention(q, batch)
        self.last = q, y
        return self.out(y.flatten(1))


def run(requests=8, prompt=200, steps=32, heads=16, kv_heads=4, head_dim=64, page_size=32, seed=0):
    """Returns the layer, the batch of the last step and seconds per decoding step."""
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.randint(1, prompt + 1, (requests,), generator=gen, dtype=torch.int32)
    most = int(lengths.max()) + steps
    slots = -(-most // page_size)
    layer = Attention(heads, kv_heads, head_dim, requests * slots, page_size, most, seed)
    free = torch.randperm(requests * slots, generator=gen).tolist()
    pages = torch.zeros(requests, slots, dtype=torch.int32)
    owned = [0] * requests

    def grow(b, n):
        while owned[b] * page_size < n:
            pages[b, owned[b]] = free.pop()
            owned[b] += 1

    # the prompts, all in one step
    for b, n in enumerate(lengths.tolist()):
        grow(b, n)
    starts = torch.cat([torch.zeros(1, dtype=torch.int32), lengths.cumsum(0, dtype=torch.int32)])
    h = torch.randn(int(lengths.sum()), heads * head_dim, generator=gen).half().cuda()
    page_table, on_gpu = pages.cuda(), lengths.cuda()
    y = layer(h, KVBatch(page_table, on_gpu, starts.cuda(), max_tokens=int(lengths.max())))

    # decoding: one token a request, fed back
    batch = KVBatch(page_table, on_gpu)
    x = y[starts[1:].long().cuda() - 1].contiguous()

    def step():
        x.copy_(layer(x, batch))

    def advance():
        lengths.add_(1)
        for b, n in enumerate(lengths.tolist()):
            grow(b, n)
        page_table.copy_(pages)
        on_gpu.copy_(lengths)

    advance()
    step()  # kernels are loaded before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    began = time.perf_counter()
    for _ in range(steps - 1):
        advance()
        graph.replay()
    torch.cuda.synchronize()
    return layer, batch, (time.perf_counter() - began) / max(steps - 1, 1)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("requests", 8), ("prompt", 200), ("steps", 32), ("heads", 16), ("kv-heads", 4),
                          ("head-dim", 64), ("page-size", 32)):
        ap.add_argument("--" + name, type=int, default=default)
    args = vars(ap.parse_args(argv))
    layer, batch, seconds = run(**args)
    c = layer.cache
    held = sum(t.numel() * t.element_size() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales))
    print(f"{args['requests']} requests, {args['steps']} tokens each: {seconds * 1e6:.1f} us a step of this layer; "
          f"cache of {c.pages} pages x {c.page_size} tokens: {held / 2**20:.1f} MiB "
          f"({held / (c.pages * c.page_size * c.kv_heads * c.head_dim * 4):.3f} of fp16)")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
