"""A server's attention over the paged 8-bit KV cache: requests arrive with a prompt, answer token by token and end. A step makes

    one plan        pages for the step's new tokens, from the requests' lengths before and after it (llmp.paged.plan)
    a layer's store the new tokens' K and V into those pages (llmp.paged.store)
    a layer's attention of the step's queries (llmp.paged.attend), over all that a request holds or, in decode steps with
                    `keep`, over the pages that could hold its largest logits (llmp.paged.select)

The layers share the plan, each with a cache of its own. Activations are synthetic. On an MI355X:

    python examples/paged_server.py
    python examples/paged_server.py --requests 8 --prompt 4000 --pages 1200 --keep 32
"""
import argparse
import math
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from llmp_amd import ops


class PagedServer:
    """`slots` requests at once; a slot without a request has a length of zero."""

    def __init__(self, slots, pages, width, layers=2, heads=32, kv_heads=8, head_dim=128, page=64, keep=0, device="cuda"):
        self.slots, self.page, self.keep, self.scale = slots, page, keep, 1.0 / math.sqrt(head_dim)
        self.caches = [ops.paged_cache(pages, kv_heads, page, head_dim, device, edges=keep > 0) for _ in range(layers)]
        self.table = torch.full((slots, width), -1, dtype=torch.int32, device=device)
        self.ring = torch.arange(pages, dtype=torch.int32, device=device)
        self.counters = torch.tensor([0, pages, 0], dtype=torch.int32, device=device)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device=device)

    def step(self, after, tokens, most, project):
        """Lengths `after` (int32 [slots], on the device: more than before for new tokens, 0 for a request that has ended), `tokens` new ones
        in all and at most `most` of a request. project(layer, x) gives the layer's q, k, v of the step's rows from the layer before's output
        (None for the first). Returns the last layer's output and the plan. When the pages run out the tokens without one (the plan's
        third counter) are not in the cache: their rows are answered from what is, and a server stores them again in a later step."""
        before = self.lengths
        plan = ops.paged_plan(before, after, self.table, self.ring, self.counters, self.page, tokens)
        self.lengths, self.counters = plan["lengths"], plan["counters"]
        where = (self.table, plan["lengths"], plan["starts"])
        x = None
        for layer, cache in enumerate(self.caches):
            q, k, v = project(layer, x)
            ops.paged_store(cache, k, v, plan["work"])
            lists = ops.paged_select(cache, q, *where, self.keep, before=before, most=most) if self.keep and most == 1 else None
            x = ops.paged_attend(cache, q, *where, self.scale, before=before, lists=lists, most=most)
        return x, plan


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=500, help="the longest prompt")
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--pages", type=int, default=2000)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--keep", type=int, default=0, help="pages a decoding query attends to; 0: all")
    args = ap.parse_args()
    heads, kv_heads, head_dim, page = 32, 8, 128, 64
    prompts = [max(1, args.prompt * (r + 1) // args.requests) for r in range(args.requests)]
    width = -(-(max(prompts) + args.steps) // page)
    server = PagedServer(args.requests, args.pages, width, args.layers, heads, kv_heads, head_dim, page, args.keep)
    torch.manual_seed(0)

    warm = PagedServer(2, 4, 2, 1, heads, kv_heads, head_dim, page, args.keep)  # (a kernel's first launch loads it)
    for tokens in (80, 2):
        values = [torch.zeros(tokens, h, head_dim, dtype=torch.bfloat16, device="cuda") for h in (heads, kv_heads, kv_heads)]
        warm.step(warm.lengths + tokens // 2, tokens, tokens // 2, lambda layer, x: values)

    def project(tokens):
        values = [[torch.randn(tokens, h, head_dim, dtype=torch.bfloat16, device="cuda") for h in (heads, kv_heads, kv_heads)] for _ in range(args.layers)]
        return lambda layer, x: values[layer]

    def timed(name, steps, tokens, most, grown):
        project_of = project(tokens)
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(steps):
            x, plan = server.step(server.lengths + grown, tokens, most, project_of)
        torch.cuda.synchronize()
        spent = (time.perf_counter() - start) / steps
        assert bool(torch.isfinite(x.float()).all())
        without = int(plan["counters"][2])
        print(f"{name}: {steps} steps of {tokens} tokens, {spent * 1e6:.0f} us a step, {tokens / spent:.0f} tokens/s, {without} tokens without a page")

    timed("prompts", 1, sum(prompts), max(prompts), torch.tensor(prompts, dtype=torch.int32, device="cuda"))
    timed("decode", args.steps, args.requests, 1, torch.ones(args.requests, dtype=torch.int32, device="cuda"))
    # Half of the requests end: their pages are free for those that come.
    after = server.lengths.clone()
    after[::2] = 0
    _, plan = server.step(after, 1, 1, project(1))
    print(f"{args.requests - args.requests // 2} requests ended: {int(plan['counters'][1])} of {args.pages} pages are free")


if __name__ == "__main__":
    main()
