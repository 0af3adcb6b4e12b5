"""Requests that come and go over one paged 8-bit key / value cache.

    python examples/serve_paged.py [--requests 8] [--steps 16] [--activation softmax]

Every request begins with a history of its own length (many queries at once, causal), then takes one token a step; whoever is long
enough leaves, gives back its blocks and a new request takes its place.  All of it is three calls a step (block tables, append,
attention) that never wait for the GPU.  At the end the last step's output is compared with a dense evaluation in fp64 over the tokens as they
were given, before the cache's 8 bits.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ads_model_kernel_library_b200.gdpa import PagedKVCache, kernel_status  # noqa: E402


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    args.add_argument("--requests", type=int, default=8)
    args.add_argument("--steps", type=int, default=16)
    args.add_argument("--heads", type=int, default=8)
    args.add_argument("--kv-heads", type=int, default=2)
    args.add_argument("--head-dim", type=int, default=128, choices=(64, 128))
    args.add_argument("--block", type=int, default=64, choices=(16, 32, 64, 128))
    args.add_argument("--most-tokens", type=int, default=1000)
    args.add_argument("--activation", default="softmax", choices=("softmax", "silu"))
    a = args.parse_args()
    gen = torch.Generator().manual_seed(0)
    scale = 1 / math.sqrt(a.head_dim) if a.activation == "softmax" else 1 / a.most_tokens
    blocks = a.requests * -(-a.most_tokens // a.block) + 1
    cache = PagedKVCache(blocks, a.block, a.kv_heads, a.head_dim, a.requests, a.most_tokens)

    def tokens(n, heads):
        return torch.randn(n, heads, a.head_dim, generator=gen).bfloat16()

    given = [([], []) for _ in range(a.requests)]  # keys and values of each request, to compare with
    lens = [0] * a.requests
    for step in range(a.steps):
        gone = [b for b in range(a.requests) if lens[b] > a.most_tokens * 0.9]
        if gone:
            cache.release(gone)
            for b in gone:
                given[b], lens[b] = ([], []), 0
        # a request that has nothing yet brings its history, the others one token
        new = [int(torch.randint(1, a.most_tokens - a.steps, (1,), generator=gen)) if n == 0 else 1 for n in lens]
        q, k, v = tokens(sum(new), a.heads), tokens(sum(new), a.kv_heads), tokens(sum(new), a.kv_heads)
        out = cache.step(q.cuda(), k.cuda(), v.cuda(), torch.tensor(new, dtype=torch.int32).cuda(), max(new), qk_scale=scale, activation=a.activation)
        for b, (keys, values) in enumerate(zip(k.split(new), v.split(new))):
            given[b][0].append(keys)
            given[b][1].append(values)
            lens[b] += new[b]

    out, at, worst = out.cpu().double(), 0, 0.0
    for b, n in enumerate(new):
        group = a.heads // a.kv_heads
        keys, values = (torch.cat(x).double().repeat_interleave(group, 1) for x in given[b])
        x = torch.einsum("qhd,khd->hqk", q[at:at + n].double(), keys)
        behind = torch.arange(lens[b]) > torch.arange(lens[b] - n, lens[b])[:, None]
        if a.activation == "softmax":
            p = torch.softmax((x * scale).masked_fill(behind, -math.inf), -1)
        else:
            p = (torch.nn.functional.silu(x) * scale).masked_fill(behind, 0)
        want = torch.einsum("hqk,khd->qhd", p, values)
        worst = max(worst, float((out[at:at + n] - want).norm() / want.norm()))
        at += n
    print(f"{a.steps} steps, {a.requests} requests, {sum(lens)} tokens held, {int(cache.num_free)} of {blocks} blocks free")
    print(f"kernel status {kernel_status()}, largest relative error of a request's output {worst:.4f} (the cache has four significant bits)")
    if kernel_status() != 0 or not worst < 0.1:
        sys.exit(1)


if __name__ == "__main__":
    main()
