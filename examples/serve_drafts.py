"""A step of generation with drafted tokens: several tokens a request and step, distributed as if they had come one by one.

    python examples/serve_drafts.py [--requests 8] [--steps 24] [--drafts 4]

The model is a toy with random weights (an embedding, one layer of attention, the embedding again); what is around the attention is the real thing.
Queries and keys of a step are normed, rotated and appended to the paged 8-bit cache in one go, the new tokens attend to all of it, and the
target's probabilities decide about the drafts, which are looked up in the request's own text: what followed the last token when
it stood there before.  Refused drafts leave the cache again.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ads_model_kernel_library_b200.gdpa import PagedKVCache, kernel_status, verify_draft_tokens  # noqa: E402


class Model:
    """Tokens to probabilities of the next one."""

    def __init__(self, vocabulary, heads, kv_heads, dim, temperature, gen):
        self.shape, self.temperature = (heads, kv_heads, dim), temperature
        width = heads * dim
        self.embedding = (torch.randn(vocabulary, width, generator=gen) / math.sqrt(width)).cuda().bfloat16()
        self.inwards = (torch.randn(width, (heads + 2 * kv_heads) * dim, generator=gen) / math.sqrt(width)).cuda().bfloat16()
        self.outwards = (torch.randn(width, width, generator=gen) / math.sqrt(width)).cuda().bfloat16()
        self.rotary = dict(inv_freq=(10000.0 ** -(torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).cuda(),
                           query_weight=torch.full((dim,), 2.0).cuda(), key_weight=torch.full((dim,), 2.0).cuda())

    def __call__(self, tokens, cache, new_lens, most):
        heads, kv_heads, dim = self.shape
        x = self.embedding[tokens]
        qkv = (x @ self.inwards).view(len(tokens), heads + 2 * kv_heads, dim)
        query, key, value = qkv.split((heads, kv_heads, kv_heads), 1)  # as they lie: nothing is copied
        out = cache.step(query, key, value, new_lens, most, rotary=self.rotary, qk_scale=1 / math.sqrt(dim))
        x = x + out.flatten(1) @ self.outwards
        return torch.softmax((x @ self.embedding.T).float() / self.temperature, -1)


def look_up(text, most):
    """What followed the last token of the text where it stood before, at most `most` tokens."""
    for i in range(len(text) - 2, -1, -1):
        if text[i] == text[-1]:
            return text[i + 1:i + 1 + most]
    return []


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    args.add_argument("--requests", type=int, default=8)
    args.add_argument("--steps", type=int, default=24)
    args.add_argument("--drafts", type=int, default=4)
    args.add_argument("--heads", type=int, default=8)
    args.add_argument("--kv-heads", type=int, default=2)
    args.add_argument("--head-dim", type=int, default=128, choices=(64, 128))
    args.add_argument("--block", type=int, default=16, choices=(16, 32, 64, 128))
    args.add_argument("--vocabulary", type=int, default=512)
    args.add_argument("--temperature", type=float, default=0.02)
    a = args.parse_args()
    gen = torch.Generator().manual_seed(0)
    most_tokens = 64 + (a.steps + 1) * (a.drafts + 1)
    cache = PagedKVCache(a.requests * -(-most_tokens // a.block), a.block, a.kv_heads, a.head_dim, a.requests, most_tokens)
    model = Model(a.vocabulary, a.heads, a.kv_heads, a.head_dim, a.temperature, gen)

    def int32(x):
        return torch.tensor(x, dtype=torch.int32).cuda()

    def offsets(lens):
        return int32([sum(lens[:b]) for b in range(len(lens) + 1)])

    # the prompts: of each, the row of its last token says what comes next
    texts = [torch.randint(0, a.vocabulary, (int(torch.randint(1, 64, (1,), generator=gen)),), generator=gen).tolist() for _ in range(a.requests)]
    lens = [len(t) for t in texts]
    probs = model(torch.tensor(sum(texts, [])).cuda(), cache, int32(lens), max(lens))
    drafts, rows = [[] for _ in texts], offsets([1] * a.requests)
    probs = probs[offsets(lens)[1:].long() - 1]
    drafted = kept = 0
    for step in range(a.steps + 1):
        if step > 0:  # the last known token of each request and the drafts behind it
            drafts = [look_up(t, a.drafts) for t in texts]
            lens = [1 + len(d) for d in drafts]
            rows = offsets(lens)
            probs = model(torch.tensor([x for t, d in zip(texts, drafts) for x in [t[-1], *d]]).cuda(), cache, int32(lens), a.drafts + 1)
        n = sum(len(d) for d in drafts)
        tokens, accepted, refused = verify_draft_tokens(probs, None, torch.tensor(sum(drafts, []), dtype=torch.int64).cuda(), rows,
                                                        offsets([len(d) for d in drafts]), torch.rand(n, generator=gen).cuda(),
                                                        torch.rand(a.requests, generator=gen).cuda(), a.drafts)
        cache.drop(refused)
        for text, new, count in zip(texts, tokens.tolist(), accepted.tolist()):  # the host reads them: it looks up the next drafts
            text += new[:count + 1]
        drafted, kept = drafted + n, kept + int(accepted.sum())
    held = cache.seq_lens.tolist()
    print(f"{a.steps} steps, {a.requests} requests, {sum(map(len, texts))} tokens of text, {kept} of {drafted} drafts accepted")
    print(f"kernel status {kernel_status()}, {sum(held)} tokens held, {int(cache.num_free)} blocks free")
    # the cache holds every token but the last of each text
    if kernel_status() != 0 or held != [len(t) - 1 for t in texts] or int(cache.num_free) != cache.free_blocks.numel() - sum(-(-n // a.block) for n in held):
        sys.exit(1)


if __name__ == "__main__":
    main()
