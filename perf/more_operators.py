"""The operators on either side of the attention, as cases that can be timed and whose outputs can be compared.

Between the projections and the attention, queries and keys are normalised head by head and rotated by their positions ("rotate", with
its gradient "rotate_grad"); when a model is served, the rotated keys and the values go into the paged 8-bit cache in the same pass
("rotate_append").  What the cache holds is read back as packed tensors ("read").  After the attention and the rest of the model, drafted
tokens are verified against the target's probabilities ("verify"), and the refused ones leave the cache ("drop").

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU from a seed (the lengths of a case are fixed by its
``len_seed``; the seed deals them out to the requests and draws the values), ``run`` is one call, ``exact`` is the same in 64 bits.
Where ``own`` is false, ``run`` computes the operators in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

# ------------------------------------------------------------------------------------------------------ the cases

# Field values a case starts from.
_BASE = {
    "op": "rotate", "batch": 1, "heads": 8, "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "weight": "fp32", "len_seed": 0,
    "new_lo": 1, "new_hi": 1,   # new tokens of a request ("read": tokens that are read, the last of its history; "drop": tokens that leave)
    "kv_lo": 0, "kv_hi": 0,     # tokens of a request before them
    "rotary": 128, "axes": 1, "interleaved": False, "base": 10000.0,
    "block": 64, "vocab": 0, "agree": 0.7, "lookup": False,
}


def _case(**fields):
    c = dict(_BASE)
    c.update(fields)
    if "kv_heads" not in fields:
        c["kv_heads"] = c["heads"]
    if "rotary" not in fields:
        c["rotary"] = c["head_dim"]
    return c


def listed():
    return [
        # A token for each of 64 requests, far into their histories, as the slices of a packed projection.  Latency is all of it.
        _case(name="rotate_one_token", batch=64, heads=32, kv_heads=4, kv_lo=1, kv_hi=262144, base=500000.0),
        # Prompts of 16 to 2048 tokens, four query heads to a key's, half of each head rotated.
        _case(name="rotate_prompts", batch=64, heads=16, kv_heads=4, new_lo=16, new_hi=2048, rotary=64, weight="bf16"),
        # A training step on sequences of 512 to 4096 tokens, eight heads: forward and backward.
        _case(name="train_sequences", op="rotate_grad", batch=128, heads=8, new_lo=512, new_hi=4096),
        # Images and video in fp32: three axes (time, height, width), neighbouring pairs, three heads of 64.
        _case(name="train_three_axes", op="rotate_grad", batch=24, heads=3, head_dim=64, dtype="fp32", new_lo=16, new_hi=1000, axes=3,
              interleaved=True, base=100.0),
        # A step of generation for 256 requests: rotated, quantised and stored.
        _case(name="append_one_token", op="rotate_append", batch=256, heads=32, kv_heads=4, kv_lo=1, kv_hi=2048),
        # New requests' prompts of 512 to 4096 tokens into an empty cache.
        _case(name="append_prompts", op="rotate_append", batch=48, heads=16, kv_heads=4, new_lo=512, new_hi=4096, base=500000.0),
        # One request's last 1500 tokens of 1600, two heads, small blocks: read for an operator that wants packed tensors.
        _case(name="read_one_request", op="read", heads=2, block=16, kv_lo=100, kv_hi=100, new_lo=1500, new_hi=1500),
        # Whole histories of 512 to 4096 tokens, eight heads.
        _case(name="read_histories", op="read", batch=128, heads=8, new_lo=512, new_hi=4096),
        # One request with four drafted tokens.
        _case(name="verify_one_request", op="verify", new_lo=4, new_hi=4, vocab=32000),
        # A batch of 256 with one to eight drafted tokens each; an odd vocabulary, so rows begin anywhere.
        _case(name="verify_batch", op="verify", batch=256, new_lo=1, new_hi=8, vocab=131071),
        # The refused ones of up to eight drafted tokens leave the cache, 256 requests.
        _case(name="drop_refused", op="drop", batch=256, block=16, kv_lo=1, kv_hi=4096, new_lo=0, new_hi=8),
        # Thousands of requests end or are cut back.
        _case(name="drop_histories", op="drop", batch=4096, block=32, kv_lo=0, kv_hi=2048, new_lo=0, new_hi=4096),
    ]


_MOST_VALUES = 3.0e8   # of queries and keys ("rotate" and its gradient, "rotate_append") or keys ("read"); the largest listed case has 6.0e8
_MOST_ROWS = 2.6e8     # batch * most drafts * vocab of "verify"; the largest listed case has 2.7e8
_MOST_DROPPED = 4.0e6  # tokens of a "drop" case; the largest listed case has 8.4e6


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above: a family at random, sizes spread over its range."""
    op = rng.choice(["rotate", "rotate_grad", "rotate_append", "rotate_append", "read", "verify", "verify", "drop"])
    block = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128])
    if op in ("rotate", "rotate_grad", "rotate_append"):
        one = rng.random() < 0.3
        hi = 1 if one else _log_int(rng, 2, 4096)
        c = _case(op=op, batch=_log_int(rng, 1, 300), kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 2, 4, 8]), head_dim=dim,
                  dtype=rng.choice(["bf16", "bf16", "fp32"]), weight=rng.choice(["fp32", "bf16"]), new_lo=1 if one else rng.randint(1, hi), new_hi=hi,
                  kv_lo=0, kv_hi=_log_int(rng, 1, 2048 if op == "rotate_append" else 262144), rotary=rng.choice([dim, dim, dim // 2, 16, 48]),
                  axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.4, base=rng.choice([100.0, 10000.0, 500000.0]), block=block)
    elif op == "read":
        hi = _log_int(rng, 1, 4096)
        c = _case(op=op, batch=_log_int(rng, 1, 300), heads=kv_heads, head_dim=dim, dtype=rng.choice(["bf16", "bf16", "fp32"]), block=block,
                  new_lo=0, new_hi=hi, kv_lo=0, kv_hi=_log_int(rng, 1, 1024))
    elif op == "verify":
        c = _case(op=op, batch=_log_int(rng, 1, 512), new_lo=rng.randint(0, 2), new_hi=rng.randint(2, 12), vocab=_log_int(rng, 100, 152000),
                  dtype=rng.choice(["fp32", "fp32", "bf16"]), agree=rng.choice([0.3, 0.7, 0.9]), lookup=rng.random() < 0.25)
    else:
        c = _case(op=op, batch=_log_int(rng, 1, 8192), block=block, kv_lo=0, kv_hi=_log_int(rng, 1, 4096), new_lo=0,
                  new_hi=_log_int(rng, 1, 4096))
    c["len_seed"] = rng.randrange(1 << 20)
    while c["batch"] > 1 and _too_much(c):
        c["batch"] = c["batch"] * 2 // 3
    return c


def _too_much(c):
    before, new = _lengths(c)
    if c["op"] == "verify":
        return c["batch"] * c["new_hi"] * c["vocab"] > _MOST_ROWS
    if c["op"] == "drop":
        return int((before + new).sum()) > _MOST_DROPPED
    heads = c["kv_heads"] if c["op"] == "read" else c["heads"] + c["kv_heads"]
    tokens = int(new.sum()) + (int(before.sum()) if c["op"] in ("read", "rotate_append") else 0)
    return tokens * heads * c["head_dim"] > _MOST_VALUES


def _lengths(case):
    """(tokens before, new tokens) of the requests."""
    rng = np.random.default_rng(case["len_seed"])
    before = rng.integers(case["kv_lo"], case["kv_hi"] + 1, case["batch"])
    return before, rng.integers(case["new_lo"], case["new_hi"] + 1, case["batch"])


# ----------------------------------------------------------------------------------------------- inputs and a pass


def _up(x, m):
    return (x + m - 1) // m


def _device(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dtype)


def _int32(x):
    return _device(x, torch.int32)


def _type(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _sections(pairs, axes):
    """How many of a head's pairs turn with each axis: of three, height and width have three eighths each."""
    return (pairs,) if axes == 1 else (pairs - 2 * (pairs * 3 // 8), pairs * 3 // 8, pairs * 3 // 8)


def _positions(case, before, new, deal):
    """Positions [axes, tokens]: tokens of a request follow one another; with three axes they are frames of rows of a request's own size."""
    owner = np.repeat(np.arange(len(new)), new)
    i = np.arange(len(owner)) - (np.cumsum(new) - new)[owner]
    if case["axes"] == 1:
        return (before[owner] + i)[None]
    wide, high = deal.integers(1, 33, len(new))[owner], deal.integers(1, 25, len(new))[owner]
    return np.stack([before[owner] + i // (wide * high), i // wide % high, i % wide])


def _power_of_two(amax):
    """The smallest power of two with amax / scale <= 448, at least 2^-100 (fp32, exact)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = torch.where(amax > 0, exponent - 9 + (mantissa > 0.875).int(), -100).clamp_min(-100)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _cache(case, blocks, gen):
    """A filled cache [blocks, block, heads, head_dim] of e4m3 values and its scales [blocks, heads]."""
    x = torch.randn((blocks, case["block"], case["kv_heads"], case["head_dim"]), generator=gen, device="cuda")
    x *= torch.exp(0.3 * torch.randn((blocks, 1, case["kv_heads"], 1), generator=gen, device="cuda"))  # blocks differ in size
    s = _power_of_two(x.abs().amax((1, 3)))
    return (x / s[:, None, :, None]).to(torch.float8_e4m3fn), s


def _prepare_rotary(case, s, before, new, gen, deal):
    H, Hk, D, dtype = case["heads"], case["kv_heads"], case["head_dim"], _type(case)
    pairs, tokens = case["rotary"] // 2, int(new.sum())
    positions = _device(_positions(case, before, new, deal), torch.int64)
    weight = torch.float32 if case["weight"] == "fp32" else torch.bfloat16
    s.update(inv_freq=case["base"] ** -(torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs), eps=1e-6, interleaved=case["interleaved"],
             sections=_sections(pairs, case["axes"]) if case["axes"] > 1 else None, positions=positions if case["axes"] > 1 else positions[0],
             query_weight=(1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(weight),
             key_weight=(1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(weight))
    if case["op"] == "rotate_grad":
        for name, heads in (("query", H), ("key", Hk)):
            s[name] = torch.randn((tokens, heads, D), generator=gen, device="cuda").to(dtype).requires_grad_()
            s[name + "_grad"] = torch.randn((tokens, heads, D), generator=gen, device="cuda").to(dtype)
            s[name + "_weight"].requires_grad_()
        return
    packed = torch.randn((tokens, H + 2 * Hk, D), generator=gen, device="cuda").to(dtype)  # as one projection leaves them
    s["query"], s["key"], s["value"] = packed.split([H, Hk, Hk], 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    deal = np.random.default_rng(seed)
    before, new = _lengths(case)
    order = deal.permutation(len(before))  # which request has which lengths
    before, new = before[order], new[order]
    s = {"op": case["op"]}
    if case["op"] == "verify":
        _prepare_verify(case, s, new, gen)
        return s
    if case["op"] in ("rotate", "rotate_grad"):
        _prepare_rotary(case, s, before, new, gen, deal)
        return s
    S, after = case["block"], before + new
    held = _up(after, S)
    width, blocks = max(1, int(held.max())), int(held.sum()) + 8
    pool = deal.permutation(blocks)  # blocks come in any order
    table = np.full((len(after), width), -1, dtype=np.int64)
    table[np.arange(width) < held[:, None]] = pool[:int(held.sum())]
    s.update(block=S, block_tables=_int32(table), seq_lens=_int32(after))
    if case["op"] == "drop":
        s.update(dropped=_int32(new), free_blocks=_int32(np.concatenate([pool[int(held.sum()):], np.full(int(held.sum()), -1)])), num_free=_int32(np.array([8])))
        return s
    offsets = np.concatenate([[0], np.cumsum(new)])
    s["offsets"] = _int32(offsets)
    s["k_cache"], s["k_scales"] = _cache(case, blocks, gen)
    s["v_cache"], s["v_scales"] = _cache(case, blocks, gen)
    if case["op"] == "read":
        s.update(first=_int32(before), total=int(new.sum()), dtype=_type(case))
        return s
    _prepare_rotary(case, s, before, new, gen, deal)
    if case["axes"] == 1:
        s["positions"] = None  # they follow from the lengths
    owner = np.repeat(np.arange(len(new)), new)
    p = before[owner] + np.arange(len(owner)) - offsets[owner]
    s["slots"] = _device(table[owner, p // S] * S + p % S, torch.int64)
    s["most_runs"] = int((_up(after, S) - before // S).sum())  # blocks that the new tokens touch
    return s


def _prepare_verify(case, s, drafts, gen):
    """Drafts come from the target's distribution mixed with another, so that about ``agree`` of them are accepted; or, as looked up in the text, from no
    distribution (one token that the target finds likely or not)."""
    V, dtype = case["vocab"], _type(case)
    n_drafts, rows = int(drafts.sum()), int(drafts.sum()) + len(drafts)
    first = np.cumsum(drafts) - drafts

    def distribution(n):
        return torch.softmax(2.5 * torch.randn((n, V), generator=gen, device="cuda"), 1)

    target = distribution(rows)
    own_row = _device(np.concatenate([np.arange(n) + f + b for b, (n, f) in enumerate(zip(drafts, first))]), torch.int64)  # the target's row for each draft
    draft = case["agree"] * target[own_row] + (1 - case["agree"]) * distribution(n_drafts)
    tokens = torch.multinomial(draft, 1, generator=gen)[:, 0] if n_drafts else torch.zeros(0, dtype=torch.int64, device="cuda")
    s.update(target=target.to(dtype), draft=None if case["lookup"] else draft.to(dtype), tokens=tokens, most=int(drafts.max()),
             offsets=_int32(np.concatenate([[0], np.cumsum(drafts + 1)])), draft_offsets=_int32(np.concatenate([[0], np.cumsum(drafts)])),
             accept=torch.rand(n_drafts, generator=gen, device="cuda"), sample=torch.rand(len(drafts), generator=gen, device="cuda"))


def run(state):
    if not own:
        with torch.no_grad():
            return {"rotate": _rotate_plain, "rotate_grad": _rotate_grad_plain, "rotate_append": _rotate_append_plain, "read": _read_plain,
                    "verify": _verify_plain, "drop": _drop_plain}[state["op"]](state)
    import ads_model_kernel_library_b200.gdpa as gdpa

    s = state
    if s["op"] in ("rotate", "rotate_grad"):
        q, k = gdpa.qk_norm_rotary(s["query"], s["key"], s["inv_freq"], s["positions"], query_weight=s["query_weight"], key_weight=s["key_weight"],
                                   eps=s["eps"], interleaved=s["interleaved"], sections=s["sections"])
        if s["op"] == "rotate":
            return {"query": q, "key": k}
        grads = torch.autograd.grad((q, k), (s["query"], s["key"], s["query_weight"], s["key_weight"]), (s["query_grad"], s["key_grad"]))
        return {"query": q.detach(), "key": k.detach(), **dict(zip(("d_query", "d_key", "d_query_weight", "d_key_weight"), grads))}
    if s["op"] == "rotate_append":
        q = gdpa.append_rotated_kv_cache_fp8(
            s["query"], s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["slots"], s["offsets"], s["seq_lens"], s["inv_freq"],
            positions=s["positions"], query_weight=s["query_weight"], key_weight=s["key_weight"], eps=s["eps"], interleaved=s["interleaved"],
            sections=s["sections"])
        return {"query": q, **{n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}}
    if s["op"] == "read":
        k, v = gdpa.read_kv_cache_fp8(s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["block_tables"], s["offsets"], s["total"],
                                      first_tokens=s["first"], dtype=s["dtype"])
        return {"key": k, "value": v}
    if s["op"] == "verify":
        tokens, accepted, refused = gdpa.verify_draft_tokens(s["target"], s["draft"], s["tokens"], s["offsets"], s["draft_offsets"], s["accept"], s["sample"],
                                                             s["most"])
        return {"tokens": tokens, "accepted": accepted, "refused": refused}
    lens, num_free = gdpa.drop_cached_tokens(s["block_tables"], s["seq_lens"], s["dropped"], s["free_blocks"], s["num_free"], s["block"])
    return {"seq_lens": lens, "num_free": num_free, "free_blocks": s["free_blocks"]}


def _angles(s, positions):
    """Cosine and sine of every token's angles, fp32 [tokens, 1, pairs]; the angles of far positions need 64 bits."""
    if s["sections"] is None:
        p = positions.reshape(1, -1).expand(s["inv_freq"].numel(), -1)
    else:
        axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=positions.device), torch.tensor(s["sections"], device=positions.device),
                                       output_size=s["inv_freq"].numel())
        p = positions[axis]
    angle = (p.double() * s["inv_freq"].double()[:, None]).t()[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _turn(x, cos, sin, interleaved):
    """The first 2 * pairs values of every head, turned."""
    pairs = cos.shape[-1]
    head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :pairs], head[..., pairs:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _normed(x, eps):
    """Unit rows of `x` in fp32, and the factors that made them so."""
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _rotate_plain(s):
    cos, sin = _angles(s, s["positions"])
    out = {}
    for name in ("query", "key"):
        unit, _ = _normed(s[name], s["eps"])
        out[name] = _turn(unit * s[name + "_weight"].float(), cos, sin, s["interleaved"]).to(s[name].dtype)
    return out


def _rotate_grad_plain(s):
    cos, sin = _angles(s, s["positions"])
    out = {}
    for name in ("query", "key"):
        w = s[name + "_weight"].float()
        unit, r = _normed(s[name], s["eps"])
        out[name] = _turn(unit * w, cos, sin, s["interleaved"]).to(s[name].dtype)
        back = _turn(s[name + "_grad"].float(), cos, -sin, s["interleaved"])
        out["d_" + name + "_weight"] = (back * unit).sum((0, 1)).to(s[name + "_weight"].dtype)
        back = back * w
        out["d_" + name] = (r * (back - unit * (back * unit).mean(-1, keepdim=True))).to(s[name].dtype)
    return out


def _append_one(x, cache, scales, slots, most_runs):
    """New rows `x` [tokens, heads, dim] into their slots of one cache (every run of slots lies in one block)."""
    blocks, S, H, D = cache.shape
    raw = cache.view(torch.uint8)
    block, row = slots // S, slots % S
    begins = torch.cat([torch.ones_like(slots[:1], dtype=torch.bool), (block[1:] != block[:-1]) | (slots[1:] != slots[:-1] + 1)])
    run = torch.cumsum(begins, 0) - 1
    # block and first row of each run; rows past the last run repeat the first run's
    run_block = block[:1].repeat(most_runs).scatter_(0, run, block)
    run_row = row[:1].repeat(most_runs).scatter_reduce_(0, run, row, "amin", include_self=False)
    amax = torch.zeros(most_runs, H, device=x.device).scatter_reduce_(0, run[:, None].expand(-1, H), x.float().abs().amax(2), "amax")
    amax = torch.where((torch.arange(most_runs, device=x.device) <= run[-1])[:, None], amax, amax[:1])
    fresh, before = _power_of_two(amax), scales[run_block]
    after = torch.where((run_row > 0)[:, None], torch.maximum(before, fresh), fresh)
    held = raw[run_block].view(torch.float8_e4m3fn).float()
    scaled = (held * (before / after)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = torch.arange(S, device=x.device)[None, :] < run_row[:, None]
    raw[run_block] = torch.where(keep[:, :, None, None], scaled, raw[run_block])
    scales[run_block] = after
    raw.view(blocks * S, H, D)[slots] = (x.float() / after[run][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _rotate_append_plain(s):
    positions = s["positions"]
    if positions is None:
        t = torch.arange(s["query"].shape[0], device=s["query"].device)
        b = torch.searchsorted(s["offsets"][1:].long(), t, right=True)
        positions = s["seq_lens"].long()[b] - s["offsets"].long()[b + 1] + t
    cos, sin = _angles(s, positions)
    q, k = (_turn(_normed(s[n], s["eps"])[0] * s[n + "_weight"].float(), cos, sin, s["interleaved"]) for n in ("query", "key"))
    _append_one(k, s["k_cache"], s["k_scales"], s["slots"], s["most_runs"])
    _append_one(s["value"], s["v_cache"], s["v_scales"], s["slots"], s["most_runs"])
    return {"query": q.to(s["query"].dtype), **{n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}}


def _read_plain(s):
    S, offsets = s["block"], s["offsets"].long()
    t = torch.arange(s["total"], device=offsets.device)
    b = torch.searchsorted(offsets[1:], t, right=True)
    p = s["first"].long()[b] + t - offsets[b]
    block = s["block_tables"].long()[b, p // S]
    return {name: (s[c + "_cache"].view(torch.uint8)[block, p % S].view(torch.float8_e4m3fn).float() * s[c + "_scales"][block][:, :, None]).to(s["dtype"])
            for name, c in (("key", "k"), ("value", "v"))}


def _verify_plain(s):
    V = s["target"].shape[1]
    rows, first = s["offsets"].long()[:-1], s["draft_offsets"].long()
    n = first[1:] - first[:-1]
    batch, n_drafts, device = len(n), s["tokens"].numel(), rows.device
    d = torch.arange(n_drafts, device=device)
    b = torch.searchsorted(first[1:], d, right=True)
    j = d - first[b]
    # accepted: the drafts before the first that is refused
    p = s["target"][rows[b] + j, s["tokens"]].double()
    q = torch.ones_like(p) if s["draft"] is None else s["draft"][d, s["tokens"]].double()
    accepted = n.scatter_reduce(0, b, torch.where(s["accept"].double() * q < p, n[b], j), "amin")
    refused = n - accepted
    # the next token: from max(p - q, 0) where a draft was refused, from p where none was
    p = s["target"][rows + accepted].double()
    at = (first[:-1] + accepted).clamp_max(max(n_drafts - 1, 0))
    if n_drafts == 0:
        left = p
    else:
        if s["draft"] is None:
            q = torch.where(torch.arange(V, device=device) == s["tokens"][at][:, None], math.inf, 0.0).double()
        else:
            q = s["draft"][at].double()
        left = torch.where((refused > 0)[:, None], (p - q).clamp_min(0), p)
        left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
    below = torch.cumsum(left, 1)
    found = (below > s["sample"].double()[:, None] * below[:, -1:]) & (left > 0)
    token = torch.where(found.any(1), found.to(torch.int8).argmax(1), -1)
    out = torch.full((batch, s["most"] + 1), -1, dtype=torch.int64, device=device)
    keep = j < accepted[b]
    place = torch.where(keep, b * (s["most"] + 1) + j, out.numel())
    out = torch.cat([out.flatten(), out.new_zeros(1)]).scatter_(0, place, s["tokens"])[:-1].view(batch, -1)
    out.scatter_(1, accepted[:, None], token[:, None])
    return {"tokens": out, "accepted": accepted.int(), "refused": refused.int()}


def _drop_plain(s):
    S, width = s["block"], s["block_tables"].shape[1]
    lens = s["seq_lens"].long()
    after = lens - torch.minimum(s["dropped"].long().clamp_min(0), lens)
    j = torch.arange(width, device=lens.device)
    free = (j >= _up(after, S)[:, None]) & (j < _up(lens, S)[:, None]) & (s["block_tables"] >= 0)
    have = s["num_free"].long().clamp_min(0)
    place = have + torch.cumsum(free.flatten(), 0) - 1
    # entries that stay go to a place behind the stack
    stack = torch.cat([s["free_blocks"], s["free_blocks"].new_zeros(1)])
    stack.scatter_(0, torch.where(free.flatten(), place, s["free_blocks"].numel()), s["block_tables"].flatten())
    s["free_blocks"].copy_(stack[:-1])
    return {"seq_lens": after.int(), "num_free": (have + free.sum()).int(), "free_blocks": s["free_blocks"]}


# ---------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    before, new = _lengths(case)
    H, Hk, D, S, n = case["heads"], case["kv_heads"], case["head_dim"], case["block"], int(new.sum())
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotate":
        return {"bytes": 2 * n * (H + Hk) * D * size + 8 * n * case["axes"], "flops": 10 * n * (H + Hk) * D}
    if case["op"] == "rotate_grad":  # forward, and the gradient from the inputs and the outputs' gradient
        return {"bytes": 5 * n * (H + Hk) * D * size + 8 * n * case["axes"], "flops": 30 * n * (H + Hk) * D}
    if case["op"] == "rotate_append":
        runs = int((_up(before + new, S) - before // S).sum())
        return {"bytes": n * D * (2 * H * size + 2 * Hk * (size + 1)) + 8 * n + 16 * runs * Hk, "flops": n * (10 * (H + Hk) + 4 * Hk) * D}
    if case["op"] == "read":
        runs = int(np.where(new > 0, _up(before + new, S) - before // S, 0).sum())
        return {"bytes": 2 * n * Hk * D * (1 + size) + runs * (8 * Hk + 4), "flops": 2 * n * Hk * D}
    if case["op"] == "verify":  # one row of the target for each request, and one of the draft's where a token was refused
        refused = 0 if case["lookup"] else float((1 - case["agree"] ** new).sum())
        return {"bytes": size * case["vocab"] * (case["batch"] + refused) + 20 * n, "flops": 3 * case["vocab"] * case["batch"]}
    after = np.maximum(before + new - new, 0)
    freed = int((_up(before + new, S) - _up(after, S)).sum())
    return {"bytes": 12 * case["batch"] + 8 * freed + 8, "flops": 0}


# ------------------------------------------------------------------------------------- the same pass in 64 bits


def _e4m3(x):
    """`x` (fp64) rounded to the nearest e4m3 value, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_rotated(s, x, weight, positions):
    """RMS norm and rotation as complex products, in fp64."""
    pairs, x = s["inv_freq"].numel(), x.double()
    n = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + s["eps"]) * weight.double()
    sections = s["sections"] or (pairs,)
    turns, i = [], 0
    for a, m in enumerate(sections):
        p = (positions if s["sections"] else positions.reshape(1, -1))[a].double()
        turns.append(p[:, None] * s["inv_freq"][i:i + m].double())
        i += m
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.cat(turns, 1))[:, None]
    head = n[..., :2 * pairs].unflatten(-1, (pairs, 2) if s["interleaved"] else (2, pairs))
    if not s["interleaved"]:
        head = head.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * unit)
    if not s["interleaved"]:
        z = z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), n[..., 2 * pairs:]], -1)


def exact(case, seed):
    if case["op"] in ("verify", "drop"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return {n: _exact_rotated(s, s[n], s[n + "_weight"], s["positions"]) for n in ("query", "key")}
    if case["op"] == "rotate_grad":
        out = {}
        for name in ("query", "key"):
            x, w = (s[n].detach().double().requires_grad_() for n in (name, name + "_weight"))
            dw = torch.zeros_like(w)
            y, dx = torch.empty_like(x), torch.empty_like(x)
            step = 1 << 15  # tokens at a time
            for i in range(0, x.shape[0], step):
                part = x.detach()[i:i + step].requires_grad_()
                o = _exact_rotated(s, part, w, s["positions"][..., i:i + step])
                g, gw = torch.autograd.grad(o, (part, w), s[name + "_grad"][i:i + step].double())
                y.data[i:i + step], dx.data[i:i + step] = o.detach(), g
                dw = dw + gw
            out[name], out["d_" + name], out["d_" + name + "_weight"] = y.detach(), dx.detach(), dw.detach()
        return out
    S = case["block"]
    before, new = ((s["seq_lens"].long() - torch.diff(s["offsets"].long())).tolist(), torch.diff(s["offsets"].long()).tolist())
    if case["op"] == "read":
        out = {}
        for name, c in (("key", "k"), ("value", "v")):
            rows = []
            for b, (f, n) in enumerate(zip(before, new)):
                blocks = s["block_tables"][b, f // S:_up(f + n, S)].long()
                x = s[c + "_cache"].view(torch.uint8)[blocks].view(torch.float8_e4m3fn).double() * s[c + "_scales"][blocks].double()[:, None, :, None]
                rows.append(x.flatten(0, 1)[f % S:f % S + n])
            out[name] = torch.cat(rows)
        return out
    positions = s["positions"]
    if positions is None:
        positions = torch.cat([torch.arange(f, f + n, device="cuda") for f, n in zip(before, new)])
    if s["most_runs"] > 12000:
        return None
    q, k = (_exact_rotated(s, s[n], s[n + "_weight"], positions) for n in ("query", "key"))
    out = {"query": q}
    for name, x in (("k", k), ("v", s["value"].double())):
        cache, scales, i = s[name + "_cache"].double(), s[name + "_scales"].double(), 0
        for b, (f, n) in enumerate(zip(before, new)):
            p = f
            while p < f + n:  # a run: the tokens of one block
                row, m = p % S, min(S - p % S, f + n - p)
                block = s["block_tables"][b, p // S].long()
                part = x[i:i + m]
                least = torch.exp2(torch.ceil(torch.log2(part.abs().amax((0, 2)).clamp_min(1e-45) / 448)).clamp_min(-100))
                scale = torch.maximum(scales[block], least) if row else least
                if row:
                    cache[block, :row] = _e4m3(cache[block, :row] * (scales[block] / scale)[:, None])
                cache[block, row:row + m] = _e4m3(part / scale[:, None])
                scales[block] = scale
                i, p = i + m, p + m
        out[name + "_cache"], out[name + "_scales"] = cache, scales
    return out
