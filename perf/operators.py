"""The operators of a served model's key / value cache, as cases that can be timed and whose outputs can be compared.

A request's keys and values stay in a paged cache of 8-bit values (e4m3) between calls, with one scale for each block of tokens and
head.  Three operators serve it: the block tables and slot maps of a batch are built from the requests' lengths ("tables"), new keys and
values are quantised into their slots ("append"), and queries attend to what the cache holds ("attend").

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU from a seed (the lengths of a case are fixed by its
``len_seed``; the seed deals them out to the requests and draws the values), ``run`` is one call, ``exact`` is the same in 64 bits.
Where ``own`` is false, ``run`` computes the operators in elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

# ------------------------------------------------------------------------------------------------------ the cases

# Field values a case starts from.  Lengths are uniform in lo .. hi or, "zipf", multiples of 32 up to hi with a heavy tail.
_BASE = {
    "op": "attend", "batch": 1, "heads": 8, "kv_heads": 8, "head_dim": 128, "block": 64, "dtype": "bf16", "activation": "softmax",
    "kv": "uniform", "kv_lo": 1, "kv_hi": 256,  # tokens of a request that are in the cache (for "tables" and "append": before the call)
    "new_lo": 1, "new_hi": 1,  # new tokens ("tables", "append") or queries ("attend") of a request
    "causal": False, "window": -1, "len_seed": 0,
}


def _case(**fields):
    c = dict(_BASE)
    c.update(fields)
    if "kv_heads" not in fields:
        c["kv_heads"] = c["heads"]
    return c


def listed():
    return [
        # One token for each of 64 requests: what precedes every step of generation.  Latency is all of it.
        _case(name="tables_one_token", op="tables", batch=64, kv_lo=1, kv_hi=4096),
        # A batch of new requests of 512 to 4096 tokens, nothing cached yet, small blocks.
        _case(name="tables_new_requests", op="tables", batch=512, block=16, kv_lo=0, kv_hi=0, new_lo=512, new_hi=4096),
        # Thousands of requests with heavily skewed histories, each a few tokens longer than before.
        _case(name="tables_many_requests", op="tables", batch=8192, block=32, kv="zipf", kv_hi=8192, new_lo=1, new_hi=64),
        # One new token for each of 256 requests, most of them into a block that is partly full.
        _case(name="append_one_token", op="append", batch=256, kv_lo=1, kv_hi=2048),
        # The keys and values of whole histories, 512 to 4096 tokens, eight heads.
        _case(name="append_histories", op="append", batch=128, kv_lo=0, kv_hi=0, new_lo=512, new_hi=4096),
        # A few tokens a request that begin and end inside blocks of 16; three heads of 64, fp32 keys and values.
        _case(name="append_ragged", op="append", batch=300, heads=3, head_dim=64, block=16, dtype="fp32", kv_lo=0, kv_hi=100,
              new_lo=1, new_hi=37),
        # One request, one token: the answer is waited for.  Two heads, so the history has to be split.
        _case(name="decode_one_request", batch=1, heads=8, kv_heads=2, block=16, kv_lo=1500, kv_hi=1500),
        # A step of generation for a large batch: histories of 1 to 4096 tokens, eight query heads to a cached one.
        _case(name="decode_ragged", batch=256, heads=32, kv_heads=4, kv_lo=1, kv_hi=4096),
        # A few very long histories.
        _case(name="decode_long", batch=6, heads=16, kv_heads=2, block=128, kv_lo=32768, kv_hi=262144),
        # One to four draft tokens a request, each with its own heads of 64, attention limited to the last 1024 tokens, small blocks.
        _case(name="draft_window", batch=96, heads=8, head_dim=64, block=16, kv_lo=64, kv_hi=2048, new_lo=1, new_hi=4, causal=True,
              window=1024),
        # A ranking model's requests: 64 to 1024 candidates attend, element by element (SiLU), to one cached history.
        _case(name="candidates_silu", batch=64, heads=8, activation="silu", kv_lo=512, kv_hi=4096, new_lo=64, new_hi=1024),
        # A chunk of 256 to 1024 tokens of each prompt attends to what came before and, causally, to itself.
        _case(name="chunk_causal", batch=16, heads=16, kv_heads=4, block=128, kv_lo=1024, kv_hi=4096, new_lo=256, new_hi=1024, causal=True),
    ]


_MOST_TOKENS = 6.0e5   # of a cache, times kv_heads * head_dim / 1024; the largest listed case has 3.0e5, and as many bytes again to read
_MOST_PAIRS = 1.0e9    # (query, key) pairs of the padded rectangle, times heads; the largest listed case has 2.1e9
_MOST_SLOTS = 1.0e6    # new tokens of a "tables" case; the largest listed case has 1.2e6


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above: a family at random, sizes spread over its range."""
    family = rng.choice(["tables", "append", "append_tokens", "decode", "decode", "decode_long", "draft", "candidates", "chunk"])
    block = rng.choice([16, 32, 64, 128])
    if family == "tables":
        c = _case(op="tables", batch=_log_int(rng, 1, 8192), block=block, kv=rng.choice(["uniform", "zipf"]), kv_lo=0,
                  kv_hi=_log_int(rng, 32, 8192), new_lo=0, new_hi=_log_int(rng, 1, 4096))
    elif family in ("append", "append_tokens"):
        hi = _log_int(rng, 2, 4096) if family == "append" else 1
        c = _case(op="append", batch=_log_int(rng, 1, 300), heads=rng.choice([1, 2, 3, 4, 8]), head_dim=rng.choice([64, 128]), block=block,
                  dtype=rng.choice(["bf16", "bf16", "fp32"]), kv_lo=0, kv_hi=_log_int(rng, 1, 2048), new_lo=1, new_hi=hi)
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        common = dict(heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128]), block=block)
        if family == "decode":
            c = _case(batch=_log_int(rng, 1, 256), kv_lo=0, kv_hi=_log_int(rng, 64, 4096), activation=rng.choice(["softmax", "softmax", "silu"]),
                      **common)
        elif family == "decode_long":
            hi = _log_int(rng, 16384, 262144)
            c = _case(batch=_log_int(rng, 1, 8), kv_lo=hi // 8, kv_hi=hi, **common)
        elif family == "draft":
            c = _case(batch=_log_int(rng, 1, 256), kv_lo=16, kv_hi=_log_int(rng, 64, 4096), new_lo=1, new_hi=rng.randint(2, 8), causal=True,
                      window=rng.choice([-1, 128, 300, 1024]), **common)
        else:
            hi = _log_int(rng, 16, 1024)
            c = _case(batch=_log_int(rng, 1, 64), kv_lo=hi, kv_hi=_log_int(rng, 1024, 4096), new_lo=rng.randint(1, hi), new_hi=hi,
                      causal=family == "chunk", activation="softmax" if family == "chunk" else rng.choice(["silu", "gelu_approx", "relu"]),
                      **common)
    c["len_seed"] = rng.randrange(1 << 20)
    while c["batch"] > 1 and (_tokens(c) > _MOST_TOKENS or _rectangle(c) > _MOST_PAIRS or _slots(c) > _MOST_SLOTS):
        c["batch"] = c["batch"] * 2 // 3
    return c


# ------------------------------------------------------------------------------------------------------- lengths


def _lengths(case):
    """(tokens in the cache, new tokens or queries) of the requests; for "attend" the queries are the last of the cached tokens."""
    rng = np.random.default_rng(case["len_seed"])
    n = case["batch"]
    if case["kv"] == "zipf":
        cached = 32 * np.minimum(rng.zipf(1.2, n), max(1, case["kv_hi"] // 32)).astype(np.int64)
    else:
        cached = rng.integers(case["kv_lo"], case["kv_hi"] + 1, n)
    return cached, rng.integers(case["new_lo"], case["new_hi"] + 1, n)


def _tokens(case):
    cached, new = _lengths(case)
    total = int((cached + new).sum()) if case["op"] == "append" else int(cached.sum()) if case["op"] == "attend" else 0
    return total * case["kv_heads"] * case["head_dim"] / 1024


def _rectangle(case):
    return 0 if case["op"] != "attend" else case["batch"] * case["heads"] * case["new_hi"] * int(_lengths(case)[0].max())


def _slots(case):
    return int(_lengths(case)[1].sum()) if case["op"] == "tables" else 0


def _ranges(case):
    """Keys [first, end) that each query of each request takes part with, as flat arrays over the queries, and the union by request."""
    cached, new = _lengths(case)
    first, end, union = [], [], 0
    for n, q in zip(cached.tolist(), new.tolist()):
        p = n - q + np.arange(q)
        lo = np.maximum(p - case["window"], 0) if case["window"] >= 0 else np.zeros(q, dtype=np.int64)
        hi = np.full(q, n)
        if case["causal"]:
            hi = np.minimum(hi, p + 1)
        if case["window"] >= 0:
            hi = np.minimum(hi, p + case["window"] + 1)
        first.append(lo)
        end.append(np.maximum(hi, lo))
        live = hi > lo
        union += int(hi[live].max() - lo[live].min()) if live.any() else 0
    return np.concatenate(first), np.concatenate(end), union


# ----------------------------------------------------------------------------------------------- inputs and a pass


def _up(x, m):
    return (x + m - 1) // m


def _power_of_two(amax):
    """The smallest power of two with amax / scale <= 448, at least 2^-100 (fp32, exact)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = torch.where(amax > 0, exponent - 9 + (mantissa > 0.875).int(), -100).clamp_min(-100)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _int32(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", torch.int32)


def _cache(case, blocks, gen):
    """A filled cache [blocks, block, heads, head_dim] of e4m3 values and its scales [blocks, heads]."""
    shape = (blocks, case["block"], case["kv_heads"], case["head_dim"])
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(shape[0], shape[2], device="cuda")
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        x = torch.randn((n, *shape[1:]), generator=gen, device="cuda")
        x *= torch.exp(0.3 * torch.randn((n, 1, shape[2], 1), generator=gen, device="cuda"))  # blocks differ in size
        s = _power_of_two(x.abs().amax((1, 3)))
        out[i:i + n] = (x / s[:, None, :, None]).to(torch.float8_e4m3fn)
        scales[i:i + n] = s
    return out, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cached, new = _lengths(case)
    deal = np.random.default_rng(seed)
    order = deal.permutation(len(cached))  # which request has which lengths
    cached, new = cached[order], new[order]
    S, H, Hk, D = case["block"], case["heads"], case["kv_heads"], case["head_dim"]
    after = cached + new if case["op"] != "attend" else cached
    held = _up(cached, S) if case["op"] == "tables" else _up(after, S)  # blocks in the table before the call
    width, n_held = max(1, int(_up(after, S).max())), int(held.sum())
    blocks = int(_up(after, S).sum()) + 8
    pool = deal.permutation(blocks)  # blocks come in any order
    table = np.full((len(cached), width), -1, dtype=np.int64)
    table[np.arange(width) < held[:, None]] = pool[:n_held]
    s = {"op": case["op"], "block": S, "width": width, "block_tables": _int32(table), "total_new": int(new.sum())}
    if case["op"] == "tables":
        s.update(cached_lens=_int32(cached), new_lens=_int32(new), free_blocks=_int32(pool[n_held:]), num_free=_int32(np.array([blocks - n_held])))
        return s
    offsets = np.concatenate([[0], np.cumsum(new)])
    s["k_cache"], s["k_scales"] = _cache(case, blocks, gen)
    s["v_cache"], s["v_scales"] = _cache(case, blocks, gen)

    def values(heads, dtype):
        return torch.randn((s["total_new"], heads, D), generator=gen, device="cuda").to(dtype)

    if case["op"] == "append":
        owner = np.repeat(np.arange(len(new)), new)
        p = cached[owner] + np.arange(len(owner)) - offsets[owner]
        s["slots"] = torch.from_numpy(table[owner, p // S] * S + p % S).cuda()
        dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        s["key"], s["value"] = values(Hk, dtype), values(Hk, dtype)
        s["most_runs"] = int((_up(cached + new, S) - cached // S).sum())  # blocks that the new tokens touch
        return s
    s.update(query=values(H, torch.bfloat16), query_offset=_int32(offsets), seq_lens=_int32(cached), max_q=int(new.max()),
             activation=case["activation"], causal=case["causal"], window=case["window"] if case["window"] >= 0 else None,
             scale=1.0 / math.sqrt(D) if case["activation"] == "softmax" else 1.0 / int(cached.max()))
    return s


def run(state):
    if not own:
        return {"tables": _tables_plain, "append": _append_plain, "attend": _attend_plain}[state["op"]](state)
    import ads_model_kernel_library_b200.gdpa as gdpa

    s = state
    if s["op"] == "tables":
        slots, offsets, lens, free = gdpa.build_block_tables(
            s["block_tables"], s["cached_lens"], s["new_lens"], s["free_blocks"], s["num_free"], s["block"], s["total_new"])
        return {"block_tables": s["block_tables"], "slots": slots, "query_offset": offsets, "seq_lens": lens, "num_free": free}
    if s["op"] == "append":
        gdpa.append_kv_cache_fp8(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["slots"])
        return {n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}
    return gdpa.generalized_dot_product_attention_paged_fp8(
        s["query"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["block_tables"], s["query_offset"], s["seq_lens"], s["max_q"],
        qk_scale=s["scale"], activation=s["activation"], is_causal=s["causal"], window_size=s["window"])


def _tables_plain(s):
    S, width, table = s["block"], s["width"], s["block_tables"]
    cached, new = s["cached_lens"].long(), s["new_lens"].long()
    lens, ends = cached + new, torch.cumsum(new, 0)
    old, tot = (_up(cached, S)).clamp_max(width), (_up(lens, S)).clamp_max(width)
    need = tot - old
    base = torch.cumsum(need, 0) - need
    j = torch.arange(width, device=table.device)
    at = s["num_free"].long() - 1 - (base[:, None] + j - old[:, None])  # the free blocks are a stack
    fresh = torch.where(at >= 0, s["free_blocks"].long()[at.clamp(0, s["free_blocks"].numel() - 1)], -1)
    table.copy_(torch.where((j >= old[:, None]) & (j < tot[:, None]), fresh, table.long()))
    t = torch.arange(s["total_new"], device=table.device)
    b = torch.searchsorted(ends, t, right=True)
    p = cached[b] + t - (ends - new)[b]
    block = torch.where(p // S < width, table.long()[b, (p // S).clamp_max(width - 1)], -1)
    slots = torch.where(block >= 0, block * S + p % S, -1)
    offsets = torch.cat([ends.new_zeros(1), ends])
    return {"block_tables": table, "slots": slots, "query_offset": offsets.int(), "seq_lens": lens.int(),
            "num_free": (s["num_free"].long() - need.sum()).int()}


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


def _append_plain(s):
    _append_one(s["key"], s["k_cache"], s["k_scales"], s["slots"], s["most_runs"])
    _append_one(s["value"], s["v_cache"], s["v_scales"], s["slots"], s["most_runs"])
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}


def _gather(cache, scales, table):
    """The rows of a batch of requests in fp32: [requests, heads, tokens, dim]."""
    x = cache.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scales[table][:, :, None, :, None]
    return x.flatten(1, 2).transpose(1, 2)


_ACTIVATIONS = {
    "silu": lambda x: x / (1 + torch.exp(-x)),
    "gelu_approx": lambda x: 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * x * (1 + 0.044715 * x * x))),
    "relu": lambda x: x.clamp_min(0),
}


def _attend_plain(s):
    table, offsets, lens = s["block_tables"].long().clamp_min(0), s["query_offset"].long(), s["seq_lens"].long()
    k, v = _gather(s["k_cache"], s["k_scales"], table), _gather(s["v_cache"], s["v_scales"], table)
    B, Hk, N, D = k.shape
    T, H = s["query"].shape[:2]
    t = torch.arange(T, device=k.device)
    b = torch.searchsorted(offsets, t, right=True) - 1
    i = t - offsets[b]
    rows = (offsets[:-1, None] + torch.arange(s["max_q"], device=k.device)).clamp_max(max(T - 1, 0))
    q = s["query"].float()[rows].unflatten(2, (Hk, H // Hk)).permute(0, 2, 3, 1, 4)  # [B, Hk, group, max_q, D]
    x = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).unflatten(2, (H // Hk, s["max_q"]))
    j = torch.arange(N, device=k.device)
    p = (lens - (offsets[1:] - offsets[:-1]))[:, None, None] + torch.arange(s["max_q"], device=k.device)[:, None]
    keep = (j < lens[:, None, None]).expand(B, s["max_q"], N)
    if s["causal"]:
        keep = keep & (j <= p)
    if s["window"] is not None:
        keep = keep & ((j - p).abs() <= s["window"])
    keep = keep[:, None, None]
    if s["activation"] == "softmax":
        x = torch.where(keep, x * s["scale"], -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-3e38))
        x = x / x.sum(-1, keepdim=True).clamp_min(1e-37)
    else:
        x = torch.where(keep, _ACTIVATIONS[s["activation"]](x) * s["scale"], 0)
    o = torch.matmul(x.flatten(2, 3), v).unflatten(2, (H // Hk, s["max_q"])).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, max_q, H, D]
    return o[b, i].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    cached, new = _lengths(case)
    S, H, Hk, D = case["block"], case["heads"], case["kv_heads"], case["head_dim"]
    n = case["batch"]
    if case["op"] == "tables":
        need = int((_up(cached + new, S) - _up(cached, S)).sum())
        partly = int((cached % S != 0).sum())
        return {"bytes": 8 * n + 4 * need + 4 * partly + 4 * need + 8 * int(new.sum()) + 8 * n + 8, "flops": 0}
    if case["op"] == "append":
        values = 2 * int(new.sum()) * Hk * D
        runs = int((_up(cached + new, S) - cached // S).sum())
        return {"bytes": values * ((4 if case["dtype"] == "fp32" else 2) + 1) + 8 * int(new.sum()) + 16 * runs * Hk, "flops": 2 * values}
    first, end, union = _ranges(case)
    n_bytes = 2 * union * Hk * D + 2 * 4 * union // S * Hk + 4 * (union // S) + 2 * 2 * int(new.sum()) * H * D
    return {"bytes": n_bytes, "flops": 4 * H * D * int((end - first).sum())}


# ------------------------------------------------------------------------------------- the same pass in 64 bits


def _e4m3(x):
    """`x` (fp64) rounded to the nearest e4m3 value, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    S, Hk, D = case["block"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        slots = s["slots"].tolist()
        out = {}
        runs, i = [], 0
        while i < len(slots):
            n = 1
            while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % S:
                n += 1
            runs.append((i, n, slots[i] // S, slots[i] % S))
            i += n
        for name, x in (("k", s["key"]), ("v", s["value"])):
            cache, scales = s[name + "_cache"].double(), s[name + "_scales"].double()
            for i, n, block, row in runs:
                new = x[i:i + n].double()
                least = torch.exp2(torch.ceil(torch.log2(new.abs().amax((0, 2)).clamp_min(1e-45) / 448)).clamp_min(-100))
                scale = torch.maximum(scales[block], least) if row else least
                if row:
                    cache[block, :row] = _e4m3(cache[block, :row] * (scales[block] / scale)[:, None])
                cache[block, row:row + n] = _e4m3(new / scale[:, None])
                scales[block] = scale
            out[name + "_cache"], out[name + "_scales"] = cache, scales
        return {n: out[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}
    first, end, _ = _ranges(case)
    cached, new = _lengths(case)
    lens, offsets = s["seq_lens"].tolist(), s["query_offset"].tolist()
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    F = torch.nn.functional
    act = {"silu": F.silu, "gelu_approx": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}
    for b, n in enumerate(lens):
        lo, hi = offsets[b], offsets[b + 1]
        if hi == lo or n == 0:
            continue
        blocks = s["block_tables"][b, :_up(n, S)].long()
        k, v = (s[c + "_cache"].view(torch.uint8)[blocks].view(torch.float8_e4m3fn).double() * s[c + "_scales"][blocks].double()[:, None, :, None]
                for c in ("k", "v"))
        k, v = (t.reshape(-1, Hk, D)[:n].repeat_interleave(case["heads"] // Hk, 1).transpose(0, 1) for t in (k, v))
        x = s["query"][lo:hi].double().transpose(0, 1) @ k.transpose(1, 2)
        p, j = torch.arange(n - (hi - lo), n, device="cuda")[:, None], torch.arange(n, device="cuda")
        off = torch.zeros(hi - lo, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            off |= j > p
        if case["window"] >= 0:
            off |= (j - p).abs() > case["window"]
        if case["activation"] == "softmax":
            w = torch.softmax((x * s["scale"]).masked_fill(off, -math.inf), -1).masked_fill(off.all(1)[:, None], 0)
        else:
            w = (act[case["activation"]](x) * s["scale"]).masked_fill(off, 0)
        out[lo:hi] = (w @ v).transpose(0, 1)
    return out
