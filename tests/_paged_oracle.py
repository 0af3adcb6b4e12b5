"""The paged cache's operators in plain 64-bit form, on the CPU, and how far the kernels may be from them."""
import math

import torch


def tables(block_tables, cached, new, free, num_free, size, total_new):
    """(block_tables, slots, query_offset, seq_lens, num_free) of build_block_tables, request by request."""
    table, width = block_tables.clone(), block_tables.shape[1]
    left, slots, offsets = min(num_free, len(free)), [], [0]
    for b, (c, n) in enumerate(zip(cached, new)):
        for j in range(min(-(-c // size), width), min(-(-(c + n) // size), width)):
            left -= 1
            table[b, j] = free[left] if left >= 0 else -1
        for p in range(c, c + n):
            blk = int(table[b, p // size]) if p // size < width else -1
            slots.append(blk * size + p % size if blk >= 0 else -1)
        offsets.append(offsets[-1] + n)
    slots = (slots + [-1] * total_new)[:total_new]
    return table, torch.tensor(slots, dtype=torch.int64), torch.tensor(offsets), torch.tensor([c + n for c, n in zip(cached, new)]), left


def e4m3_bytes(x):
    """Bytes of the nearest e4m3 values (ties to even) of fp64 `x`; beyond 448: 448; NaN: NaN."""
    x = x.double().clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    r = torch.round(x / step) * step
    return torch.where(torch.isnan(x), x, torch.copysign(r, x)).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)


def least_scale(x):
    x = x.double().abs()
    amax = float(x[torch.isfinite(x)].max()) if torch.isfinite(x).any() else 0.0
    return 2.0 ** max(-100, math.ceil(math.log2(amax / 448))) if amax > 0 else 2.0 ** -100


def append(x, cache, scales, slots):
    """New rows into one cache ([blocks, size, heads, dim] bytes) and its scales (fp64), in place."""
    size, i, slots = cache.shape[1], 0, slots.tolist()
    while i < len(slots):
        if not 0 <= slots[i] < cache.shape[0] * size:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % size:
            n += 1
        blk, row = slots[i] // size, slots[i] % size
        for h in range(cache.shape[2]):
            scale = least_scale(x[i:i + n, h])
            old = float(scales[blk, h])
            if row:
                scale = max(scale, old)
                if scale != old:
                    held = cache[blk, :row, h].view(torch.float8_e4m3fn).double()
                    cache[blk, :row, h] = e4m3_bytes(held * (old / scale))
            cache[blk, row:row + n, h] = e4m3_bytes(x[i:i + n, h].double() / scale)
            scales[blk, h] = scale
        i += n


ACT = {
    "raw": lambda x: x,
    "gelu": lambda x: torch.nn.functional.gelu(x),
    "gelu_approx": lambda x: torch.nn.functional.gelu(x, approximate="tanh"),
    "leaky_relu": lambda x: torch.nn.functional.leaky_relu(x, 0.01),
    "relu": torch.relu,
    "silu": torch.nn.functional.silu,
    "hardswish": torch.nn.functional.hardswish,
    "relu_square": lambda x: torch.relu(x) ** 2,
}


def gather(cache, scales, table, n):
    """(e4m3 values, scales) of a request's first n tokens, [n, heads, dim] and [n, heads], in fp64."""
    size = cache.shape[1]
    t = table[: -(-n // size)].long()
    x = cache[t].view(torch.float8_e4m3fn).double().reshape(-1, *cache.shape[2:])[:n]
    return x, scales[t].double().repeat_interleave(size, 0)[:n]


def attend(query, k, v, ks, vs, table, offsets, lens, scale, activation, causal=False, window=None):
    """(O, tolerance) of generalized_dot_product_attention_paged_fp8; caches as bytes, everything on the CPU.

    What the kernels round, in units that the sums here carry:
      * O to bf16, 2^-9 of it; fp32 steps on the way (2^-8 |O| covers both);
      * P, times V's scale and a factor of its row, to fp16 and then to the sum of two e4m3 values: 2^-11 + 2^-8 of it, or, below the
        smallest normal value of the second, 2^-10 where the row's largest is at least 32 (2^-15 of the row's largest);
        a score's fp32 rounding in P stays below 2^-9 of P for the inputs here (2^-7 |P| covers all three);
      * tanh.approx of an activation: 2^-10.98 of tanh, times |x| / 2 (2^-11 |x| scale covers it).
    """
    out = torch.zeros(query.shape, dtype=torch.float64)
    tol = torch.zeros(query.shape, dtype=torch.float64)
    heads = query.shape[1]
    for b, n in enumerate(lens):
        lo, hi = offsets[b], offsets[b + 1]
        if hi == lo or n == 0:
            continue
        k8, sk = gather(k, ks, table[b], n)
        v8, sv = gather(v, vs, table[b], n)
        group = heads // k8.shape[1]
        p0, j = torch.arange(n - (hi - lo), n)[:, None], torch.arange(n)
        off = torch.zeros(hi - lo, n, dtype=torch.bool)
        if causal:
            off |= j > p0
        if window is not None:
            off |= (j - p0).abs() > window
        for h in range(heads):
            kv = h // group
            x = query[lo:hi, h].double() @ (k8[:, kv] * sk[:, kv, None]).T
            if activation == "softmax":
                p = torch.softmax((x * scale).masked_fill(off, -math.inf), -1).masked_fill(off.all(1)[:, None], 0)
                act_err = 0.0
            else:
                p = (ACT[activation](x) * scale).masked_fill(off, 0)
                act_err = (2.0 ** -11 * x.abs() * abs(scale)).masked_fill(off, 0) if activation in ("gelu_approx", "silu") else torch.zeros_like(x)
            vv = v8[:, kv] * sv[:, kv, None]
            out[lo:hi, h] = p @ vv
            t = 2.0 ** -8 * out[lo:hi, h].abs() + 2.0 ** -7 * (p.abs() @ vv.abs())
            t = t + 2.0 ** -15 * (p.abs() * sv[:, kv]).amax(1, keepdim=True) * ((~off).double() @ v8[:, kv].abs())
            if activation != "softmax":
                t = t + act_err @ vv.abs()
            tol[lo:hi, h] = t
    return out, tol
